// Group norm with an activation (and a dropout mask), channels last: x [B, N, C] (N rows of an item), G groups of cpg = C / G
// adjacent channels, m = N cpg values per (item, group).
//
//   mean = sum x / m     var = sum (x - mean)^2 / m     r = rsqrt(var + eps)
//   xhat = (x - mean) r     z = gamma xhat + beta     y = k s act(z)          k, s: keep bit and factor of the mask (norm_drop.h)
//
//   dz = gy k s act'(z)     gbeta = sum_{b,n} dz     ggamma = sum_{b,n} dz xhat
//   gx = r (gamma dz - c1 - xhat c2)     c1 = sum_group gamma dz / m     c2 = sum_group gamma dz xhat / m
//
// Two launches per direction: partial sums of chunks of rows, then a pass that joins the partials of its groups and applies.  z is
// formed again from x in the backward, so y is not kept.  No atomics: partials are joined in a fixed order.
//
// Statistics: a thread takes the mean of a few rows in registers, then the squared deviations from it, and joins such
// batches by Chan's update of (count, mean, M2); so does everything above it.  Nothing is a difference of large sums, whatever
// the mean of a group is against its deviation.
#include "norm_drop.h"

namespace sfm {
namespace {

#ifndef SFM_GN_TARGET
#define SFM_GN_TARGET 2048
#endif
#ifndef SFM_GN_U
#define SFM_GN_U 4
#endif
#ifndef NT_STATS
#define NT_STATS false
#endif
#ifndef NT_LAST
#define NT_LAST false
#endif
#ifndef NT_STORE
#define NT_STORE false
#endif
#ifndef NT_SUMS
#define NT_SUMS false
#endif
constexpr int kTargetBlocks = SFM_GN_TARGET;  // eight workgroups of four waves per CU
constexpr int kMaxChunks = 512;
constexpr int kU = SFM_GN_U;                  // rows a thread has in flight

// How an item is cut: channels into slabs (whole groups, or an even part of one wide group), rows into chunks.
struct GnPlan {
  long long N;
  int C, G, cpg;
  int V;                 // elements per thread and row
  int cs;                // channels of a slab (the last one of a group or of the row may have fewer)
  int slabs;             // slabs of a row
  int groups_per_slab;   // >= 1; 1 where a group has parts
  int parts;             // slabs of a group (1 where a slab holds whole groups)
  int lanes;             // cs / V
  int row_lanes;         // kBlock / lanes: rows a workgroup takes at once
  int chunks;
  int rows_per_chunk;
  int P;                 // partials of a group: chunks * parts
};

static inline int gcd_int(int a, int b) {
  while (b) { const int t = a % b; a = b; b = t; }
  return a;
}

// (the arguments have been checked; false: an item is too large)
static bool gn_plan(long long B, long long N, int C, int G, int es, GnPlan& p) {
  p.N = N; p.C = C; p.G = G; p.cpg = C / G;
  p.V = 16 / es;
  while (C % p.V) p.V /= 2;
  // a slab of whole groups is a multiple of lcm(cpg, V); where that is too wide for a workgroup and V does not divide a group
  // either (a part of a group has to start at a multiple of V), a smaller V does
  for (;; p.V /= 2) {
    if (p.cpg % p.V == 0) break;
    if (p.cpg / gcd_int(p.cpg, p.V) <= kBlock) break;
  }
  const int unit_groups = p.V / gcd_int(p.cpg, p.V);                      // groups of the smallest slab
  const long long unit = (long long)p.cpg * unit_groups;
  if (unit / p.V <= kBlock) {
    long long k = 1;  // at least 128 bytes of a row, so that a slab's lines are its own
    while (k * unit * es < 128 && k * unit < C) ++k;
    while (k > 1 && k * unit / p.V > kBlock) --k;
    p.groups_per_slab = k * unit_groups < G ? (int)k * unit_groups : G;
    p.cs = p.groups_per_slab * p.cpg;
    p.parts = 1;
    p.slabs = (G + p.groups_per_slab - 1) / p.groups_per_slab;
  } else {
    const int vecs = p.cpg / p.V;
    p.groups_per_slab = 1;
    p.parts = (vecs + kBlock - 1) / kBlock;
    p.cs = (vecs + p.parts - 1) / p.parts * p.V;
    p.parts = (p.cpg + p.cs - 1) / p.cs;
    if ((long long)G * p.parts > 0x7fffffffll) return false;
    p.slabs = G * p.parts;
  }
  p.lanes = p.cs / p.V;
  p.row_lanes = kBlock / p.lanes;
  const long long per = (long long)B * p.slabs, step = (long long)kU * p.row_lanes;
  long long chunks = (kTargetBlocks + per - 1) / per;
  const long long most = (N + step - 1) / step;  // a full batch per thread at least
  if (chunks > most) chunks = most;
  if (chunks > kMaxChunks) chunks = kMaxChunks;
  if (chunks < 1) chunks = 1;
  long long rows = (N + chunks - 1) / chunks;
  if (rows > step) rows = (rows + step - 1) / step * step;  // whole batches in all chunks but the last
  if (rows > 0x7fffffffll) return false;
  p.rows_per_chunk = (int)rows;
  p.chunks = (int)((N + rows - 1) / rows);
  p.P = p.chunks * p.parts;
  return true;
}

// ---- what a workgroup works on
struct Where {
  int b, slab, chunk, part;
  int c0, cc, g0, ng;  // first channel and channels of the slab, first group and groups of it
  long long r0;        // first row, in the item
  int rows;
};
__device__ __forceinline__ Where where(const GnPlan& p, unsigned bid) {
  Where w;
  w.chunk = bid % (unsigned)p.chunks;
  bid /= (unsigned)p.chunks;
  w.slab = bid % (unsigned)p.slabs;
  w.b = bid / (unsigned)p.slabs;
  if (p.parts == 1) {
    w.part = 0;
    w.g0 = w.slab * p.groups_per_slab;
    w.ng = min(p.groups_per_slab, p.G - w.g0);
    w.c0 = w.g0 * p.cpg;
    w.cc = w.ng * p.cpg;
  } else {
    w.g0 = w.slab / p.parts;
    w.part = w.slab % p.parts;
    w.ng = 1;
    w.c0 = w.g0 * p.cpg + w.part * p.cs;
    w.cc = min(p.cs, p.cpg - w.part * p.cs);
  }
  w.r0 = (long long)w.chunk * p.rows_per_chunk;
  w.rows = (int)min((long long)p.rows_per_chunk, p.N - w.r0);
  return w;
}

// The rows of a thread: vector vx of the slab in rows ry, ry + row_lanes, ... of the chunk, one per step, in batches of kU steps.  The
// address of a load is a uniform pointer that moves with the step and a 32-bit offset of the thread (gn_setup keeps row_lanes rows
// under 2^31 bytes).
struct Rows {
  int vx, ry;
  bool mine;     // this thread has a vector at all
  int steps;     // of the chunk
  int last;      // rows of its last step (1 .. row_lanes)
  int full;      // steps in which every row lane has a row
  __device__ __forceinline__ Rows(const GnPlan& p, const Where& w) {
    vx = threadIdx.x % (unsigned)p.lanes;
    ry = threadIdx.x / (unsigned)p.lanes;
    mine = ry < p.row_lanes && vx * p.V < w.cc;
    steps = (w.rows + p.row_lanes - 1) / p.row_lanes;
    last = w.rows - (steps - 1) * p.row_lanes;
    full = last == p.row_lanes ? steps : steps - 1;
  }
  __device__ __forceinline__ bool valid(int t) const { return t < steps - 1 || (t == steps - 1 && ry < last); }
};

template <int DT, int V, bool NT = false> struct Stream {
  static constexpr int kES = ElemBytes<DT>::value;
  const char* base;
  long long step;
  unsigned off, back;  // back: in the last step a row lane without a row reads row lane 0's
  __device__ __forceinline__ Stream(const void* p, long long ld, const GnPlan& pl, const Where& w, const Rows& r) {
    base = static_cast<const char*>(p) + (((long long)w.b * pl.N + w.r0) * ld + w.c0) * kES;
    step = (long long)pl.row_lanes * ld * kES;
    off = (unsigned)((r.ry * ld + r.vx * V) * kES);
    back = r.ry < r.last ? 0u : (unsigned)(r.ry * ld * kES);
  }
  __device__ __forceinline__ Raw<DT, V> load(const Rows& r, int t) const {  // t < r.steps, uniform
    return load_raw<DT, V, NT>(base + t * step, off - (t < r.steps - 1 ? 0u : back));
  }
  __device__ __forceinline__ void batch(const Rows& r, int t0, Raw<DT, V> (&raw)[kU]) const {
    if (t0 + kU <= r.full) {
      const char* at = base + t0 * step;
#pragma unroll
      for (int u = 0; u < kU; ++u) { raw[u] = load_raw<DT, V, NT>(at, off); at += step; }
    } else {
#pragma unroll
      for (int u = 0; u < kU; ++u)
        if (t0 + u < r.steps) raw[u] = load(r, t0 + u);
    }
  }
};
template <int DT, int V, bool NT>
__device__ __forceinline__ void store_row(const Stream<DT, V, NT>& s, int t, const float (&f)[V]) {
  store_vec<DT, V, NT>(const_cast<char*>(s.base) + t * s.step, s.off, f);
}

// Teams: the workgroup's threads, cut into teams of T lanes of one wave (T a power of two), one group each at a time.
struct Team { int T, id, lane, count; };
__device__ __forceinline__ Team team_of(int ng) {
  int T = 64;
  while (T > 1 && kBlock / T < ng) T >>= 1;
  return {T, (int)threadIdx.x / T, (int)threadIdx.x & (T - 1), kBlock / T};
}
template <typename F> __device__ __forceinline__ F team_sum(F v, int T) {
  for (int o = T >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// values that partial q of a group covers
__device__ __forceinline__ double part_count(const GnPlan& p, int q) {
  const int chunk = p.parts == 1 ? q : q / p.parts, part = q - chunk * p.parts;
  const int rows = chunk == p.chunks - 1 ? (int)(p.N - (long long)chunk * p.rows_per_chunk) : p.rows_per_chunk;
  return (double)rows * (p.parts == 1 ? p.cpg : min(p.cs, p.cpg - part * p.cs));
}

// ---- forward, first launch: part [B][G][P] (mean, M2).  ONE: the V channels of a vector are of one group (V divides cpg), and a
// thread has one pair for them; else one pair per channel.
template <int DT, int V, bool ONE>
__global__ __launch_bounds__(kBlock) void gn_stats_kernel(const void* __restrict__ x, long long ldx, GnPlan p,
                                                          float2* __restrict__ part) {
  constexpr int A = ONE ? 1 : V, E = V / A;  // accumulators, and elements of one in a row
  __shared__ float2 red[kBlock * A];         // [row lane][vector or channel of the slab]
  const Where w = where(p, blockIdx.x);
  const Rows r(p, w);
  if (r.mine) {
    const Stream<DT, V, NT_STATS> xs(x, ldx, p, w, r);
    float n = 0.0f, mean[A], m2[A];
#pragma unroll
    for (int a = 0; a < A; ++a) { mean[a] = 0.0f; m2[a] = 0.0f; }
    Raw<DT, V> raw[kU];
    int t = 0;
    for (; t + kU <= r.full; t += kU) {
      xs.batch(r, t, raw);
      float s[A], q[A];
#pragma unroll
      for (int a = 0; a < A; ++a) { s[a] = 0.0f; q[a] = 0.0f; }
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float f[V];
        unpack<DT, V>(raw[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) s[k / E] += f[k];
      }
#pragma unroll
      for (int a = 0; a < A; ++a) s[a] *= 1.0f / (kU * E);
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        float f[V];
        unpack<DT, V>(raw[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) { const float d = f[k] - s[k / E]; q[k / E] = __builtin_fmaf(d, d, q[k / E]); }
      }
      const float nn = n + kU * E, share = (kU * E) / nn, cross = n * share;
#pragma unroll
      for (int a = 0; a < A; ++a) {
        const float delta = s[a] - mean[a];
        mean[a] = __builtin_fmaf(delta, share, mean[a]);
        m2[a] += __builtin_fmaf(delta * delta, cross, q[a]);
      }
      n = nn;
    }
    for (; t < r.steps; ++t) {  // fewer than kU steps, and the last one where it is not full
      if (!r.valid(t)) break;
      float f[V], s[A], q[A];
      unpack<DT, V>(xs.load(r, t), f);
#pragma unroll
      for (int a = 0; a < A; ++a) { s[a] = 0.0f; q[a] = 0.0f; }
#pragma unroll
      for (int k = 0; k < V; ++k) s[k / E] += f[k];
#pragma unroll
      for (int a = 0; a < A; ++a) s[a] *= 1.0f / E;
#pragma unroll
      for (int k = 0; k < V; ++k) { const float d = f[k] - s[k / E]; q[k / E] = __builtin_fmaf(d, d, q[k / E]); }
      const float nn = n + E, share = E / nn, cross = n * share;
#pragma unroll
      for (int a = 0; a < A; ++a) {
        const float delta = s[a] - mean[a];
        mean[a] = __builtin_fmaf(delta, share, mean[a]);
        m2[a] += __builtin_fmaf(delta * delta, cross, q[a]);
      }
      n = nn;
    }
#pragma unroll
    for (int a = 0; a < A; ++a) red[(r.ry * p.lanes + r.vx) * A + a] = make_float2(mean[a], m2[a]);
  }
  __syncthreads();
  // over the row lanes and the vectors of a group.  Means are taken against one of them, so a common part costs no digits.
  const Team tm = team_of(w.ng);
  const int per_row = (p.parts == 1 ? p.cpg : w.cc) / E;           // pairs of a group in a row lane
  const int busy = r.steps > 1 ? p.row_lanes : r.last;             // row lanes that have seen a row
  const float inv = 1.0f / ((float)w.rows * per_row);
  for (int j = tm.id; j < w.ng; j += tm.count) {
    const float ref = red[j * per_row].x;
    float s = 0.0f;
    for (int e = tm.lane; e < busy * per_row; e += tm.T) {
      const int l = e / per_row, c = e - l * per_row;
      s = __builtin_fmaf((float)(r.steps - 1 + (l < r.last)), red[l * p.lanes * A + j * per_row + c].x - ref, s);
    }
    const float off = team_sum(s, tm.T) * inv;
    float q = 0.0f;
    for (int e = tm.lane; e < busy * per_row; e += tm.T) {
      const int l = e / per_row, c = e - l * per_row;
      const float2 v = red[l * p.lanes * A + j * per_row + c];
      const float d = (v.x - ref) - off;
      q += __builtin_fmaf((float)(E * (r.steps - 1 + (l < r.last))) * d, d, v.y);
    }
    q = team_sum(q, tm.T);
    if (tm.lane == 0) part[((long long)w.b * p.G + w.g0 + j) * p.P + w.chunk * p.parts + w.part] = make_float2(ref + off, q);
  }
}

// joins the partials of a workgroup's groups: stat[j] = (mean, r) in LDS.  All threads call it; it ends with a barrier.
__device__ __forceinline__ void join_stats(const float2* __restrict__ part, const GnPlan& p, const Where& w, float eps,
                                           float2* __restrict__ stat) {
  const Team t = team_of(w.ng);
  const double inv = 1.0 / ((double)p.N * p.cpg);
  for (int j = t.id; j < w.ng; j += t.count) {
    const float2* src = part + ((long long)w.b * p.G + w.g0 + j) * p.P;
    const float ref = src[0].x;
    double s = 0.0;
    for (int q = t.lane; q < p.P; q += t.T) s += part_count(p, q) * (src[q].x - ref);
    const double off = team_sum(s, t.T) * inv;
    double q2 = 0.0;
    for (int q = t.lane; q < p.P; q += t.T) {
      const float2 v = src[q];
      const double d = (v.x - ref) - off;
      q2 += v.y + part_count(p, q) * d * d;
    }
    q2 = team_sum(q2, t.T);
    if (t.lane == 0) stat[j] = make_float2((float)(ref + off), (float)(1.0 / sqrt(q2 * inv + (double)eps)));
  }
  __syncthreads();
}

// ---- forward, second launch.  The first batch is on its way while the partials are joined.
template <int DT, int V, bool ONE, bool DROP>
__global__ __launch_bounds__(kBlock) void gn_apply_kernel(const void* __restrict__ x, long long ldx,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          const float2* __restrict__ part, GnPlan p, float eps, int act, Drop drop,
                                                          void* __restrict__ y, long long ldy, float* __restrict__ save_mean,
                                                          float* __restrict__ save_r) {
  constexpr int A = ONE ? 1 : V, E = V / A;
  __shared__ float2 stat[kBlock * A];
  const Where w = where(p, blockIdx.x);
  const Rows r(p, w);
  const Stream<DT, V, NT_LAST> xs(x, ldx, p, w, r);
  const Stream<DT, V, NT_STORE> ys(y, ldy, p, w, r);
  Raw<DT, V> raw[kU];
  float sc[V], sh[V];
  const int c = w.c0 + r.vx * V;
  if (r.mine) {
    xs.batch(r, 0, raw);
#pragma unroll
    for (int k = 0; k < V; ++k) { sc[k] = gamma[c + k]; sh[k] = beta[c + k]; }
  }
  join_stats(part, p, w, eps, stat);
  if (save_mean && w.chunk == 0 && w.part == 0)
    for (int j = threadIdx.x; j < w.ng; j += kBlock) {
      save_mean[(long long)w.b * p.G + w.g0 + j] = stat[j].x;
      save_r[(long long)w.b * p.G + w.g0 + j] = stat[j].y;
    }
  if (!r.mine) return;
  float mu[A];
#pragma unroll
  for (int a = 0; a < A; ++a) {
    const float2 st = stat[(c + a * E) / p.cpg - w.g0];
    mu[a] = st.x;
#pragma unroll
    for (int k = a * E; k < (a + 1) * E; ++k) sc[k] *= st.y;
  }
  DropKey key{};
  unsigned keep = 0;
  if (DROP) {
    key = drop_key(drop);
    if (drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, c);
  }
  const unsigned long long place = (unsigned long long)(w.r0 + r.ry) * p.C + c;
  for (int t = 0;;) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (t + u >= r.steps) break;
      float f[V];
      unpack<DT, V>(raw[u], f);
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = __builtin_fmaf(f[k] - mu[k / E], sc[k], sh[k]);
      act_fwd<V>(f, act);
      if (DROP) {
        if (!drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, place + (unsigned long long)(t + u) * p.row_lanes * p.C);
        drop_apply<V>(f, keep, drop.scale);
      }
      if (r.valid(t + u)) store_row(ys, t + u, f);
    }
    t += kU;
    if (t >= r.steps) break;
    xs.batch(r, t, raw);
  }
}

// dL/dy: the sum of up to three tensors, each a channel slice with its own row stride (what an activation's several readers
// hand back in a decoder level without concats)
struct GySrc {
  const void* p[3];
  long long ld[3];
  int n;
};
template <int DT, int V>
__device__ __forceinline__ void add_more_gy(const GySrc& s, const GnPlan& p, const Where& w, const Rows& r, int t, float (&g)[V]) {
  for (int k = 1; k < s.n; ++k) {  // uniform
    const Stream<DT, V> more(s.p[k], s.ld[k], p, w, r);
    float f[V];
    unpack<DT, V>(more.load(r, t), f);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] += f[e];
  }
}

// ---- backward, first launch: per_group [B][G][P] (sum gamma dz, sum gamma dz xhat), per_channel [C][B][chunks] (sum dz, sum dz xhat)
template <int DT, int V, bool ONE, bool DROP>
__global__ __launch_bounds__(kBlock) void gn_bwd_sums_kernel(const void* __restrict__ x, long long ldx, GySrc gy,
                                                             const float* __restrict__ gamma, const float* __restrict__ beta,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             GnPlan p, int B, int act, Drop drop, float2* __restrict__ per_group,
                                                             float2* __restrict__ per_channel) {
  constexpr int A = ONE ? 1 : V, E = V / A;
  __shared__ float2 red[kBlock * V];
  const Where w = where(p, blockIdx.x);
  const Rows r(p, w);
  if (r.mine) {
    const Stream<DT, V, NT_SUMS> xs(x, ldx, p, w, r), gs(gy.p[0], gy.ld[0], p, w, r);
    Raw<DT, V> xr[kU], gr[kU];
    xs.batch(r, 0, xr);
    gs.batch(r, 0, gr);
    const int c = w.c0 + r.vx * V;
    float mu[A], is[A], ga[V], be[V], s1[V], s2[V];
#pragma unroll
    for (int a = 0; a < A; ++a) {
      const long long g = (long long)w.b * p.G + (c + a * E) / p.cpg;
      mu[a] = mean[g]; is[a] = rstd[g];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) { ga[k] = gamma[c + k]; be[k] = beta[c + k]; s1[k] = 0.0f; s2[k] = 0.0f; }
    DropKey key{};
    unsigned keep = 0;
    if (DROP) {
      key = drop_key(drop);
      if (drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, c);
    }
    const unsigned long long place = (unsigned long long)(w.r0 + r.ry) * p.C + c;
    for (int t = 0;;) {
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        if (t + u >= r.steps) break;
        if (!r.valid(t + u)) break;
        float f[V], g[V], z[V];
        unpack<DT, V>(xr[u], f);
        unpack<DT, V>(gr[u], g);
        if (gy.n > 1) add_more_gy<DT, V>(gy, p, w, r, t + u, g);
        if (DROP) {
          if (!drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, place + (unsigned long long)(t + u) * p.row_lanes * p.C);
          drop_apply<V>(g, keep, drop.scale);
        }
#pragma unroll
        for (int k = 0; k < V; ++k) { f[k] = (f[k] - mu[k / E]) * is[k / E]; z[k] = __builtin_fmaf(f[k], ga[k], be[k]); }
        act_bwd<V>(g, z, act);
#pragma unroll
        for (int k = 0; k < V; ++k) { s1[k] += g[k]; s2[k] = __builtin_fmaf(g[k], f[k], s2[k]); }
      }
      t += kU;
      if (t >= r.steps) break;
      xs.batch(r, t, xr);
      gs.batch(r, t, gr);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) red[r.ry * p.cs + r.vx * V + k] = make_float2(s1[k], s2[k]);
  }
  __syncthreads();
  // over the row lanes: S threads per channel take every S-th row lane each, then one adds the S.  In order: the same bits every time.
  const int S = max(1, kBlock / w.cc);
  const int cl = threadIdx.x % (unsigned)w.cc, seg = threadIdx.x / (unsigned)w.cc;
  for (int c = cl; seg < S && c < w.cc; c += kBlock) {  // (cc > kBlock: S = 1 and a thread has several channels)
    float a = 0.0f, b = 0.0f;
    for (int l = seg; l < p.row_lanes; l += S) { const float2 v = red[l * p.cs + c]; a += v.x; b += v.y; }
    if (seg < p.row_lanes) red[seg * p.cs + c] = make_float2(a, b);  // (only this thread reads or writes that place)
  }
  __syncthreads();
  const int left = min(S, p.row_lanes);
  for (int c = threadIdx.x; c < w.cc; c += kBlock) {
    float2 v = red[c];
    for (int l = 1; l < left; ++l) { const float2 o = red[l * p.cs + c]; v.x += o.x; v.y += o.y; }
    red[c] = v;
    per_channel[((long long)(w.c0 + c) * B + w.b) * p.chunks + w.chunk] = v;
  }
  __syncthreads();
  const Team t = team_of(w.ng);
  const int cg = p.parts == 1 ? p.cpg : w.cc;
  for (int j = t.id; j < w.ng; j += t.count) {
    float a = 0.0f, b = 0.0f;
    for (int e = t.lane; e < cg; e += t.T) {
      const float2 v = red[j * cg + e];
      const float ga = gamma[w.c0 + j * cg + e];
      a = __builtin_fmaf(ga, v.x, a);
      b = __builtin_fmaf(ga, v.y, b);
    }
    a = team_sum(a, t.T);
    b = team_sum(b, t.T);
    if (t.lane == 0) per_group[((long long)w.b * p.G + w.g0 + j) * p.P + w.chunk * p.parts + w.part] = make_float2(a, b);
  }
}

// ---- backward, second launch: the first param_blocks workgroups sum the channel partials over items and chunks (a wave per
// channel), the others write gx
template <int DT, int V, bool ONE, bool DROP>
__global__ __launch_bounds__(kBlock) void gn_bwd_apply_kernel(const void* __restrict__ x, long long ldx, GySrc gy,
                                                              const float* __restrict__ gamma, const float* __restrict__ beta,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              GnPlan p, int B, int act, Drop drop,
                                                              const float2* __restrict__ per_group,
                                                              const float2* __restrict__ per_channel, unsigned param_blocks,
                                                              void* __restrict__ gx, float* __restrict__ ggamma,
                                                              float* __restrict__ gbeta) {
  constexpr int A = ONE ? 1 : V, E = V / A;
  __shared__ float2 stat[kBlock * A];
  if (blockIdx.x < param_blocks) {
    const int c = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (c >= p.C) return;
    const long long n = (long long)B * p.chunks;
    const float2* src = per_channel + c * n;
    double a = 0.0, b = 0.0;
    for (long long k = lane; k < n; k += 64) { const float2 v = src[k]; a += v.x; b += v.y; }
    a = team_sum(a, 64);
    b = team_sum(b, 64);
    if (lane == 0) { gbeta[c] = (float)a; ggamma[c] = (float)b; }
    return;
  }
  const Where w = where(p, blockIdx.x - param_blocks);
  const Rows r(p, w);
  const Stream<DT, V, NT_LAST> xs(x, ldx, p, w, r), gs(gy.p[0], gy.ld[0], p, w, r);
  const Stream<DT, V, NT_STORE> os(gx, p.C, p, w, r);
  Raw<DT, V> xr[kU], gr[kU];
  const int c = w.c0 + r.vx * V;
  float mu[A], is[A], ga[V], be[V], c1[A], c2[A];
  if (r.mine) {
    xs.batch(r, 0, xr);
    gs.batch(r, 0, gr);
#pragma unroll
    for (int a = 0; a < A; ++a) {
      const long long g = (long long)w.b * p.G + (c + a * E) / p.cpg;
      mu[a] = mean[g]; is[a] = rstd[g];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) { ga[k] = gamma[c + k]; be[k] = beta[c + k]; }
  }
  {
    const Team t = team_of(w.ng);
    const double inv = 1.0 / ((double)p.N * p.cpg);
    for (int j = t.id; j < w.ng; j += t.count) {
      const float2* src = per_group + ((long long)w.b * p.G + w.g0 + j) * p.P;
      double a = 0.0, b = 0.0;
      for (int q = t.lane; q < p.P; q += t.T) { const float2 v = src[q]; a += v.x; b += v.y; }
      a = team_sum(a, t.T);
      b = team_sum(b, t.T);
      if (t.lane == 0) stat[j] = make_float2((float)(a * inv), (float)(b * inv));
    }
    __syncthreads();
  }
  if (!r.mine) return;
#pragma unroll
  for (int a = 0; a < A; ++a) {
    const float2 st = stat[(c + a * E) / p.cpg - w.g0];
    c1[a] = st.x;
    c2[a] = st.y;
  }
  DropKey key{};
  unsigned keep = 0;
  if (DROP) {
    key = drop_key(drop);
    if (drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, c);
  }
  const unsigned long long place = (unsigned long long)(w.r0 + r.ry) * p.C + c;
  for (int t = 0;;) {
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (t + u >= r.steps) break;
      float f[V], g[V], z[V];
      unpack<DT, V>(xr[u], f);
      unpack<DT, V>(gr[u], g);
      if (gy.n > 1) add_more_gy<DT, V>(gy, p, w, r, t + u, g);
      if (DROP) {
        if (!drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, place + (unsigned long long)(t + u) * p.row_lanes * p.C);
        drop_apply<V>(g, keep, drop.scale);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) { f[k] = (f[k] - mu[k / E]) * is[k / E]; z[k] = __builtin_fmaf(f[k], ga[k], be[k]); }
      act_bwd<V>(g, z, act);
#pragma unroll
      for (int k = 0; k < V; ++k)
        g[k] = is[k / E] * __builtin_fmaf(-f[k], c2[k / E], __builtin_fmaf(ga[k], g[k], -c1[k / E]));
      if (r.valid(t + u)) store_row(os, t + u, g);
    }
    t += kU;
    if (t >= r.steps) break;
    xs.batch(r, t, xr);
    gs.batch(r, t, gr);
  }
}

// dispatch on the type, the vector width and whether a vector lies in one group: fn(DT, V, ONE) as integral constants
template <typename F> static void by_type(int dtype, const GnPlan& p, F&& fn) {
  using std::integral_constant;
  const bool one = p.cpg % p.V == 0;
  auto width = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    auto go = [&](auto v) {
      if (one) fn(dt, v, std::true_type{});
      else if constexpr (decltype(v)::value > 1) fn(dt, v, std::false_type{});
    };
    if constexpr (DT != kF32) { if (p.V == 8) return go(integral_constant<int, 8>{}); }
    if (p.V == 4) return go(integral_constant<int, 4>{});
    if (p.V == 2) return go(integral_constant<int, 2>{});
    go(integral_constant<int, 1>{});
  };
  if (dtype == kF32) return width(integral_constant<int, kF32>{});
  if (dtype == kBF16) return width(integral_constant<int, kBF16>{});
  width(integral_constant<int, kF16>{});
}

}  // namespace
}  // namespace sfm

using namespace sfm;

// rows of C elements of es bytes, ld elements apart
static bool rows_ok(const void* q, long long ld, int C, int es) { return q && ld >= C && ((uintptr_t)q & (es - 1)) == 0; }

// ld: the widest row stride of the call
static int gn_setup(long long B, long long N, int C, int G, int dtype, long long ld, GnPlan& p, unsigned& grid) {
  if (dtype < kF32 || dtype > kF16 || B < 1 || N < 1 || C < 1 || G < 1 || C % G || ld < C) return SFM_ERR_ARG;
  const int es = dtype == kF32 ? 4 : 2;
  // items are counted in 32 bits, workgroups in 31, elements in 60 with room for strides; the rows that a workgroup takes at once
  // lie within 31 bits of bytes of each other
  if (B > 0x7fffffffll || (__int128)B * N > ((__int128)1 << 40) || ld > 0x7fffffffll / es || !gn_plan(B, N, C, G, es, p))
    return SFM_ERR_TOO_LARGE;
  p.row_lanes = (int)std::min<long long>(p.row_lanes, 0x7fffffffll / (ld * es));
  const __int128 blocks = (__int128)B * p.slabs * p.chunks;
  if (blocks + C > 0x7fffffffll) return SFM_ERR_TOO_LARGE;
  grid = (unsigned)blocks;
  return SFM_OK;
}

extern "C" long long sfm_group_norm_workspace_floats(long long B, long long N, int C, int G, int dtype, int backward) {
  GnPlan p;
  unsigned grid;
  const int rc = gn_setup(B, N, C, G, dtype, C, p, grid);
  if (rc) return rc;
  return 2 * (B * G * p.P + (backward ? B * C * p.chunks : 0));
}

extern "C" int sfm_group_norm_act_fwd(const void* x, long long ld_x, int dtype, const float* gamma, const float* beta, long long B,
                                      long long N, int C, int G, float eps, int act, const void* rng, unsigned long long seed,
                                      unsigned step, unsigned layer, unsigned item0, int threshold, int per_channel, void* y,
                                      long long ld_y, float* save_mean, float* save_rstd, float* ws, void* stream_) {
  GnPlan p;
  Drop d;
  unsigned grid;
  const int es = dtype == kF32 ? 4 : 2;
  const int rc = gn_setup(B, N, C, G, dtype, std::max(ld_x, ld_y), p, grid);
  if (rc) return rc;
  if (!rows_ok(x, ld_x, C, es) || !rows_ok(y, ld_y, C, es) || !gamma || !beta || !ws || ((uintptr_t)ws & 7) || !(eps > 0.0f) ||
      act < kActNone || act > kActSilu || (!save_mean != !save_rstd) ||
      !drop_args(rng, seed, step, layer, item0, threshold, per_channel, d))
    return SFM_ERR_ARG;
  if (threshold && ((__int128)N * C > ((__int128)1 << 35) || B > 0xffffffffll - item0)) return SFM_ERR_TOO_LARGE;
  hipStream_t stream = (hipStream_t)stream_;
  float2* part = reinterpret_cast<float2*>(ws);
  by_type(dtype, p, [&](auto dt, auto v, auto one) {
    constexpr int DT = decltype(dt)::value, V = decltype(v)::value;
    constexpr bool ONE = decltype(one)::value;
    hipLaunchKernelGGL((gn_stats_kernel<DT, V, ONE>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, p, part);
    if (threshold)
      hipLaunchKernelGGL((gn_apply_kernel<DT, V, ONE, true>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, gamma, beta, part, p, eps, act,
                         d, y, ld_y, save_mean, save_rstd);
    else
      hipLaunchKernelGGL((gn_apply_kernel<DT, V, ONE, false>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, gamma, beta, part, p, eps,
                         act, d, y, ld_y, save_mean, save_rstd);
  });
  return sfm_last_error();
}

extern "C" int sfm_group_norm_act_bwd(const void* x, long long ld_x, int dtype, const void* const* gy, const long long* ld_gy,
                                      int n_gy, const float* gamma, const float* beta, const float* save_mean,
                                      const float* save_rstd, long long B, long long N, int C, int G, int act, const void* rng,
                                      unsigned long long seed, unsigned step, unsigned layer, unsigned item0, int threshold,
                                      int per_channel, void* gx, float* ggamma, float* gbeta, float* ws, void* stream_) {
  GnPlan p;
  Drop d;
  unsigned grid;
  const int es = dtype == kF32 ? 4 : 2;
  if (!gy || !ld_gy || n_gy < 1 || n_gy > 3) return SFM_ERR_ARG;
  long long ld = ld_x;
  for (int k = 0; k < n_gy; ++k) ld = std::max(ld, ld_gy[k]);
  const int rc = gn_setup(B, N, C, G, dtype, ld, p, grid);
  if (rc) return rc;
  if (!rows_ok(x, ld_x, C, es) || !gamma || !beta || !save_mean || !save_rstd ||
      (!gx && !ggamma) || (gx && !rows_ok(gx, C, C, es)) || (!ggamma != !gbeta) || !ws || ((uintptr_t)ws & 7) || act < kActNone ||
      act > kActSilu || !drop_args(rng, seed, step, layer, item0, threshold, per_channel, d))
    return SFM_ERR_ARG;
  if (threshold && ((__int128)N * C > ((__int128)1 << 35) || B > 0xffffffffll - item0)) return SFM_ERR_TOO_LARGE;
  GySrc src{};
  src.n = n_gy;
  for (int k = 0; k < n_gy; ++k) {
    if (!rows_ok(gy[k], ld_gy[k], C, es)) return SFM_ERR_ARG;
    src.p[k] = gy[k];
    src.ld[k] = ld_gy[k];
  }
  hipStream_t stream = (hipStream_t)stream_;
  float2* per_group = reinterpret_cast<float2*>(ws);
  float2* per_channel_sums = per_group + B * G * p.P;
  const unsigned params = ggamma ? (unsigned)((C + kBlock / 64 - 1) / (kBlock / 64)) : 0u;
  const unsigned second = params + (gx ? grid : 0u);
  by_type(dtype, p, [&](auto dt, auto v, auto one) {
    constexpr int DT = decltype(dt)::value, V = decltype(v)::value;
    constexpr bool ONE = decltype(one)::value;
    auto both = [&](auto dropped) {
      constexpr bool DROP = decltype(dropped)::value;
      hipLaunchKernelGGL((gn_bwd_sums_kernel<DT, V, ONE, DROP>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, src, gamma, beta, save_mean,
                         save_rstd, p, (int)B, act, d, per_group, per_channel_sums);
      hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, V, ONE, DROP>), dim3(second), dim3(kBlock), 0, stream, x, ld_x, src, gamma, beta,
                         save_mean, save_rstd, p, (int)B, act, d, per_group, per_channel_sums, params, gx, ggamma, gbeta);
    };
    if (threshold) both(std::true_type{});
    else both(std::false_type{});
  });
  return sfm_last_error();
}
