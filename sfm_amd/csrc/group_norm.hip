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

constexpr int kTargetBlocks = 2048;  // eight workgroups of four waves per CU
constexpr int kMaxChunks = 512;

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
  long long rows_per_chunk;
  int P;                 // partials of a group: chunks * parts
};

static inline int gcd_int(int a, int b) {
  while (b) { const int t = a % b; a = b; b = t; }
  return a;
}

static bool gn_plan(long long B, long long N, int C, int G, int es, GnPlan& p) {
  if (B < 1 || N < 1 || C < 1 || G < 1 || C % G) return false;
  p.N = N; p.C = C; p.G = G; p.cpg = C / G;
  p.V = 16 / es;
  while (C % p.V) p.V /= 2;
  // a slab of whole groups is a multiple of lcm(cpg, V); where that is too wide for a workgroup and V does not divide a group
  // either (a part of a group has to start at a multiple of V), a smaller V does
  for (;; p.V /= 2) {
    if (p.cpg % p.V == 0) break;
    if ((long long)p.cpg / gcd_int(p.cpg, p.V) <= kBlock) break;
  }
  const int unit_groups = p.V / gcd_int(p.cpg, p.V);                      // groups of the smallest slab
  const int unit = p.cpg * unit_groups;
  if (unit / p.V <= kBlock) {
    int k = 1;  // at least 128 bytes of a row, so that a slab's lines are its own
    while (k * unit * es < 128 && k * unit < C) ++k;
    while (k > 1 && k * unit / p.V > kBlock) --k;
    p.groups_per_slab = k * unit_groups < G ? k * unit_groups : G;
    p.cs = p.groups_per_slab * p.cpg;
    p.parts = 1;
    p.slabs = (G + p.groups_per_slab - 1) / p.groups_per_slab;
  } else {
    p.groups_per_slab = 1;
    p.parts = (p.cpg + kBlock * p.V - 1) / (kBlock * p.V);
    p.cs = ((p.cpg / p.V + p.parts - 1) / p.parts) * p.V;
    p.parts = (p.cpg + p.cs - 1) / p.cs;
    p.slabs = G * p.parts;
  }
  p.lanes = p.cs / p.V;
  p.row_lanes = kBlock / p.lanes;
  const long long per = (long long)B * p.slabs;
  long long chunks = (kTargetBlocks + per - 1) / per;
  const long long most = (N + 4ll * p.row_lanes - 1) / (4ll * p.row_lanes);  // four rows per thread at least
  if (chunks > most) chunks = most;
  if (chunks > kMaxChunks) chunks = kMaxChunks;
  if (chunks < 1) chunks = 1;
  p.rows_per_chunk = (N + chunks - 1) / chunks;
  p.chunks = (int)((N + p.rows_per_chunk - 1) / p.rows_per_chunk);
  p.P = p.chunks * p.parts;
  return true;
}

// ---- what a workgroup works on
struct Where {
  int b, slab, chunk, part;
  int c0, cc, g0, ng;  // first channel and channels of the slab, first group and groups of it
  long long r0, r1;
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
  w.r0 = w.chunk * p.rows_per_chunk;
  w.r1 = min(p.N, w.r0 + p.rows_per_chunk);
  return w;
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

// values that partial `q` of a group covers
__device__ __forceinline__ double part_count(const GnPlan& p, int q) {
  const int chunk = q / p.parts, part = q - chunk * p.parts;
  const long long rows = min(p.N, (chunk + 1) * p.rows_per_chunk) - chunk * p.rows_per_chunk;
  return (double)rows * (p.parts == 1 ? p.cpg : min(p.cs, p.cpg - part * p.cs));
}

// ---- forward, first launch: part [B][G][P] (mean, M2)
template <int DT, int V>
__global__ __launch_bounds__(kBlock) void gn_stats_kernel(const void* __restrict__ x, long long ldx, GnPlan p,
                                                          float2* __restrict__ part) {
  constexpr int U = 4;
  __shared__ float2 red[kBlock * V];  // [row lane][channel of the slab]
  const Where w = where(p, blockIdx.x);
  const int vx = threadIdx.x % p.lanes, ry = threadIdx.x / p.lanes;
  const bool mine = ry < p.row_lanes && vx * V < w.cc;
  float mean[V], m2[V];
#pragma unroll
  for (int k = 0; k < V; ++k) { mean[k] = 0.0f; m2[k] = 0.0f; }
  float n = 0.0f;
  if (mine) {
    const long long base = (long long)w.b * p.N * ldx + w.c0 + vx * V;
    long long r = w.r0 + ry;
    for (; r + (U - 1) * p.row_lanes < w.r1; r += U * p.row_lanes) {
      Raw<DT, V> raw[U];
#pragma unroll
      for (int u = 0; u < U; ++u) raw[u] = load_raw<DT, V>(x, base + (r + u * p.row_lanes) * ldx);
      float f[U][V];
#pragma unroll
      for (int u = 0; u < U; ++u) unpack<DT, V>(raw[u], f[u]);
      const float nn = n + U, part_new = (float)U / nn, cross = n * part_new;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        float s = 0.0f, q = 0.0f;
#pragma unroll
        for (int u = 0; u < U; ++u) s += f[u][k];
        s *= 1.0f / U;
#pragma unroll
        for (int u = 0; u < U; ++u) { const float d = f[u][k] - s; q = __builtin_fmaf(d, d, q); }
        const float delta = s - mean[k];
        mean[k] = __builtin_fmaf(delta, part_new, mean[k]);
        m2[k] += __builtin_fmaf(delta * delta, cross, q);
      }
      n = nn;
    }
    for (; r < w.r1; r += p.row_lanes) {
      float f[V];
      unpack<DT, V>(load_raw<DT, V>(x, base + r * ldx), f);
      const float nn = n + 1.0f, part_new = 1.0f / nn, cross = n * part_new;
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const float delta = f[k] - mean[k];
        mean[k] = __builtin_fmaf(delta, part_new, mean[k]);
        m2[k] = __builtin_fmaf(delta * delta, cross, m2[k]);
      }
      n = nn;
    }
#pragma unroll
    for (int k = 0; k < V; ++k) red[ry * p.cs + vx * V + k] = make_float2(mean[k], m2[k]);
  }
  __syncthreads();
  const Team t = team_of(w.ng);
  const int cg = p.parts == 1 ? p.cpg : w.cc;  // channels of a group in this slab
  const long long rows = w.r1 - w.r0;
  const int busy = (int)min((long long)p.row_lanes, rows);  // row lanes that have seen a row
  for (int j = t.id; j < w.ng; j += t.count) {
    double s = 0.0;
    for (int e = t.lane; e < busy * cg; e += t.T) {
      const int l = e / cg, c = e - l * cg;
      s += (double)((rows - l + p.row_lanes - 1) / p.row_lanes) * red[l * p.cs + j * cg + c].x;
    }
    const double mu = team_sum(s, t.T) / ((double)rows * cg);
    double q = 0.0;
    for (int e = t.lane; e < busy * cg; e += t.T) {
      const int l = e / cg, c = e - l * cg;
      const float2 v = red[l * p.cs + j * cg + c];
      const double d = v.x - mu;
      q += v.y + (double)((rows - l + p.row_lanes - 1) / p.row_lanes) * d * d;
    }
    q = team_sum(q, t.T);
    if (t.lane == 0) part[((long long)w.b * p.G + w.g0 + j) * p.P + w.chunk * p.parts + w.part] = make_float2((float)mu, (float)q);
  }
}

// joins the partials of a workgroup's groups: stat[j] = (mean, r) in LDS.  All threads call it; it ends with a barrier.
__device__ __forceinline__ void join_stats(const float2* __restrict__ part, const GnPlan& p, const Where& w, float eps,
                                           float2* __restrict__ stat) {
  const Team t = team_of(w.ng);
  const double m = (double)p.N * p.cpg;
  for (int j = t.id; j < w.ng; j += t.count) {
    const float2* src = part + ((long long)w.b * p.G + w.g0 + j) * p.P;
    double s = 0.0;
    for (int q = t.lane; q < p.P; q += t.T) s += part_count(p, q) * src[q].x;
    const double mu = team_sum(s, t.T) / m;
    double q2 = 0.0;
    for (int q = t.lane; q < p.P; q += t.T) {
      const float2 v = src[q];
      const double d = v.x - mu;
      q2 += v.y + part_count(p, q) * d * d;
    }
    q2 = team_sum(q2, t.T);
    if (t.lane == 0) stat[j] = make_float2((float)mu, (float)(1.0 / sqrt(q2 / m + (double)eps)));
  }
  __syncthreads();
}

// ---- forward, second launch
template <int DT, int V, bool DROP>
__global__ __launch_bounds__(kBlock) void gn_apply_kernel(const void* __restrict__ x, long long ldx,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          const float2* __restrict__ part, GnPlan p, float eps, int act, Drop drop,
                                                          void* __restrict__ y, long long ldy, float* __restrict__ save_mean,
                                                          float* __restrict__ save_r) {
  __shared__ float2 stat[kBlock * V];
  const Where w = where(p, blockIdx.x);
  join_stats(part, p, w, eps, stat);
  if (save_mean && w.chunk == 0 && w.part == 0)
    for (int j = threadIdx.x; j < w.ng; j += kBlock) {
      save_mean[(long long)w.b * p.G + w.g0 + j] = stat[j].x;
      save_r[(long long)w.b * p.G + w.g0 + j] = stat[j].y;
    }
  const int vx = threadIdx.x % p.lanes, ry = threadIdx.x / p.lanes;
  if (ry >= p.row_lanes || vx * V >= w.cc) return;
  const int c = w.c0 + vx * V;
  float mu[V], sc[V], sh[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const float2 st = stat[(c + k) / p.cpg - w.g0];
    mu[k] = st.x;
    sc[k] = gamma[c + k] * st.y;
    sh[k] = beta[c + k];
  }
  DropKey key{};
  unsigned keep = 0;
  if (DROP) {
    key = drop_key(drop);
    if (drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, c);
  }
  const long long xb = (long long)w.b * p.N * ldx + c, yb = (long long)w.b * p.N * ldy + c;
#pragma unroll 4
  for (long long r = w.r0 + ry; r < w.r1; r += p.row_lanes) {
    float f[V];
    unpack<DT, V>(load_raw<DT, V>(x, xb + r * ldx), f);
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = __builtin_fmaf(f[k] - mu[k], sc[k], sh[k]);
    act_fwd<V>(f, act);
    if (DROP) {
      if (!drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, (unsigned long long)r * p.C + c);
      drop_apply<V>(f, keep, drop.scale);
    }
    store_vec<DT, V>(y, yb + r * ldy, f);
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
__device__ __forceinline__ void load_gy(const GySrc& s, long long row, int c, float (&g)[V]) {
  unpack<DT, V>(load_raw<DT, V>(s.p[0], row * s.ld[0] + c), g);
  for (int k = 1; k < s.n; ++k) {  // uniform
    float u[V];
    unpack<DT, V>(load_raw<DT, V>(s.p[k], row * s.ld[k] + c), u);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] += u[e];
  }
}

// ---- backward, first launch: per_group [B][G][P] (sum gamma dz, sum gamma dz xhat), per_channel [B][C][chunks] (sum dz, sum dz xhat)
template <int DT, int V, bool DROP>
__global__ __launch_bounds__(kBlock) void gn_bwd_sums_kernel(const void* __restrict__ x, long long ldx, GySrc gy,
                                                             const float* __restrict__ gamma, const float* __restrict__ beta,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             GnPlan p, int act, Drop drop, float2* __restrict__ per_group,
                                                             float2* __restrict__ per_channel) {
  __shared__ float2 red[kBlock * V];
  const Where w = where(p, blockIdx.x);
  const int vx = threadIdx.x % p.lanes, ry = threadIdx.x / p.lanes;
  const bool mine = ry < p.row_lanes && vx * V < w.cc;
  if (mine) {
    const int c = w.c0 + vx * V;
    float mu[V], is[V], ga[V], be[V], s1[V], s2[V];
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const long long g = (long long)w.b * p.G + (c + k) / p.cpg;
      mu[k] = mean[g]; is[k] = rstd[g]; ga[k] = gamma[c + k]; be[k] = beta[c + k];
      s1[k] = 0.0f; s2[k] = 0.0f;
    }
    DropKey key{};
    unsigned keep = 0;
    if (DROP) {
      key = drop_key(drop);
      if (drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, c);
    }
    const long long row0 = (long long)w.b * p.N;
#pragma unroll 2
    for (long long r = w.r0 + ry; r < w.r1; r += p.row_lanes) {
      float f[V], g[V], z[V];
      unpack<DT, V>(load_raw<DT, V>(x, (row0 + r) * ldx + c), f);
      load_gy<DT, V>(gy, row0 + r, c, g);
      if (DROP) {
        if (!drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, (unsigned long long)r * p.C + c);
        drop_apply<V>(g, keep, drop.scale);
      }
#pragma unroll
      for (int k = 0; k < V; ++k) { f[k] = (f[k] - mu[k]) * is[k]; z[k] = __builtin_fmaf(f[k], ga[k], be[k]); }
      act_bwd<V>(g, z, act);
#pragma unroll
      for (int k = 0; k < V; ++k) { s1[k] += g[k]; s2[k] = __builtin_fmaf(g[k], f[k], s2[k]); }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) red[ry * p.cs + vx * V + k] = make_float2(s1[k], s2[k]);
  }
  __syncthreads();
  // over the row lanes, in order; the slab's channel sums stay in row lane 0's place
  for (int c = threadIdx.x; c < w.cc; c += kBlock) {
    float a = 0.0f, b = 0.0f;
    for (int l = 0; l < p.row_lanes; ++l) { const float2 v = red[l * p.cs + c]; a += v.x; b += v.y; }
    red[c] = make_float2(a, b);
    per_channel[((long long)w.b * p.C + w.c0 + c) * p.chunks + w.chunk] = make_float2(a, b);
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
template <int DT, int V, bool DROP>
__global__ __launch_bounds__(kBlock) void gn_bwd_apply_kernel(const void* __restrict__ x, long long ldx, GySrc gy,
                                                              const float* __restrict__ gamma, const float* __restrict__ beta,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              GnPlan p, int B, int act, Drop drop,
                                                              const float2* __restrict__ per_group,
                                                              const float2* __restrict__ per_channel, unsigned param_blocks,
                                                              void* __restrict__ gx, float* __restrict__ ggamma,
                                                              float* __restrict__ gbeta) {
  __shared__ float2 stat[kBlock * V];
  if (blockIdx.x < param_blocks) {
    const int c = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (c >= p.C) return;
    double a = 0.0, b = 0.0;
    for (long long k = lane; k < (long long)B * p.chunks; k += 64) {
      const long long item = k / p.chunks;
      const float2 v = per_channel[(item * p.C + c) * p.chunks + (k - item * p.chunks)];
      a += v.x;
      b += v.y;
    }
    a = team_sum(a, 64);
    b = team_sum(b, 64);
    if (lane == 0) { gbeta[c] = (float)a; ggamma[c] = (float)b; }
    return;
  }
  const Where w = where(p, blockIdx.x - param_blocks);
  {
    const Team t = team_of(w.ng);
    const double m = (double)p.N * p.cpg;
    for (int j = t.id; j < w.ng; j += t.count) {
      const float2* src = per_group + ((long long)w.b * p.G + w.g0 + j) * p.P;
      double a = 0.0, b = 0.0;
      for (int q = t.lane; q < p.P; q += t.T) { const float2 v = src[q]; a += v.x; b += v.y; }
      a = team_sum(a, t.T);
      b = team_sum(b, t.T);
      if (t.lane == 0) stat[j] = make_float2((float)(a / m), (float)(b / m));
    }
    __syncthreads();
  }
  const int vx = threadIdx.x % p.lanes, ry = threadIdx.x / p.lanes;
  if (ry >= p.row_lanes || vx * V >= w.cc) return;
  const int c = w.c0 + vx * V;
  float mu[V], is[V], ga[V], be[V], c1[V], c2[V];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    const int j = (c + k) / p.cpg;
    const long long g = (long long)w.b * p.G + j;
    mu[k] = mean[g]; is[k] = rstd[g]; ga[k] = gamma[c + k]; be[k] = beta[c + k];
    c1[k] = stat[j - w.g0].x; c2[k] = stat[j - w.g0].y;
  }
  DropKey key{};
  unsigned keep = 0;
  if (DROP) {
    key = drop_key(drop);
    if (drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, c);
  }
  const long long row0 = (long long)w.b * p.N;
#pragma unroll 2
  for (long long r = w.r0 + ry; r < w.r1; r += p.row_lanes) {
    float f[V], g[V], z[V];
    unpack<DT, V>(load_raw<DT, V>(x, (row0 + r) * ldx + c), f);
    load_gy<DT, V>(gy, row0 + r, c, g);
    if (DROP) {
      if (!drop.per_channel) keep = keep_bits<V>(drop, key, drop.item0 + w.b, (unsigned long long)r * p.C + c);
      drop_apply<V>(g, keep, drop.scale);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) { f[k] = (f[k] - mu[k]) * is[k]; z[k] = __builtin_fmaf(f[k], ga[k], be[k]); }
    act_bwd<V>(g, z, act);
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] = is[k] * (__builtin_fmaf(ga[k], g[k], -c1[k]) - f[k] * c2[k]);
    store_vec<DT, V>(gx, (row0 + r) * p.C + c, g);
  }
}

// dispatch on the type and the vector width: fn(DT, V) as integral constants
template <typename F> static bool by_type(int dtype, int V, F&& fn) {
  using std::integral_constant;
  auto width = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    switch (V) {
      case 8: if constexpr (DT != kF32) { fn(dt, integral_constant<int, 8>{}); return true; } return false;
      case 4: fn(dt, integral_constant<int, 4>{}); return true;
      case 2: fn(dt, integral_constant<int, 2>{}); return true;
      case 1: fn(dt, integral_constant<int, 1>{}); return true;
    }
    return false;
  };
  if (dtype == kF32) return width(integral_constant<int, kF32>{});
  if (dtype == kBF16) return width(integral_constant<int, kBF16>{});
  return width(integral_constant<int, kF16>{});
}

}  // namespace
}  // namespace sfm

using namespace sfm;

// rows of C elements of es bytes, ld elements apart
static bool rows_ok(const void* q, long long ld, int C, int es) { return q && ld >= C && ((uintptr_t)q & (es - 1)) == 0; }

static int gn_setup(long long B, long long N, int C, int G, int dtype, GnPlan& p, unsigned& grid) {
  if (dtype < kF32 || dtype > kF16 || !gn_plan(B, N, C, G, dtype == kF32 ? 4 : 2, p)) return SFM_ERR_ARG;
  // items are counted in 32 bits, workgroups in 31, elements in 60 with room for strides
  if (B > 0x7fffffffll || (__int128)B * N > ((__int128)1 << 40)) return SFM_ERR_TOO_LARGE;
  const __int128 blocks = (__int128)B * p.slabs * p.chunks;
  if (blocks + C > 0x7fffffffll) return SFM_ERR_TOO_LARGE;
  grid = (unsigned)blocks;
  return SFM_OK;
}

extern "C" long long sfm_group_norm_workspace_floats(long long B, long long N, int C, int G, int dtype, int backward) {
  GnPlan p;
  unsigned grid;
  const int rc = gn_setup(B, N, C, G, dtype, p, grid);
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
  const int rc = gn_setup(B, N, C, G, dtype, p, grid);
  if (rc) return rc;
  if (!rows_ok(x, ld_x, C, es) || !rows_ok(y, ld_y, C, es) || !gamma || !beta || !ws || ((uintptr_t)ws & 7) || !(eps > 0.0f) ||
      act < kActNone || act > kActSilu || (!save_mean != !save_rstd) ||
      !drop_args(rng, seed, step, layer, item0, threshold, per_channel, d))
    return SFM_ERR_ARG;
  if (threshold && ((__int128)N * C > ((__int128)1 << 35) || B > 0xffffffffll - item0)) return SFM_ERR_TOO_LARGE;
  hipStream_t stream = (hipStream_t)stream_;
  float2* part = reinterpret_cast<float2*>(ws);
  by_type(dtype, p.V, [&](auto dt, auto v) {
    constexpr int DT = decltype(dt)::value, V = decltype(v)::value;
    hipLaunchKernelGGL((gn_stats_kernel<DT, V>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, p, part);
    if (threshold)
      hipLaunchKernelGGL((gn_apply_kernel<DT, V, true>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, gamma, beta, part, p, eps, act,
                         d, y, ld_y, save_mean, save_rstd);
    else
      hipLaunchKernelGGL((gn_apply_kernel<DT, V, false>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, gamma, beta, part, p, eps,
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
  const int rc = gn_setup(B, N, C, G, dtype, p, grid);
  if (rc) return rc;
  if (!rows_ok(x, ld_x, C, es) || !gy || !ld_gy || n_gy < 1 || n_gy > 3 || !gamma || !beta || !save_mean || !save_rstd ||
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
  by_type(dtype, p.V, [&](auto dt, auto v) {
    constexpr int DT = decltype(dt)::value, V = decltype(v)::value;
    auto both = [&](auto dropped) {
      constexpr bool DROP = decltype(dropped)::value;
      hipLaunchKernelGGL((gn_bwd_sums_kernel<DT, V, DROP>), dim3(grid), dim3(kBlock), 0, stream, x, ld_x, src, gamma, beta, save_mean,
                         save_rstd, p, act, d, per_group, per_channel_sums);
      hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, V, DROP>), dim3(second), dim3(kBlock), 0, stream, x, ld_x, src, gamma, beta,
                         save_mean, save_rstd, p, (int)B, act, d, per_group, per_channel_sums, params, gx, ggamma, gbeta);
    };
    if (threshold) both(std::true_type{});
    else both(std::false_type{});
  });
  return sfm_last_error();
}
