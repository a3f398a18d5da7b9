// Group norm with an activation: the forward (group_norm.h has the mathematics and the plan).
#include "group_norm.h"

namespace sfm {
namespace {

// (mean, M2) of the groups of a workgroup from those of its threads: red [row lane][vector][A], a pair for each E adjacent channels of
// a vector.  Every row lane has seen per_lane rows, the first `more` one more.  cg: channels of a group in the slab.  Means are
// taken against one of them, so a common part costs no digits.  out(j, mean, M2) by one thread per group.
template <int T, int A, int E, typename F>
__device__ __forceinline__ void reduce_stats(const float2* red, int lanes, int row_lanes, int per_lane, int more, int cg, int ng, F&& out) {
  const Team tm = team_of<T>(ng);
  const int per_row = cg / E, busy = per_lane > 0 ? row_lanes : more;
  const float per_row_inv = __builtin_amdgcn_rcpf((float)per_row);
  const float rows = (float)per_lane, inv = 1.0f / ((rows * row_lanes + more) * per_row);
  for (int j = tm.id; j < ng; j += tm.count) {
    const float ref = red[j * per_row].x;
    float s = 0.0f;
    for (int e = tm.lane; e < busy * per_row; e += tm.T) {
      const int row = (int)(((float)e + 0.5f) * per_row_inv), c = e - row * per_row;  // e / per_row: e < 2^13, 0.5 / per_row covers the rounding
      s = __builtin_fmaf(rows + (row < more), red[row * lanes * A + j * per_row + c].x - ref, s);
    }
    const float off = team_sum(s, tm.T) * inv;
    float q = 0.0f;
    for (int e = tm.lane; e < busy * per_row; e += tm.T) {
      const int row = (int)(((float)e + 0.5f) * per_row_inv), c = e - row * per_row;  // e / per_row: e < 2^13, 0.5 / per_row covers the rounding
      const float2 v = red[row * lanes * A + j * per_row + c];
      const float d = (v.x - ref) - off;
      q += __builtin_fmaf(E * (rows + (row < more)) * d, d, v.y);
    }
    q = team_sum(q, tm.T);
    if (tm.lane == 0) out(j, ref + off, q);
  }
}

// ---- forward, first launch: part [B][G][P] (mean, M2).  A thread has one pair for E adjacent channels of a group.
// Bound by memory: 4x1024x2048x32 bf16 (0.54 GB) 86 us, 6.2 TB/s, what plain loads of this card's memory give.
template <int DT, int V, int E>
__global__ __launch_bounds__(kBlock, bound_of(V / E, waves_stats(ElemBytes<DT>::value, V))) void gn_stats_kernel(const void* __restrict__ x, long long ldx, GnPlan p,
                                                          float2* __restrict__ part) {
  constexpr int A = V / E, U = batch_of(V * ElemBytes<DT>::value); // accumulators
  __shared__ float2 red[kBlock * A];         // [row lane][E channels of the slab]
  const Where w = where(p, blockIdx.x, blockIdx.y, blockIdx.z);
  const Lane l(p, w, p.row_lanes);
  if (l.mine) {
    const Stream<DT, V> xs(x, ldx, p, w, l);
    float n = 0.0f, mean[A], m2[A];
#pragma unroll
    for (int a = 0; a < A; ++a) { mean[a] = 0.0f; m2[a] = 0.0f; }
    // a batch of R rows: its mean, its squared deviations from that, joined to (n, mean, m2)
    auto join = [&](auto rows, const Raw<DT, V>* raw) {
      constexpr int R = decltype(rows)::value;
      float s[A], q[A];
#pragma unroll
      for (int a = 0; a < A; ++a) { s[a] = 0.0f; q[a] = 0.0f; }
#pragma unroll
      for (int u = 0; u < R; ++u) {
        float f[V];
        unpack<DT, V>(raw[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) s[k / E] += f[k];
      }
#pragma unroll
      for (int a = 0; a < A; ++a) s[a] *= 1.0f / (R * E);
#pragma unroll
      for (int u = 0; u < R; ++u) {
        float f[V];
        unpack<DT, V>(raw[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) { const float d = f[k] - s[k / E]; q[k / E] = __builtin_fmaf(d, d, q[k / E]); }
      }
      const float nn = n + R * E, share = (R * E) / nn, cross = n * share;
#pragma unroll
      for (int a = 0; a < A; ++a) {
        const float delta = s[a] - mean[a];
        mean[a] = __builtin_fmaf(delta, share, mean[a]);
        m2[a] += __builtin_fmaf(delta * delta, cross, q[a]);
      }
      n = nn;
    };
    for (long long i = w.chunk; i < p.tiles; i += p.first.chunks) {
      const Tile<U> t(p, i);
      Raw<DT, V> raw[U];
      xs.load(t, l.ry, raw);
      if (t.full) join(std::integral_constant<int, U>{}, raw);
      else {
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (t.valid(u, l.ry)) join(std::integral_constant<int, 1>{}, raw + u);
      }
    }
#pragma unroll
    for (int a = 0; a < A; ++a) red[(l.ry * p.lanes + l.vx) * A + a] = make_float2(mean[a], m2[a]);
  }
  __syncthreads();
  const bool partial = w.chunk == p.first.owner && p.left < p.tile_rows;
  const long long whole = p.first.own + (w.chunk < p.first.extra) - partial;   // whole tiles of this chunk
  const int per_lane = (int)whole * U + (partial ? p.left / p.row_lanes : 0), more = partial ? p.left % p.row_lanes : 0;
  reduce_stats<kBlock, A, E>(red, p.lanes, p.row_lanes, per_lane, more, p.parts == 1 ? p.cpg : w.cc, w.ng, [&](int j, float mean, float m2) {
    part[((long long)w.b * p.G + w.g0 + j) * p.P + w.chunk * p.parts + w.part] = make_float2(mean, m2);
  });
}

__device__ __forceinline__ float rsqrt_of(float var, float eps) { return 1.0f / sqrtf(var + eps); }

// joins the partials of a workgroup's groups: stat[j] = (mean, r) in LDS.  All threads call it; it ends with a barrier.  In fp32, a
// lane adds few of them, and with the means taken against one of them; fp64 in one pass over them took 1.2 us more of a small pass.
// K: loads on their way at a time, what the registers allow beside the batch of x that is on its way as well.
template <int K> __device__ __forceinline__ void join_stats(const float2* __restrict__ part, const GnPlan& p, const Where& w, float eps,
                                           float2* __restrict__ stat) {
  const Team t = team_of(w.ng);
  const float inv = 1.0f / ((float)p.N * (float)p.cpg);
  for (int j = t.id; j < w.ng; j += t.count) {
    const float2* src = part + ((long long)w.b * p.G + w.g0 + j) * p.P;
    const float ref = src[0].x;
    float s = 0.0f, q2 = 0.0f, off;
    if (p.parts == 1) {
      const float more = p.first.rows_more * p.cpg, rows = p.first.rows * p.cpg, less = (float)(p.tile_rows - p.left) * p.cpg;
      auto count = [&](int q) { return (q < p.first.extra ? more : rows) - (q == p.first.owner ? less : 0.0f); };
      float2 v[K];  // the first K of the lane are loaded once
#pragma unroll
      for (int k = 0; k < K; ++k) v[k] = src[min(t.lane + k * t.T, p.P - 1)];
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int q = t.lane + k * t.T;
        v[k].x -= ref;
        if (q < p.P) s = __builtin_fmaf(count(q), v[k].x, s);
      }
      each_partial<K>(src, p.P, t.lane + K * t.T, t.T, [&](int q, float2 u) { s = __builtin_fmaf(count(q), u.x - ref, s); });
      off = team_sum(s, t.T) * inv;
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const int q = t.lane + k * t.T;
        const float d = v[k].x - off;
        if (q < p.P) q2 += __builtin_fmaf(count(q) * d, d, v[k].y);
      }
      each_partial<K>(src, p.P, t.lane + K * t.T, t.T, [&](int q, float2 u) {
        const float d = (u.x - ref) - off;
        q2 += __builtin_fmaf(count(q) * d, d, u.y);
      });
    } else {
      for (int q = t.lane; q < p.P; q += t.T) s = __builtin_fmaf(part_count(p, q), src[q].x - ref, s);
      off = team_sum(s, t.T) * inv;
      for (int q = t.lane; q < p.P; q += t.T) {
        const float2 u = src[q];
        const float d = (u.x - ref) - off;
        q2 += __builtin_fmaf(part_count(p, q) * d, d, u.y);
      }
    }
    q2 = team_sum(q2, t.T);
    if (t.lane == 0) stat[j] = make_float2(ref + off, rsqrt_of(q2 * inv, eps));
  }
  __syncthreads();
}

// ---- forward, second launch.  The first batch is on its way while the partials are joined; where a cache may still hold what the
// first launch read last, the tiles go backwards (last_tile).  Bound by memory: 0.54 GB bf16 read and written in 177 us, 6.1 TB/s, where a
// plain copy in the same pattern takes 175; 54 MB fp32 in 19 us, where the launch and the joining are 6 of them.
template <int DT, int V, int E, bool DROP, bool FAR>
__global__ __launch_bounds__(kBlock, bound_of(V / E, waves_apply(ElemBytes<DT>::value, V))) void gn_apply_kernel(const void* __restrict__ x, long long ldx,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta,
                                                          const float2* __restrict__ part, GnPlan p, float eps, int act, Drop drop,
                                                          void* __restrict__ y, long long ldy, float* __restrict__ save_mean,
                                                          float* __restrict__ save_r) {
  constexpr int A = V / E, U = batch_of(V * ElemBytes<DT>::value);
  __shared__ float2 stat[kBlock * A];
  const Where w = where(p, blockIdx.x, blockIdx.y, blockIdx.z);
  const Lane l(p, w, p.row_lanes);
  const Stream<DT, V, FAR> xs(x, ldx, p, w, l), ys(y, ldy, p, w, l);
  Tile<U> t(p, FAR ? w.chunk : last_tile(p, w));
  Raw<DT, V> raw[U];
  float sc[V], sh[V];
  const int c = w.c0 + l.vx * V;
  if (l.mine) {
    xs.load(t, l.ry, raw);
#pragma unroll
    for (int k = 0; k < V; ++k) { sc[k] = gamma[c + k]; sh[k] = beta[c + k]; }
  }
  join_stats<V == 8 ? 4 : 2>(part, p, w, eps, stat);
  if (save_mean && w.chunk == 0 && w.part == 0)
    for (int j = threadIdx.x; j < w.ng; j += kBlock) {
      save_mean[(long long)w.b * p.G + w.g0 + j] = stat[j].x;
      save_r[(long long)w.b * p.G + w.g0 + j] = stat[j].y;
    }
  if (!l.mine) return;
  float mu[A];
#pragma unroll
  for (int a = 0; a < A; ++a) {
    const float2 st = stat[group_in_slab(p, l.vx * V + a * E)];
    mu[a] = st.x;
#pragma unroll
    for (int k = a * E; k < (a + 1) * E; ++k) sc[k] *= st.y;
  }
  std::conditional_t<DROP, Mask<V>, NoMask> mask(drop, p, w, c);
  const unsigned long long place = (unsigned long long)l.ry * p.C + c, row_places = (unsigned long long)p.row_lanes * p.C;
  for (;;) {
    const bool more = FAR ? t.index + p.last.chunks < p.tiles : t.index >= p.last.chunks;
    const Tile<U> next(p, !more ? t.index : FAR ? t.index + p.last.chunks : t.index - p.last.chunks);
    const char *a = xs.at(next), *o = ys.at(t);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= t.steps) break;
      float f[V];
      unpack<DT, V>(raw[u], f);
      if (more && u < next.steps) raw[u] = xs.row(a, next, u, l.ry);  // as a row has been used, the next tile's is asked for
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = __builtin_fmaf(f[k] - mu[k / E], sc[k], sh[k]);
      act_fwd<DT, V>(f, act);
      if constexpr (DROP) mask.apply(f, u, (unsigned long long)(t.index * U + u) * row_places + place, row_places);
      if (t.valid(u, l.ry)) ys.store(o, u, f);
    }
    if (!FAR && more && t.steps < U) {  // the item's last tile comes first where tiles go backwards; the next one has rows that it had not
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u >= t.steps && u < next.steps) raw[u] = xs.row(a, next, u, l.ry);
    }
    if (!more) break;
    t = next;
  }
}

// ---- forward in one launch, for an item whose slab fits a workgroup's registers: a thread keeps up to kHeld vectors, the statistics
// are the workgroup's own, x is read once.  The row lanes are T / lanes, whatever the plan of the two-launch form says.
// Bound by latency: 8x208 rows of 512 fp32 6.5 us, 3.6 of them a launch's; in two launches 11.
constexpr int kHeld = 4;

template <int DT, int V, int E, bool DROP, int T>
__global__ __launch_bounds__(T) void gn_held_kernel(const void* __restrict__ x, long long ldx, const float* __restrict__ gamma,
                                                    const float* __restrict__ beta, GnPlan p, float eps, int act, Drop drop,
                                                    void* __restrict__ y, long long ldy, float* __restrict__ save_mean,
                                                    float* __restrict__ save_r) {
  constexpr int A = V / E, kES = ElemBytes<DT>::value;
  __shared__ float2 red[T * A], stat[T * A];
  const Where w = where(p, blockIdx.x, 0, blockIdx.y);
  const int N = (int)p.N, row_lanes = T / p.lanes;
  const Lane l(p, w, row_lanes);
  const int per_lane = N / row_lanes, more = N % row_lanes;
  const int rows = l.mine ? per_lane + (l.ry < more) : 0;  // of this thread
  const int c = w.c0 + l.vx * V;
  const char* xs = static_cast<const char*>(x) + ((long long)w.b * N * ldx + c) * kES + l.ry * ldx * kES;
  Raw<DT, V> raw[kHeld];
#pragma unroll
  for (int u = 0; u < kHeld; ++u)
    if (u < rows) raw[u] = load_raw<DT, V>(xs, (long long)u * row_lanes * ldx * kES);
  float sc[V], sh[V];
  if (l.mine) {
#pragma unroll
    for (int k = 0; k < V; ++k) { sc[k] = gamma[c + k]; sh[k] = beta[c + k]; }
    float s[A], q[A];
#pragma unroll
    for (int a = 0; a < A; ++a) { s[a] = 0.0f; q[a] = 0.0f; }
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (u < rows) {
        float f[V];
        unpack<DT, V>(raw[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) s[k / E] += f[k];
      }
    const float share = rows ? 1.0f / (float)(rows * E) : 0.0f;
#pragma unroll
    for (int a = 0; a < A; ++a) s[a] *= share;
#pragma unroll
    for (int u = 0; u < kHeld; ++u)
      if (u < rows) {
        float f[V];
        unpack<DT, V>(raw[u], f);
#pragma unroll
        for (int k = 0; k < V; ++k) { const float d = f[k] - s[k / E]; q[k / E] = __builtin_fmaf(d, d, q[k / E]); }
      }
#pragma unroll
    for (int a = 0; a < A; ++a) red[(l.ry * p.lanes + l.vx) * A + a] = make_float2(s[a], q[a]);
  }
  __syncthreads();
  const float inv = 1.0f / ((float)N * (float)p.cpg);
  reduce_stats<T, A, E>(red, p.lanes, row_lanes, per_lane, more, p.cpg, w.ng, [&](int j, float mean, float m2) {
    const float r = rsqrt_of(m2 * inv, eps);
    stat[j] = make_float2(mean, r);
    if (save_mean) {
      save_mean[(long long)w.b * p.G + w.g0 + j] = mean;
      save_r[(long long)w.b * p.G + w.g0 + j] = r;
    }
  });
  __syncthreads();
  if (!l.mine) return;
  float mu[A];
#pragma unroll
  for (int a = 0; a < A; ++a) {
    const float2 st = stat[group_in_slab(p, l.vx * V + a * E)];
    mu[a] = st.x;
#pragma unroll
    for (int k = a * E; k < (a + 1) * E; ++k) sc[k] *= st.y;
  }
  std::conditional_t<DROP, Mask<V>, NoMask> mask(drop, p, w, c);
  char* ys = static_cast<char*>(y) + ((long long)w.b * N * ldy + c) * kES + l.ry * ldy * kES;
#pragma unroll
  for (int u = 0; u < kHeld; ++u) {
    if (u < rows) {
      float f[V];
      unpack<DT, V>(raw[u], f);
#pragma unroll
      for (int k = 0; k < V; ++k) f[k] = __builtin_fmaf(f[k] - mu[k / E], sc[k], sh[k]);
      act_fwd<DT, V>(f, act);
      if constexpr (DROP) mask.apply(f, u, (unsigned long long)(u * row_lanes + l.ry) * p.C + c, (unsigned long long)row_lanes * p.C);
      store_vec<DT, V>(ys, (long long)u * row_lanes * ldy * kES, f);
    }
  }
}

// threads of the one-launch form, or 0 where an item's slab does not fit it
static int held_threads(const GnPlan& p, int es) {
  if (p.parts != 1 || p.V * es != 16) return 0;
  for (int T : {256, 1024})
    if (p.N <= (long long)kHeld * (T / p.lanes)) return T;
  return 0;
}

}  // namespace
}  // namespace sfm

using namespace sfm;

extern "C" long long sfm_group_norm_workspace_floats(long long B, long long N, int C, int G, int dtype, int backward) {
  GnPlan p;
  dim3 first, last;
  const int rc = gn_setup(B, N, C, G, dtype, C, backward != 0, p, first, last);
  if (rc) return rc;
  return 2 * (B * G * p.P + (backward ? B * C * p.first.chunks : 0));
}

extern "C" int sfm_group_norm_act_fwd(const void* x, long long ld_x, int dtype, const float* gamma, const float* beta, long long B,
                                      long long N, int C, int G, float eps, int act, const void* rng, unsigned long long seed,
                                      unsigned step, unsigned layer, unsigned item0, int threshold, int per_channel, void* y,
                                      long long ld_y, float* save_mean, float* save_rstd, float* ws, void* stream_) {
  GnPlan p;
  Drop d;
  dim3 first, last;
  const int es = dtype == kF32 ? 4 : 2;
  const int rc = gn_setup(B, N, C, G, dtype, std::max(ld_x, ld_y), false, p, first, last);
  if (rc) return rc;
  if (!rows_ok(x, ld_x, C, es) || !rows_ok(y, ld_y, C, es) || !gamma || !beta || !ws || ((uintptr_t)ws & 7) || !(eps > 0.0f) ||
      act < kActNone || act > kActSilu || (!save_mean != !save_rstd) ||
      !drop_args(rng, seed, step, layer, item0, threshold, per_channel, d))
    return SFM_ERR_ARG;
  if (threshold && ((__int128)N * C > ((__int128)1 << 35) || B > (1ll << 32) - item0)) return SFM_ERR_TOO_LARGE;
  hipStream_t stream = (hipStream_t)stream_;
  float2* part = reinterpret_cast<float2*>(ws);
  const int held = held_threads(p, es);
  by_type(dtype, p, [&](auto dt, auto v, auto e) {
    constexpr int DT = decltype(dt)::value, V = decltype(v)::value;
    constexpr int E = decltype(e)::value;
    if constexpr (V * ElemBytes<DT>::value == 16) {
      auto one = [&](auto threads, auto drop) {
        constexpr int T = decltype(threads)::value;
        hipLaunchKernelGGL((gn_held_kernel<DT, V, E, decltype(drop)::value, T>), dim3((unsigned)B, p.slabs), dim3(T), 0, stream, x, ld_x, gamma, beta, p,
                           eps, act, d, y, ld_y, save_mean, save_rstd);
      };
      auto with = [&](auto threads) { threshold ? one(threads, std::true_type{}) : one(threads, std::false_type{}); };
      if (held == 256) return with(std::integral_constant<int, 256>{});
      if (held == 1024) return with(std::integral_constant<int, 1024>{});
    }
    by_use<DT, V>(threshold != 0, far(2 * B * N * C * es), [&](auto drop, auto away) {
      hipLaunchKernelGGL((gn_stats_kernel<DT, V, E>), first, dim3(kBlock), 0, stream, x, ld_x, p, part);
      hipLaunchKernelGGL((gn_apply_kernel<DT, V, E, decltype(drop)::value, decltype(away)::value>), last, dim3(kBlock), 0, stream,
                         x, ld_x, gamma, beta, part, p, eps, act, d, y, ld_y, save_mean, save_rstd);
    });
  });
  return sfm_last_error();
}
