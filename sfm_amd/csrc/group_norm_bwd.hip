// Group norm with an activation: the backward (group_norm.h has the mathematics and the plan).
#include "group_norm.h"

namespace sfm {
namespace {

// dL/dy: the sum of up to three tensors, each a channel slice with its own row stride (what an activation's several readers
// hand back in a decoder level without concats)
struct GySrc {
  const void* p[3];
  long long ld[3];
  int n;
};
template <int DT, int V, int U>
__device__ __forceinline__ void add_more_gy(const GySrc& s, const GnPlan& p, const Where& w, const Lane& l, const Tile<U>& t, int u,
                                            float (&g)[V]) {
  for (int k = 1; k < s.n; ++k) {  // uniform
    const Stream<DT, V> more(s.p[k], s.ld[k], p, w, l);
    float f[V];
    unpack<DT, V>(more.row(more.at(t), t, u, l.ry), f);
#pragma unroll
    for (int e = 0; e < V; ++e) g[e] += f[e];
  }
}

// ---- backward, first launch: per_group [B][G][P] (sum gamma dz, sum gamma dz xhat), per_channel [C][B][chunks] (sum dz, sum dz xhat)
// Bound by memory: two tensors of 0.49 GB fp32 in 160 us, 6.1 TB/s; of 0.54 GB bf16 with silu in 202, 5.3 TB/s with the ALUs busy 62 % of it
// (a tile's loads are asked for when the one before is done; row by row as in the forward's last pass 194, but 180 in fp32 with a mask, which spills).
template <int DT, int V, int E, bool DROP>
__global__ __launch_bounds__(kBlock, bound_of(V / E, waves_sums(ElemBytes<DT>::value, V))) void gn_bwd_sums_kernel(const void* __restrict__ x, long long ldx, GySrc gy,
                                                             const float* __restrict__ gamma, const float* __restrict__ beta,
                                                             const float* __restrict__ mean, const float* __restrict__ rstd,
                                                             GnPlan p, int B, int act, Drop drop, float2* __restrict__ per_group,
                                                             float2* __restrict__ per_channel) {
  constexpr int A = V / E, U = batch_of(V * ElemBytes<DT>::value);
  __shared__ float2 red[kBlock * V];
  const Where w = where(p, blockIdx.x, blockIdx.y, blockIdx.z);
  const Lane l(p, w, p.row_lanes);
  if (l.mine) {
    const Stream<DT, V> xs(x, ldx, p, w, l), gs(gy.p[0], gy.ld[0], p, w, l);
    Tile<U> t(p, w.chunk);
    Raw<DT, V> xr[U], gr[U];
    xs.load(t, l.ry, xr);
    gs.load(t, l.ry, gr);
    const int c = w.c0 + l.vx * V;
    float mu[A], is[A], sc[V], sh[V], s1[V], s2[V];  // s2: of dz (x - mean), which r makes sums of dz xhat in the end
#pragma unroll
    for (int a = 0; a < A; ++a) {
      const long long g = (long long)w.b * p.G + w.g0 + group_in_slab(p, l.vx * V + a * E);
      mu[a] = mean[g]; is[a] = rstd[g];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) { sc[k] = gamma[c + k] * is[k / E]; sh[k] = beta[c + k]; s1[k] = 0.0f; s2[k] = 0.0f; }
    std::conditional_t<DROP, Mask<V>, NoMask> mask(drop, p, w, c);
    const unsigned long long place = (unsigned long long)l.ry * p.C + c, row_places = (unsigned long long)p.row_lanes * p.C;
    for (;;) {
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (u >= t.steps) break;
        float f[V], g[V], z[V];
        unpack<DT, V>(xr[u], f);
        unpack<DT, V>(gr[u], g);
        if (gy.n > 1) add_more_gy<DT, V, U>(gy, p, w, l, t, u, g);
        if constexpr (DROP) mask.apply(g, u, (unsigned long long)(t.index * U + u) * row_places + place, row_places);
        if (!t.full) {  // a row lane without a row has read another's: nothing of it is added (a branch of its own would keep both ways' registers)
          const bool counts = t.valid(u, l.ry);
#pragma unroll
          for (int k = 0; k < V; ++k) g[k] = counts ? g[k] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) { f[k] -= mu[k / E]; z[k] = __builtin_fmaf(f[k], sc[k], sh[k]); }
        act_bwd<V>(g, z, act);
#pragma unroll
        for (int k = 0; k < V; ++k) { s1[k] += g[k]; s2[k] = __builtin_fmaf(g[k], f[k], s2[k]); }
      }
      if (t.index + p.first.chunks >= p.tiles) break;
      t = Tile<U>(p, t.index + p.first.chunks);
      xs.load(t, l.ry, xr);
      gs.load(t, l.ry, gr);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) red[l.ry * p.cs + l.vx * V + k] = make_float2(s1[k], s2[k] * is[k / E]);
  }
  __syncthreads();
  // over the row lanes: S threads per channel take every S-th row lane each, then one adds the S.  In order: the same bits every time.
  const int S = max(1, kBlock / w.cc);
  const int cl = threadIdx.x % (unsigned)w.cc, seg = threadIdx.x / (unsigned)w.cc;
  for (int c = cl; seg < S && c < w.cc; c += kBlock) {  // (cc > kBlock: S = 1 and a thread has several channels)
    float a = 0.0f, b = 0.0f;
    for (int i = seg; i < p.row_lanes; i += S) { const float2 v = red[i * p.cs + c]; a += v.x; b += v.y; }
    if (seg < p.row_lanes) red[seg * p.cs + c] = make_float2(a, b);  // (only this thread reads or writes that place)
  }
  __syncthreads();
  const int left = min(S, p.row_lanes);
  for (int c = threadIdx.x; c < w.cc; c += kBlock) {
    float2 v = red[c];
    for (int i = 1; i < left; ++i) { const float2 o = red[i * p.cs + c]; v.x += o.x; v.y += o.y; }
    red[c] = v;
    per_channel[((long long)(w.c0 + c) * B + w.b) * p.first.chunks + w.chunk] = v;
  }
  __syncthreads();
  const Team tm = team_of(w.ng);
  const int cg = p.parts == 1 ? p.cpg : w.cc;
  for (int j = tm.id; j < w.ng; j += tm.count) {
    float a = 0.0f, b = 0.0f;
    for (int e = tm.lane; e < cg; e += tm.T) {
      const float2 v = red[j * cg + e];
      const float ga = gamma[w.c0 + j * cg + e];
      a = __builtin_fmaf(ga, v.x, a);
      b = __builtin_fmaf(ga, v.y, b);
    }
    a = team_sum(a, tm.T);
    b = team_sum(b, tm.T);
    if (tm.lane == 0) per_group[((long long)w.b * p.G + w.g0 + j) * p.P + w.chunk * p.parts + w.part] = make_float2(a, b);
  }
}

// ---- backward, second launch: the first param_blocks workgroups sum the channel partials over items and chunks (a wave per
// channel), the others write gx.  Bound by memory: two tensors of 0.54 GB bf16 read and one written in 270 us, 6.0 TB/s, where the pattern
// without arithmetic takes 263.
template <int DT, int V, int E, bool DROP, bool FAR>
__global__ __launch_bounds__(kBlock, bound_of(V / E, waves_bwd_apply(ElemBytes<DT>::value, V))) void gn_bwd_apply_kernel(const void* __restrict__ x, long long ldx, GySrc gy,
                                                              const float* __restrict__ gamma, const float* __restrict__ beta,
                                                              const float* __restrict__ mean, const float* __restrict__ rstd,
                                                              GnPlan p, int B, int act, Drop drop,
                                                              const float2* __restrict__ per_group,
                                                              const float2* __restrict__ per_channel, unsigned param_blocks,
                                                              void* __restrict__ gx, float* __restrict__ ggamma,
                                                              float* __restrict__ gbeta) {
  constexpr int A = V / E, U = batch_of(V * ElemBytes<DT>::value);
  __shared__ float2 stat[kBlock * A];
  if (blockIdx.x < param_blocks) {
    const int c = blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6), lane = threadIdx.x & 63;
    if (c >= p.C) return;
    const long long n = (long long)B * p.first.chunks;
    const float2* src = per_channel + c * n;
    double a = 0.0, b = 0.0;
    each_partial<8>(src, n, lane, 64, [&](int, float2 v) { a += v.x; b += v.y; });
    a = team_sum(a, 64);
    b = team_sum(b, 64);
    if (lane == 0) { gbeta[c] = (float)a; ggamma[c] = (float)b; }
    return;
  }
  const unsigned bid = blockIdx.x - param_blocks, rest = bid / (unsigned)B;  // (items, chunks, slabs) in one dimension
  const Where w = where(p, bid - rest * B, rest % (unsigned)p.last.chunks, rest / (unsigned)p.last.chunks);
  const Lane l(p, w, p.row_lanes);
  const Stream<DT, V, FAR> xs(x, ldx, p, w, l), gs(gy.p[0], gy.ld[0], p, w, l), os(gx, p.C, p, w, l);
  Tile<U> t(p, FAR ? w.chunk : last_tile(p, w));
  Raw<DT, V> xr[U], gr[U];
  const int c = w.c0 + l.vx * V;
  float mu[A], is[A], sc[V], sh[V], c1[A], c2[A];
  if (l.mine) {
    xs.load(t, l.ry, xr);
    gs.load(t, l.ry, gr);
#pragma unroll
    for (int a = 0; a < A; ++a) {
      const long long g = (long long)w.b * p.G + w.g0 + group_in_slab(p, l.vx * V + a * E);
      mu[a] = mean[g]; is[a] = rstd[g];
    }
#pragma unroll
    for (int k = 0; k < V; ++k) { sc[k] = gamma[c + k] * is[k / E]; sh[k] = beta[c + k]; }
  }
  {
    const Team tm = team_of(w.ng);
    const float inv = 1.0f / ((float)p.N * (float)p.cpg);
    for (int j = tm.id; j < w.ng; j += tm.count) {
      const float2* src = per_group + ((long long)w.b * p.G + w.g0 + j) * p.P;
      float a = 0.0f, b = 0.0f;
      each_partial<4>(src, p.P, tm.lane, tm.T, [&](int, float2 v) { a += v.x; b += v.y; });
      a = team_sum(a, tm.T);
      b = team_sum(b, tm.T);
      if (tm.lane == 0) stat[j] = make_float2(a * inv, b * inv);
    }
    __syncthreads();
  }
  if (!l.mine) return;
#pragma unroll
  for (int a = 0; a < A; ++a) {
    const float2 st = stat[group_in_slab(p, l.vx * V + a * E)];
    c1[a] = -st.x * is[a];  // gx = r gamma dz - r c1 - (x - mean) r^2 c2
    c2[a] = -st.y * is[a] * is[a];
  }
  std::conditional_t<DROP, Mask<V>, NoMask> mask(drop, p, w, c);
  const unsigned long long place = (unsigned long long)l.ry * p.C + c, row_places = (unsigned long long)p.row_lanes * p.C;
  for (;;) {
    const char* o = os.at(t);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (u >= t.steps) break;
      float f[V], g[V], z[V];
      unpack<DT, V>(xr[u], f);
      unpack<DT, V>(gr[u], g);
      if (gy.n > 1) add_more_gy<DT, V, U>(gy, p, w, l, t, u, g);
      if constexpr (DROP) mask.apply(g, u, (unsigned long long)(t.index * U + u) * row_places + place, row_places);
#pragma unroll
      for (int k = 0; k < V; ++k) { f[k] -= mu[k / E]; z[k] = __builtin_fmaf(f[k], sc[k], sh[k]); }
      act_bwd<V>(g, z, act);
#pragma unroll
      for (int k = 0; k < V; ++k) g[k] = __builtin_fmaf(f[k], c2[k / E], __builtin_fmaf(sc[k], g[k], c1[k / E]));
      if (t.valid(u, l.ry)) os.store(o, u, g);
    }
    if (FAR ? t.index + p.last.chunks >= p.tiles : t.index < p.last.chunks) break;
    t = Tile<U>(p, FAR ? t.index + p.last.chunks : t.index - p.last.chunks);
    xs.load(t, l.ry, xr);
    gs.load(t, l.ry, gr);
  }
}

}  // namespace
}  // namespace sfm

using namespace sfm;

extern "C" int sfm_group_norm_act_bwd(const void* x, long long ld_x, int dtype, const void* const* gy, const long long* ld_gy,
                                      int n_gy, const float* gamma, const float* beta, const float* save_mean,
                                      const float* save_rstd, long long B, long long N, int C, int G, int act, const void* rng,
                                      unsigned long long seed, unsigned step, unsigned layer, unsigned item0, int threshold,
                                      int per_channel, void* gx, float* ggamma, float* gbeta, float* ws, void* stream_) {
  GnPlan p;
  Drop d;
  dim3 first, last;
  const int es = dtype == kF32 ? 4 : 2;
  if (!gy || !ld_gy || n_gy < 1 || n_gy > 3) return SFM_ERR_ARG;
  long long ld = ld_x;
  for (int k = 0; k < n_gy; ++k) ld = std::max(ld, ld_gy[k]);
  const int rc = gn_setup(B, N, C, G, dtype, ld, true, p, first, last);
  if (rc) return rc;
  if (!rows_ok(x, ld_x, C, es) || !gamma || !beta || !save_mean || !save_rstd ||
      (!gx && !ggamma) || (gx && !rows_ok(gx, C, C, es)) || (!ggamma != !gbeta) || !ws || ((uintptr_t)ws & 7) || act < kActNone ||
      act > kActSilu || !drop_args(rng, seed, step, layer, item0, threshold, per_channel, d))
    return SFM_ERR_ARG;
  if (threshold && ((__int128)N * C > ((__int128)1 << 35) || B > (1ll << 32) - item0)) return SFM_ERR_TOO_LARGE;
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
  // a multiple of eight: the workgroups behind them stay on the XCDs they were on in the first launch
  const unsigned params = ggamma ? ((unsigned)(C + kBlock / 64 - 1) / (kBlock / 64) + 7u) / 8u * 8u : 0u;
  const unsigned second = params + (gx ? last.x * last.y * last.z : 0u);
  by_type(dtype, p, [&](auto dt, auto v, auto e) {
    constexpr int DT = decltype(dt)::value, V = decltype(v)::value;
    constexpr int E = decltype(e)::value;
    by_use<DT, V>(threshold != 0, far(3 * B * N * C * es), [&](auto drop, auto away) {
      constexpr bool DROP = decltype(drop)::value;
      hipLaunchKernelGGL((gn_bwd_sums_kernel<DT, V, E, DROP>), first, dim3(kBlock), 0, stream, x, ld_x, src, gamma, beta, save_mean,
                         save_rstd, p, (int)B, act, d, per_group, per_channel_sums);
      hipLaunchKernelGGL((gn_bwd_apply_kernel<DT, V, E, DROP, decltype(away)::value>), dim3(second), dim3(kBlock), 0, stream, x, ld_x, src, gamma, beta,
                         save_mean, save_rstd, p, (int)B, act, d, per_group, per_channel_sums, params, gx, ggamma, gbeta);
    });
  });
  return sfm_last_error();
}
