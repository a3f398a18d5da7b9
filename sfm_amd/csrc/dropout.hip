// Dropout whose mask is a function of counters and never stored: y = keep ? x * scale : 0, and the same on dL/dy for the
// backward (norm_drop.h has the generator).  Bound by memory: one read and one write per element.
#include "norm_drop.h"

namespace sfm {
namespace {

constexpr int kPer = 4;  // blocks of eight elements a thread draws for; a workgroup takes kPer * kBlock consecutive ones

// the eight keep bits of block `blk` of an item
__device__ __forceinline__ unsigned keep_eight(const Drop& d, const DropKey& key, unsigned item, unsigned blk, unsigned C) {
  if (!d.per_channel) return keep_bits(d, key, d.item0 + item, (unsigned long long)blk * 8);
  if (C % 8 == 0) return keep_bits(d, key, d.item0 + item, blk % (C / 8) * 8);
  unsigned c = (unsigned)((unsigned long long)blk * 8 % C), keep = 0;  // they start anywhere in a row and cross into the next
  if (C >= 8) {  // the rest of a block, the next one (or the row's first), and where the row ends with a short block one more
    unsigned n = min(8 - (c & 7), C - c);
    keep = (keep_bits(d, key, d.item0 + item, c) >> (c & 7)) & ((1u << n) - 1);
    c = c + n == C ? 0 : c + n;
    const unsigned more = min(8u, C - c);
    keep |= (keep_bits(d, key, d.item0 + item, c) & ((1u << more) - 1)) << n;
    n += more;
    if (n < 8) keep |= keep_bits(d, key, d.item0 + item, c + more == C ? 0 : c + more) << n;
  } else {
    const unsigned all = keep_bits(d, key, d.item0 + item, 0);
    for (int e = 0; e < 8; ++e) {
      keep |= ((all >> c) & 1u) << e;
      c = c + 1 == C ? 0 : c + 1;
    }
  }
  return keep;
}

// Items of whole blocks (item_elems a multiple of eight): the tensor is one run of blocks.  A lane draws for the block of its number;
// 16-bit: that is the 16 bytes it loads.  fp32: a block is 32 bytes, and a lane that loaded both halves would touch every line twice
// (450 us for 2 x 1 GiB, nontemporal): a wave loads its 64 blocks as two runs of 16 bytes a lane, and a lane takes the bits
// of its half from the lane that drew them.
template <int DT, bool FAR>
__global__ __launch_bounds__(kBlock) void dropout_blocks_kernel(const char* __restrict__ x, char* __restrict__ y,
                                                                unsigned long long total, unsigned blocks, unsigned C, Drop d) {
  constexpr int V = DT == kF32 ? 4 : 8, R = 8 / V;
  const int lane = threadIdx.x & 63;
  const unsigned long long q0 = (unsigned long long)blockIdx.x * (kPer * kBlock);
  const unsigned item0 = (unsigned)(q0 / blocks), off0 = (unsigned)(q0 % blocks);  // uniform
  const unsigned left = (unsigned)min((unsigned long long)(kPer * kBlock), total - q0);
  const char* xs = x + q0 * (8 * ElemBytes<DT>::value);
  char* ys = y + q0 * (8 * ElemBytes<DT>::value);
  Raw<DT, V> raw[kPer][R];
#pragma unroll
  for (int k = 0; k < kPer; ++k)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned first = k * kBlock + (threadIdx.x & ~63u) + r * (64 / R);  // block of lane 0
      if (first + lane / R < left) raw[k][r] = load_raw<DT, V, FAR>(xs, (first * 8 + lane * V) * (unsigned)ElemBytes<DT>::value);
    }
  const DropKey key = drop_key(d);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const unsigned long long off = (unsigned long long)off0 + k * kBlock + threadIdx.x;
    const unsigned up = off < blocks ? 0u : (unsigned)(off / blocks);
    const unsigned keep = keep_eight(d, key, item0 + up, (unsigned)(off - (unsigned long long)up * blocks), C);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const unsigned bits = R == 1 ? keep : __shfl(keep, r * (64 / R) + lane / R, 64) >> (lane % R * V);
      const unsigned first = k * kBlock + (threadIdx.x & ~63u) + r * (64 / R);
      if (first + lane / R >= left) continue;
      float f[V];
      unpack<DT, V>(raw[k][r], f);
      keep_apply<V>(f, bits, d.scale);
      store_vec<DT, V, FAR>(ys, (first * 8 + lane * V) * (unsigned)ElemBytes<DT>::value, f);
    }
  }
}

// any item size: a thread takes whole blocks, which start anywhere in memory, and the last of an item may be short
template <int DT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const char* __restrict__ x, char* __restrict__ y, unsigned items,
                                                         unsigned long long n, unsigned blocks, unsigned C, Drop d) {
  constexpr int kBytes = ElemBytes<DT>::value;
  const DropKey key = drop_key(d);
  const unsigned long long q0 = (unsigned long long)blockIdx.x * (kPer * kBlock);
  const unsigned item0 = (unsigned)(q0 / blocks), off0 = (unsigned)(q0 % blocks);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const unsigned long long off = (unsigned long long)off0 + k * kBlock + threadIdx.x;
    const unsigned up = off < blocks ? 0u : (unsigned)(off / blocks);
    const unsigned item = item0 + up, blk = (unsigned)(off - (unsigned long long)up * blocks);
    if (item >= items) continue;
    const unsigned long long first = (unsigned long long)blk * 8;
    const long long at = (long long)(item * n + first) * kBytes;
    const unsigned keep = keep_eight(d, key, item, blk, C);
    if (first + 8 <= n) {
      float f[8];
      unpack<DT, 8>(load_raw<DT, 8>(x, at), f);
      keep_apply<8>(f, keep, d.scale);
      store_vec<DT, 8>(y, at, f);
    } else {
      for (unsigned e = 0; first + e < n; ++e) {
        float f[1];
        unpack<DT, 1>(load_raw<DT, 1>(x, at + e * kBytes), f);
        keep_apply<1>(f, keep >> e, d.scale);
        store_vec<DT, 1>(y, at + e * kBytes, f);
      }
    }
  }
}

}  // namespace
}  // namespace sfm

using namespace sfm;

extern "C" int sfm_dropout(const void* x, int dtype, long long items, long long item_elems, int C, const void* rng,
                           unsigned long long seed, unsigned step, unsigned layer, unsigned item0, int threshold,
                           int per_channel, void* y, void* stream_) {
  Drop d;
  if (!x || !y || dtype < kF32 || dtype > kF16 || items < 1 || item_elems < 1 || C < 1 || item_elems % C ||
      !drop_args(rng, seed, step, layer, item0, threshold, per_channel, d))
    return SFM_ERR_ARG;
  const int es = dtype == kF32 ? 4 : 2;
  if (((uintptr_t)x | (uintptr_t)y) & (es - 1)) return SFM_ERR_ARG;
  const long long blocks = item_elems / 8 + (item_elems % 8 != 0);
  // counters of 32 bits each; the grid's limit
  if (items > 0xffffffffll - item0 || blocks > 0xffffffffll || (__int128)items * item_elems > ((__int128)1 << 60))
    return SFM_ERR_TOO_LARGE;
  const long long groups = (items * blocks + kPer * kBlock - 1) / (kPer * kBlock);
  if (groups > kMaxGrid) return SFM_ERR_TOO_LARGE;
  const bool whole = item_elems % 8 == 0, away = far(2 * items * item_elems * es);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const char* xs = static_cast<const char*>(x);
    char* ys = static_cast<char*>(y);
    hipStream_t stream = (hipStream_t)stream_;
    const dim3 grid((unsigned)groups), block(kBlock);
    if (whole && away)
      hipLaunchKernelGGL((dropout_blocks_kernel<DT, true>), grid, block, 0, stream, xs, ys, (unsigned long long)(items * blocks),
                         (unsigned)blocks, (unsigned)C, d);
    else if (whole)
      hipLaunchKernelGGL((dropout_blocks_kernel<DT, false>), grid, block, 0, stream, xs, ys, (unsigned long long)(items * blocks),
                         (unsigned)blocks, (unsigned)C, d);
    else
      hipLaunchKernelGGL(dropout_kernel<DT>, grid, block, 0, stream, xs, ys, (unsigned)items, (unsigned long long)item_elems,
                         (unsigned)blocks, (unsigned)C, d);
  };
  if (dtype == kF32) launch(std::integral_constant<int, kF32>{});
  else if (dtype == kBF16) launch(std::integral_constant<int, kBF16>{});
  else launch(std::integral_constant<int, kF16>{});
  return sfm_last_error();
}
