// Dropout whose mask is a function of counters and never stored: y = keep ? x * scale : 0, and the same on dL/dy for the
// backward (norm_drop.h has the generator).  Bound by memory: one read and one write per element; 1 GiB fp32 345 us,
// 6.2 TB/s, what a copy reaches; 27 MB bf16 9.8 us, 5.6 TB/s, where the generator is about as long as the copy.
#include "norm_drop.h"

namespace sfm {
namespace {

// Blocks of eight elements are counted through all items in 32 bits; a workgroup takes kBlock of them.  (More of them a thread were slower: one,
// two, four a thread 10.6, 10.6, 11.5 us for 27 MB bf16, 3.5, 3.9, 4.7 for 3.4 MB fp32, 342, 355, 350 for 1 GiB fp32.)
// Which of them this workgroup begins with, and the item and block of this thread:
struct Place { unsigned first, item, blk; };
__device__ __forceinline__ Place place_of(unsigned group, unsigned blocks) {
  Place o;
  o.first = group * kBlock;
  const unsigned item0 = o.first / blocks, off = o.first - item0 * blocks + threadIdx.x;  // (the host keeps the sum within 32 bits)
  const unsigned up = blocks >= kBlock ? off >= blocks : off / blocks;
  o.item = item0 + up;
  o.blk = off - up * blocks;
  return o;
}

// the eight keep bits of block `blk` of an item (whole channels of a width that eight does not divide take two or three draws: 38 MB bf16 of 45
// channels 23 us, 17 with one number per element; the same time for 77 MB fp32 of 45 and for 199 channels)
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
__global__ __launch_bounds__(kBlock) void dropout_blocks_kernel(const char* __restrict__ x, char* __restrict__ y, unsigned total,
                                                                unsigned groups, unsigned blocks, unsigned C, Drop d) {
  constexpr int kBytes = ElemBytes<DT>::value, V = DT == kF32 ? 4 : 8, R = 8 / V;
  const unsigned group = blockIdx.y * gridDim.x + blockIdx.x;
  if (group >= groups) return;
  const int lane = threadIdx.x & 63;
  const Place at = place_of(group, blocks);
  const unsigned left = total - at.first;
  const char* xs = x + (unsigned long long)at.first * (8 * kBytes);
  char* ys = y + (unsigned long long)at.first * (8 * kBytes);
  Raw<DT, V> raw[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned first = (threadIdx.x & ~63u) + r * (64 / R);  // block of lane 0
    if (first + lane / R < left) raw[r] = load_raw<DT, V, FAR>(xs, (first * 8 + lane * V) * kBytes);
  }
  const DropKey key = drop_key(d);
  if constexpr (R == 1) {
    if (!d.per_channel || C % 8 == 0) {  // a lane's eight elements are of one block of the mask: its numbers as they are, no bits of them
      const Draw<8> now = draw<8>(d, key, d.item0 + at.item, (unsigned long long)(d.per_channel ? at.blk % (C / 8) : at.blk) * 8);
      if (threadIdx.x >= left) return;
      float f[8];
      unpack<DT, 8>(raw[0], f);
      drop_apply<8>(f, now, d);
      store_vec<DT, 8, FAR>(ys, threadIdx.x * 8 * kBytes, f);
      return;
    }
  }
  const unsigned keep = keep_eight(d, key, at.item, at.blk, C);
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const unsigned bits = R == 1 ? keep : __shfl(keep, r * (64 / R) + lane / R, 64) >> (lane % R * V);
    const unsigned first = (threadIdx.x & ~63u) + r * (64 / R);
    if (first + lane / R >= left) continue;
    float f[V];
    unpack<DT, V>(raw[r], f);
    keep_apply<V>(f, bits, d.scale);
    store_vec<DT, V, FAR>(ys, (first * 8 + lane * V) * kBytes, f);
  }
}

// any item size: blocks start anywhere in memory, and the last of an item may be short
template <int DT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const char* __restrict__ x, char* __restrict__ y, unsigned items, unsigned groups,
                                                         unsigned long long n, unsigned blocks, unsigned C, Drop d) {
  constexpr int kBytes = ElemBytes<DT>::value;
  const unsigned group = blockIdx.y * gridDim.x + blockIdx.x;
  if (group >= groups) return;
  const Place p = place_of(group, blocks);
  if (p.item >= items) return;
  const unsigned long long first = (unsigned long long)p.blk * 8;
  const long long at = (long long)(p.item * n + first) * kBytes;
  const unsigned keep = keep_eight(d, drop_key(d), p.item, p.blk, C);
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
  // items and blocks are counted in 32 bits, up to a workgroup past the last
  if (items > (1ll << 32) - item0 || (__int128)items * blocks > 0xffffffffll - kBlock) return SFM_ERR_TOO_LARGE;
  const unsigned total = (unsigned)(items * blocks), groups = (total + kBlock - 1) / kBlock;
  const bool whole = item_elems % 8 == 0, away = far(2 * items * item_elems * es);
  auto launch = [&](auto dt) {
    constexpr int DT = decltype(dt)::value;
    const char* xs = static_cast<const char*>(x);
    char* ys = static_cast<char*>(y);
    hipStream_t stream = (hipStream_t)stream_;
    const unsigned across = std::min(groups, (unsigned)kMaxGrid);
    const dim3 grid(across, (groups + across - 1) / across), block(kBlock);
    if (whole && away)
      hipLaunchKernelGGL((dropout_blocks_kernel<DT, true>), grid, block, 0, stream, xs, ys, total, groups, (unsigned)blocks, (unsigned)C, d);
    else if (whole)
      hipLaunchKernelGGL((dropout_blocks_kernel<DT, false>), grid, block, 0, stream, xs, ys, total, groups, (unsigned)blocks, (unsigned)C, d);
    else
      hipLaunchKernelGGL(dropout_kernel<DT>, grid, block, 0, stream, xs, ys, (unsigned)items, groups, (unsigned long long)item_elems,
                         (unsigned)blocks, (unsigned)C, d);
  };
  if (dtype == kF32) launch(std::integral_constant<int, kF32>{});
  else if (dtype == kBF16) launch(std::integral_constant<int, kBF16>{});
  else launch(std::integral_constant<int, kF16>{});
  return sfm_last_error();
}
