// Dropout whose mask is a function of counters and never stored: y = keep ? x * scale : 0, and the same on dL/dy for the
// backward (norm_drop.h has the generator).  Bound by memory: one read and one write per element.
#include "norm_drop.h"

namespace sfm {
namespace {

// A thread takes blocks of eight elements of an item (one generator call); a workgroup takes kPer * kBlock consecutive blocks, so
// the 64-bit division by the blocks of an item is one uniform one per workgroup.
constexpr int kPer = 4;

template <int DT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const char* __restrict__ x, char* __restrict__ y, unsigned items,
                                                         unsigned long long n, unsigned blocks, unsigned C, Drop d) {
  const DropKey key = drop_key(d);
  const unsigned long long q0 = (unsigned long long)blockIdx.x * (kPer * kBlock);
  const unsigned item0 = (unsigned)(q0 / blocks), off0 = (unsigned)(q0 % blocks);
#pragma unroll
  for (int k = 0; k < kPer; ++k) {
    const unsigned t = k * kBlock + threadIdx.x;
    const unsigned long long off = (unsigned long long)off0 + t;
    const unsigned up = off < blocks ? 0u : (unsigned)(off / blocks);
    const unsigned item = item0 + up;
    const unsigned long long first = (off - (unsigned long long)up * blocks) * 8;
    if (item >= items) continue;
    constexpr int kBytes = ElemBytes<DT>::value;
    const long long at = (long long)(item * n + first) * kBytes;
    unsigned keep;
    if (d.per_channel) {  // the eight may start anywhere in a row of C channels and cross into the next
      keep = 0;
      unsigned c = (unsigned)(first % C), have = ~0u, eight = 0;
#pragma unroll 1
      for (int e = 0; e < 8; ++e) {
        if ((c >> 3) != have) { have = c >> 3; eight = keep_bits<8>(d, key, d.item0 + item, c & ~7u); }
        keep |= ((eight >> (c & 7)) & 1u) << e;
        c = c + 1 == C ? 0 : c + 1;
      }
    } else keep = keep_bits<8>(d, key, d.item0 + item, first);
    if (first + 8 <= n) {
      const auto r = load_raw<DT, 8>(x, at);
      float f[8];
      unpack<DT, 8>(r, f);
      drop_apply<8>(f, keep, d.scale);
      store_vec<DT, 8>(y, at, f);
    } else {
      for (unsigned e = 0; first + e < n; ++e) {
        const auto r = load_raw<DT, 1>(x, at + e * kBytes);
        float f[1];
        unpack<DT, 1>(r, f);
        drop_apply<1>(f, keep >> e, d.scale);
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
  if (groups > 0x7fffffffll) return SFM_ERR_TOO_LARGE;
  const dim3 grid((unsigned)groups), block(kBlock);
  hipStream_t stream = (hipStream_t)stream_;
#define SFM_DROP(DT) hipLaunchKernelGGL(dropout_kernel<DT>, grid, block, 0, stream, static_cast<const char*>(x), static_cast<char*>(y), (unsigned)items, (unsigned long long)item_elems, (unsigned)blocks, (unsigned)C, d)
  if (dtype == kF32) SFM_DROP(kF32);
  else if (dtype == kBF16) SFM_DROP(kBF16);
  else SFM_DROP(kF16);
#undef SFM_DROP
  return sfm_last_error();
}
