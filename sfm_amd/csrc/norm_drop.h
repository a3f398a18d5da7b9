// Shared by the group norm and the dropout kernels: element types, vector loads, activations, the counter-based mask.
#pragma once
#include "sfm_device.h"
#include "sfm_internal.h"
#include <algorithm>
#include <type_traits>

namespace sfm {

constexpr long long kMaxGrid = (1ll << 32) / 1024 - 1;  // workgroups of up to 1024 threads in a dimension of a grid

// ---- element types (SFM_F32 / SFM_BF16 / SFM_F16 of the C ABI).  Everything is computed in fp32; a 16-bit tensor is rounded
// once, to nearest even, where it is stored.
enum { kF32 = 0, kBF16 = 1, kF16 = 2 };
template <int DT> struct ElemBytes { static constexpr int value = DT == kF32 ? 4 : 2; };

template <int N> struct Words;  // N bytes as unsigned words, at any element alignment (global accesses need none wider)
template <> struct Words<32> { typedef unsigned t __attribute__((ext_vector_type(8), aligned(4))); };
template <> struct Words<16> { typedef unsigned t __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct Words<8> { typedef unsigned t __attribute__((ext_vector_type(2), aligned(2))); };

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
struct __attribute__((packed, aligned(2))) PackedU32 { unsigned v; };

// V consecutive elements in the registers they arrive in (V = 1: one element, zero-extended)
template <int DT, int V> struct Raw { unsigned w[V * ElemBytes<DT>::value < 4 ? 1 : V * ElemBytes<DT>::value / 4]; };

// (macros: a template parameter would drop the pointee's alignment)
#define SFM_GET(NT, T, p) (NT ? __builtin_nontemporal_load(reinterpret_cast<const T*>(p)) : *reinterpret_cast<const T*>(p))
#define SFM_PUT(NT, T, p, v) do { if (NT) __builtin_nontemporal_store(v, reinterpret_cast<T*>(p)); else *reinterpret_cast<T*>(p) = v; } while (0)

template <int DT, int V, bool NT = false, typename Offset>
__device__ __forceinline__ Raw<DT, V> load_raw(const char* __restrict__ base, Offset bytes) {
  constexpr int kBytes = V * ElemBytes<DT>::value;
  const char* p = base + bytes;
  Raw<DT, V> r;
  if constexpr (kBytes == 2) r.w[0] = *reinterpret_cast<const unsigned short*>(p);
  else if constexpr (kBytes == 4) r.w[0] = reinterpret_cast<const PackedU32*>(p)->v;
  else if constexpr (kBytes == 32) {
    const auto a = SFM_GET(NT, Words<16>::t, p), b = SFM_GET(NT, Words<16>::t, p + 16);
#pragma unroll
    for (int k = 0; k < 4; ++k) { r.w[k] = a[k]; r.w[4 + k] = b[k]; }
  } else {
    const auto a = SFM_GET(NT, typename Words<kBytes>::t, p);
#pragma unroll
    for (int k = 0; k < kBytes / 4; ++k) r.w[k] = a[k];
  }
  return r;
}

template <int DT, int V>
__device__ __forceinline__ void unpack(const Raw<DT, V>& r, float (&f)[V]) {
  if constexpr (DT == kF32) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = __uint_as_float(r.w[k]);
  } else if constexpr (DT == kBF16) {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = __uint_as_float(k & 1 ? r.w[k / 2] & 0xffff0000u : r.w[k / 2] << 16);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = (float)__builtin_bit_cast(_Float16, (unsigned short)(k & 1 ? r.w[k / 2] >> 16 : r.w[k / 2]));
  }
}

template <int DT, int V, bool NT = false, typename Offset>
__device__ __forceinline__ void store_vec(char* __restrict__ base, Offset bytes, const float (&f)[V]) {
  constexpr int kBytes = V * ElemBytes<DT>::value;
  char* p = base + bytes;
  Raw<DT, V> r;
  if constexpr (DT == kF32) {
#pragma unroll
    for (int k = 0; k < V; ++k) r.w[k] = __float_as_uint(f[k]);
  } else if constexpr (V == 1) {
    if constexpr (DT == kBF16) r.w[0] = __builtin_bit_cast(unsigned short, (__bf16)f[0]);
    else r.w[0] = __builtin_bit_cast(unsigned short, (_Float16)f[0]);
  } else {
#pragma unroll
    for (int k = 0; k < V / 2; ++k) {
      const f32x2 v = {f[2 * k], f[2 * k + 1]};
      if constexpr (DT == kBF16) r.w[k] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2));
      else r.w[k] = __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2));
    }
  }
  if constexpr (kBytes == 2) *reinterpret_cast<unsigned short*>(p) = (unsigned short)r.w[0];
  else if constexpr (kBytes == 4) reinterpret_cast<PackedU32*>(p)->v = r.w[0];
  else if constexpr (kBytes == 32) {
    Words<16>::t a, b;
#pragma unroll
    for (int k = 0; k < 4; ++k) { a[k] = r.w[k]; b[k] = r.w[4 + k]; }
    SFM_PUT(NT, Words<16>::t, p, a);
    SFM_PUT(NT, Words<16>::t, p + 16, b);
  } else {
    typename Words<kBytes>::t a;
#pragma unroll
    for (int k = 0; k < kBytes / 4; ++k) a[k] = r.w[k];
    SFM_PUT(NT, typename Words<kBytes>::t, p, a);
  }
}

// A last pass over tensors that together pass the memory-side cache (256 MB) reads and writes nontemporally: nothing of them would be found
// there again.  1024x2048x32 bf16 serve 650 -> 605 us, train 863 -> 778; under it a reader of the result may still find it, and
// the pass itself gains little (concat4 of the 128x416 decoder, 54 MB a tensor: 87.1 -> 84.5 us for four passes).
static inline bool far(long long bytes) { return bytes > (256ll << 20); }

// ---- activations (SFM_ACT_* of the C ABI)
enum { kActNone = 0, kActElu = 1, kActRelu = 2, kActSilu = 3 };
constexpr float kLog2e = 1.44269504088896341f;

// e^z by the hardware's base-2 exponential: relative error |z| 2^-24 from the rounded argument and an ulp of the instruction.
// Results under 2^-126 become 0, which no activation below can tell from what they are.
__device__ __forceinline__ float exp_fast(float z) { return __builtin_amdgcn_exp2f(z * kLog2e); }

// elu(z) = z > 0 ? z : e^z - 1.  e^z - 1 as it stands is off by 2^-24 of 1, which leaves nothing of a small z (with small gamma and beta all of
// them are, and as exact as any).  So next to 0 it is a polynomial, with min(z, 0) for its argument: a positive z comes out as it is.
//   fp32: z + z^2 (a + b z + c z^2) from -1/4, a least-squares fit of the relative error there: 2^-21 at most on either side of the border.
//   16 bits: z + z^2 / 2 from -2^-7: 2^-16 on either side, a 32nd of fp16's own rounding (a memory-bound pass with half the bytes an
//   element has less time for arithmetic).
// Against e^z - 1 alone: 8x1024x2048x32 bf16 serve 560 -> 571 us, 16x192x624x64 fp32 train 652 -> 654, 8x128x416x32 fp32 train 84.2 -> 84.9.
template <int DT> __device__ __forceinline__ float elu(float z) {
  const float m = __builtin_elementwise_minimum(z, 0.0f), e = exp_fast(z) - 1.0f;
  if constexpr (DT == kF32) {
    const float q = __builtin_fmaf(m, __builtin_fmaf(m, 0.03786944f, 0.1661234f), 0.49997758f);
    return z > -0.25f ? __builtin_fmaf(m * m, q, z) : e;
  } else {
    return z > -0x1p-7f ? __builtin_fmaf(0.5f * m, m, z) : e;  // (a NaN is one in e)
  }
}

__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.0f + exp_fast(-z)); }

template <int DT, int V>
__device__ __forceinline__ void act_fwd(float (&z)[V], int act) {  // act is uniform
  if (act == kActElu) {
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = elu<DT>(z[k]);
  } else if (act == kActRelu) {
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = z[k] < 0.0f ? 0.0f : z[k];  // a NaN stays one
  } else if (act == kActSilu) {
#pragma unroll
    for (int k = 0; k < V; ++k) z[k] = z[k] * sigmoid(z[k]);
  }
}

// g[k] *= act'(z[k]); relu'(0) = 0, elu'(0) = 1
template <int V>
__device__ __forceinline__ void act_bwd(float (&g)[V], const float (&z)[V], int act) {
  if (act == kActElu) {
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] *= exp_fast(__builtin_elementwise_minimum(z[k], 0.0f));  // (a NaN stays one)
  } else if (act == kActRelu) {
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] = z[k] > 0.0f ? g[k] : 0.0f;
  } else if (act == kActSilu) {
#pragma unroll
    for (int k = 0; k < V; ++k) {
      const float s = sigmoid(z[k]);
      g[k] *= s * __builtin_fmaf(z[k], 1.0f - s, 1.0f);
    }
  }
}

// ---- the dropout mask: a function of (seed, step, layer, item, place), never stored.
// Philox 4x32 with seven rounds (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011; seven is the
// fewest rounds that paper reports as passing BigCrush).  A call gives four words = eight 16-bit numbers, one per element: a
// round is two 32 x 32 -> 64 bit products at a quarter of the ALU rate, so at 32 bits per element the generator and not memory
// would bound a bf16 pass.  An element is kept where its number is >= threshold; what is kept is multiplied by
// 65536 / (65536 - threshold), so the expectation is exact for the probability threshold / 65536 that is really used.
struct Drop {
  const unsigned long long* rng;  // device (seed, step), or NULL: the two below
  unsigned long long seed;
  unsigned step, layer, item0;
  unsigned threshold;  // 0: nothing is dropped
  float scale;
  int per_channel;  // one number per (item, channel) instead of one per element
};

struct DropKey { unsigned k0, k1, step; };
__device__ __forceinline__ DropKey drop_key(const Drop& d) {
  const unsigned long long seed = d.rng ? d.rng[0] : d.seed;
  return {(unsigned)seed, (unsigned)(seed >> 32), d.rng ? (unsigned)d.rng[1] : d.step};
}

// XOR3: a ^ b ^ c as one instruction, two less a round.  Not where eight elements of two 16-bit tensors are in registers with their sums and
// scales: it takes a few registers more, and those are spilled (backward's sums of 13.6 MB bf16 12.3 -> 15.1 us; elsewhere: dropout alone
// of 27 MB bf16 12.0 -> 11.5, forward's last pass of 0.5 GB fp32 173 -> 168).
template <bool XOR3> __device__ __forceinline__ uint4 philox7(unsigned c0, unsigned c1, unsigned c2, unsigned c3, unsigned k0, unsigned k1) {
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const unsigned long long a = (unsigned long long)c0 * 0xD2511F53u, b = (unsigned long long)c2 * 0xCD9E8D57u;
    const unsigned hi_a = (unsigned)(a >> 32), hi_b = (unsigned)(b >> 32);
    c0 = XOR3 ? __builtin_amdgcn_bitop3_b32(hi_b, c1, k0, 0x96) : hi_b ^ c1 ^ k0;
    c1 = (unsigned)b;
    c2 = XOR3 ? __builtin_amdgcn_bitop3_b32(hi_a, c3, k1, 0x96) : hi_a ^ c3 ^ k1;
    c3 = (unsigned)a;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

template <bool XOR3 = true> __device__ __forceinline__ uint4 block_words(const Drop& d, const DropKey& key, unsigned item, unsigned long long place) {
  return philox7<XOR3>((unsigned)(place >> 3), item, key.step, d.layer, key.k0, key.k1);
}

// the 16-bit numbers of elements place .. place + V - 1 of an item, two in a word.  V is a power of two <= 8 that divides place: the V
// elements lie in one block of eight.
template <int V> struct Draw { unsigned w[(V + 1) / 2]; };
template <int V, bool XOR3 = true>
__device__ __forceinline__ Draw<V> draw(const Drop& d, const DropKey& key, unsigned item, unsigned long long place) {
  const uint4 r = block_words<XOR3>(d, key, item, place);
  Draw<V> o;
  if constexpr (V == 8) { o.w[0] = r.x; o.w[1] = r.y; o.w[2] = r.z; o.w[3] = r.w; }
  else if constexpr (V == 4) { o.w[0] = place & 4 ? r.z : r.x; o.w[1] = place & 4 ? r.w : r.y; }
  else {
    const unsigned lo = place & 2 ? r.y : r.x, hi = place & 2 ? r.w : r.z, w = place & 4 ? hi : lo;
    o.w[0] = V == 2 || !(place & 1) ? w : w >> 16;
  }
  return o;
}

// Two draws of four elements by lanes 2i and 2i + 1 that hold the two halves of one block of eight in each of two rows: the even lane
// draws the first row's block, the odd one the second's, and they swap the halves (a quad permutation): one draw a lane for
// eight elements, not two.
__device__ __forceinline__ void draw_pair(const Drop& d, const DropKey& key, unsigned item, unsigned long long place,
                                          unsigned long long row, Draw<4>& first, Draw<4>& second) {
  const bool odd = threadIdx.x & 1;
  const uint4 r = block_words(d, key, item, place + (odd ? row : 0));
  const unsigned s0 = odd ? r.x : r.z, s1 = odd ? r.y : r.w;  // what the other lane needs
  const unsigned o0 = __builtin_amdgcn_update_dpp(0, (int)s0, 0xB1, 0xF, 0xF, true);
  const unsigned o1 = __builtin_amdgcn_update_dpp(0, (int)s1, 0xB1, 0xF, 0xF, true);
  first.w[0] = odd ? o0 : r.x;
  first.w[1] = odd ? o1 : r.y;
  second.w[0] = odd ? r.z : o0;
  second.w[1] = odd ? r.w : o1;
}

template <int V>
__device__ __forceinline__ void drop_apply(float (&f)[V], const Draw<V>& r, const Drop& d) {
  const unsigned t = d.threshold << 16;
#pragma unroll
  for (int k = 0; k < V; ++k)  // a dropped infinity or NaN is 0 as well
    f[k] = (k & 1 ? r.w[k / 2] >= t : (unsigned short)r.w[k / 2] >= (unsigned short)d.threshold) ? f[k] * d.scale : 0.0f;
}

// the same as bits: what a lane hands to others
__device__ __forceinline__ unsigned keep_bits(const Drop& d, const DropKey& key, unsigned item, unsigned long long place) {
  const uint4 r = block_words(d, key, item, place);
  const unsigned w[4] = {r.x, r.y, r.z, r.w}, t = d.threshold << 16;
  unsigned all = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) all |= ((k & 1 ? w[k / 2] : w[k / 2] << 16) >= t ? 1u : 0u) << k;
  return all;
}

template <int V>
__device__ __forceinline__ void keep_apply(float (&f)[V], unsigned keep, float scale) {
#pragma unroll
  for (int k = 0; k < V; ++k) f[k] = (keep >> k) & 1 ? f[k] * scale : 0.0f;
}

// the arguments of one mask as the C ABI passes them -> false if they are none
static inline bool drop_args(const void* rng, unsigned long long seed, unsigned step, unsigned layer, unsigned item0,
                             int threshold, int per_channel, Drop& d) {
  if (threshold < 0 || threshold > 65535 || ((uintptr_t)rng & 7) != 0) return false;
  d = Drop{static_cast<const unsigned long long*>(rng), seed, step, layer, item0, (unsigned)threshold,
           65536.0f / (float)(65536 - threshold), per_channel != 0};
  return true;
}

}  // namespace sfm
