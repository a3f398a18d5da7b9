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
//
// This file: what both directions share.
#pragma once
#include "norm_drop.h"

namespace sfm {
namespace {


// Workgroups per CU that a pass is launched with; a workgroup is one wave per SIMD, and all of a launch have to be resident (the
// kernels' bounds hold their registers down to that): one more than fits is a second round of the whole length.  Some masked kernels
// of the backward meet their bound with scratch: 8-48 bytes in the sums (16 bits with one or two channels of a group in a vector, and fp32
// by single elements), 80-84 in the last pass of 16 bits in eights with one, 20 in that of vectors of four.  Measured without a mask, at 0.5 GB
// a tensor, us: statistics at 4 / 6 / 8: 97 / 94 / 98; forward's last pass fp32 at 4 / 6: 180 / 171, bf16 at 4 / 6: 193 / 200; backward's sums fp32 at 4 / 5: 194 / 172
// (16-bit types hold two vectors of eight in registers: 4); its last pass fp32 at 4 / 5: 251 / 245.
// Vectors of up to four bytes take few registers and have few bytes in flight: more.  (Without and with, us for a step of 8x128x416 rows: 45
// channels fp32 159 and 144, bf16 151 and 128; 199 bf16 729 and 544.)
constexpr int waves_stats(int es, int V) { return es * V <= 4 ? 8 : 6; }
constexpr int waves_apply(int es, int V) { return es * V <= 4 || es == 4 ? 6 : 4; }
constexpr int waves_sums(int es, int V) { return es * V <= 4 ? 8 : es == 4 ? 5 : 4; }
constexpr int waves_bwd_apply(int es, int V) { return es * V <= 4 ? 6 : es == 4 ? 5 : 4; }
// (a vector that crosses many groups has a set of statistics for each and takes what registers it needs)
constexpr int bound_of(int groups_of_vector, int waves) { return groups_of_vector <= 2 ? waves : 4; }
constexpr int kCUs = 256;
constexpr int kMaxChunks = 1024;
// Rows a thread has in flight: more of them where an odd channel count makes its vectors short.  Four and eight, us for a step of 8x128x416
// rows: 45 channels bf16 134 and 128, 90 bf16 144 and 135; with vectors of eight bytes 100 bf16 148 and 153, 50 fp32 137 and 141.
constexpr int batch_of(int vector_bytes) { return vector_bytes > 4 ? 4 : 8; }

// How an item is cut: channels into slabs (whole groups, or an even part of one wide group), rows into tiles of U * row_lanes
// rows (U = batch_of), and the tiles in turn to the chunks (tile t to chunk t % chunks), one workgroup each.  In turn and not in runs: the
// workgroups then move through memory side by side.  Passes over tensors of 512 MB, nontemporal: read + write 175 us in turn, 190 in
// runs; two reads + write 263 and 283.
struct GnPlan {
  long long N;
  int C, G, cpg;
  int V, U;              // elements per thread and row; rows in a batch of a thread
  int cs;                // channels of a slab (the last one of a group or of the row may have fewer)
  int slabs;             // slabs of a row
  int groups_per_slab;   // >= 1; 1 where a group has parts
  int parts;             // slabs of a group (1 where a slab holds whole groups)
  int lanes;             // cs / V
  unsigned lanes_inv, cpg_inv;  // ceil(2^20 / lanes), ceil(2^32 / cpg) (0: one channel per group): quotients by a product
  int row_lanes;         // kBlock / lanes: rows a workgroup takes at once
  int tile_rows;
  long long tiles;
  int left;              // rows of the last tile
  struct Turn {          // how a pass deals out the tiles
    int chunks;
    long long own;       // tiles of a chunk; the first `extra` chunks have one more
    int extra;
    int owner;           // the chunk of the last tile
    float rows, rows_more;  // rows of a chunk of `own` tiles and of one more, were the last tile full
  } first, last;         // the pass that makes partial sums, and the one that joins and applies them
  bool pairs;            // lanes 2i and 2i + 1 always hold the halves of a block of eight channels (fp32; draw_pair)
  int P;                 // partials of a group: first.chunks * parts
};

static inline int gcd_int(int a, int b) {
  while (b) { const int t = a % b; a = b; b = t; }
  return a;
}

// (also once the numbers of chunks are known: a row stride may ask for fewer row lanes, which makes more tiles of the same chunks)
static void gn_tiles(GnPlan& p, int row_lanes) {
  p.row_lanes = row_lanes;
  p.tile_rows = p.U * row_lanes;
  p.tiles = (p.N + p.tile_rows - 1) / p.tile_rows;
  p.left = (int)(p.N - (p.tiles - 1) * p.tile_rows);
  for (GnPlan::Turn* t : {&p.first, &p.last}) {
    if (t->chunks < 1) t->chunks = 1;
    t->own = p.tiles / t->chunks;
    t->extra = (int)(p.tiles % t->chunks);
    t->owner = (int)((p.tiles - 1) % t->chunks);
    t->rows = (float)(t->own * p.tile_rows);
    t->rows_more = (float)((t->own + 1) * p.tile_rows);
  }
}

// (the arguments have been checked; false: an item is too large)
static bool gn_plan(long long B, long long N, int C, int G, int es, bool backward, GnPlan& p) {
  p = GnPlan{};
  p.N = N; p.C = C; p.G = G; p.cpg = C / G;
  p.V = 16 / es;
  while (C % p.V) p.V /= 2;
  // a slab of whole groups is a multiple of lcm(cpg, V); where that is too wide for a workgroup and V does not divide a group
  // either (a part of a group has to start at a multiple of V), a smaller V does
  for (;; p.V /= 2) {
    if (p.cpg % p.V == 0) break;
    if (p.cpg / gcd_int(p.cpg, p.V) <= kBlock) break;
  }
  p.U = batch_of(p.V * es);
  const int unit_groups = p.V / gcd_int(p.cpg, p.V);                      // groups of the smallest slab
  const long long unit = (long long)p.cpg * unit_groups;
  if (unit / p.V <= kBlock) {
    // The narrowest slab of whole 128-byte lines: fewer partials for a workgroup to join than with a wide one.  Where rows are no whole lines
    // that would have workgroups all over the chip read each other's lines, so a slab is then as wide as a workgroup.
    const long long widest = std::min<long long>(kBlock * (long long)p.V, C) / unit;
    long long k = widest;
    if ((long long)C * es % 128 == 0)
      for (long long n = 1; n < widest; ++n)
        if (n * unit * es % 128 == 0) { k = n; break; }
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
  p.pairs = p.V == 4 && es == 4 && C % 8 == 0 && p.cs % 8 == 0 && (p.parts == 1 || p.cpg % 8 == 0);  // every slab starts and ends with a block
  p.lanes_inv = ((1u << 20) + p.lanes - 1) / p.lanes;
  p.cpg_inv = p.cpg == 1 ? 0u : (unsigned)(((1ull << 32) + p.cpg - 1) / p.cpg);
  gn_tiles(p, kBlock / p.lanes);
  auto deal = [&](int waves) {
    const long long per = (long long)B * p.slabs;
    const long long chunks = std::min({((long long)waves * kCUs + per - 1) / per, p.tiles, (long long)kMaxChunks});
    const long long each = (p.tiles + chunks - 1) / chunks;  // as even as whole tiles allow
    return (int)((p.tiles + each - 1) / each);
  };
  p.first.chunks = deal(backward ? waves_sums(es, p.V) : waves_stats(es, p.V));
  p.last.chunks = deal(backward ? waves_bwd_apply(es, p.V) : waves_apply(es, p.V));
  p.P = p.first.chunks * p.parts;
  gn_tiles(p, p.row_lanes);
  return true;
}

// ---- what a workgroup works on
struct Where {
  int b, slab, chunk, part;
  int c0, cc, g0, ng;  // first channel and channels of the slab, first group and groups of it
};
// a grid is (items, chunks, slabs): with a multiple of eight items all of an item is on one XCD in every pass
__device__ __forceinline__ Where where(const GnPlan& p, unsigned b, unsigned chunk, unsigned slab) {
  Where w;
  w.b = b;
  w.chunk = chunk;
  w.slab = slab;
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
  return w;
}

// A tile's rows go to the row lanes in U steps: step u, row lane ry: row u * row_lanes + ry of the tile.  Everything here but
// the thread's own place is uniform: the address of a load is a uniform pointer and a 32-bit offset of the thread (gn_setup
// keeps the rows of a step within 31 bits of bytes).
struct Lane {
  int vx, ry;
  bool mine;  // this thread has a vector at all
  __device__ __forceinline__ Lane(const GnPlan& p, const Where& w, int row_lanes) {
    ry = threadIdx.x * p.lanes_inv >> 20;  // threadIdx.x / lanes: exact, 1024 * 256 < 2^20
    vx = threadIdx.x - ry * p.lanes;
    mine = ry < row_lanes && vx * p.V < w.cc;
  }
};
// the group of a slab's channel, in the slab: channel / cpg, exact, 2048 * 2048 < 2^32
__device__ __forceinline__ int group_in_slab(const GnPlan& p, int channel) {
  return p.parts > 1 ? 0 : p.cpg_inv ? (int)__umulhi((unsigned)channel, p.cpg_inv) : channel;
}
template <int U> struct Tile {
  long long index;
  int steps;  // steps in which row lane 0 has a row
  int last;   // rows of the last of them (1 .. row_lanes)
  bool full;
  __device__ __forceinline__ Tile(const GnPlan& p, long long i) : index(i) {
    full = i < p.tiles - 1 || p.left == p.tile_rows;
    steps = full ? U : (p.left + p.row_lanes - 1) / p.row_lanes;
    last = full ? p.row_lanes : p.left - (steps - 1) * p.row_lanes;
  }
  __device__ __forceinline__ bool valid(int u, int ry) const { return full || u < steps - 1 || (u == steps - 1 && ry < last); }
};

// The last pass goes through a workgroup's tiles from the last one down: the first pass has left the latest of them in the caches
// (the same workgroup on the same XCD, whose L2 is its own).  54 MB a tensor: 87.1 -> 83.8 us for the four passes; 0.5 GB a
// tensor: 768 -> 784, so not there (FAR).
__device__ __forceinline__ long long last_tile(const GnPlan& p, const Where& w) {
  return w.chunk + (p.last.own + (w.chunk < p.last.extra) - 1) * p.last.chunks;
}

template <int DT, int V, bool NT = false> struct Stream {  // NT: nontemporal, for tensors that no cache holds until they are read again (far())
  static constexpr int kES = ElemBytes<DT>::value, U = batch_of(V * kES);
  const char* base;
  long long step;      // bytes of the rows of a step
  unsigned off, lead;  // of this thread; lead: its row lane's share of it
  __device__ __forceinline__ Stream(const void* p, long long ld, const GnPlan& pl, const Where& w, const Lane& l) {
    base = static_cast<const char*>(p) + ((long long)w.b * pl.N * ld + w.c0) * kES;
    step = (long long)pl.row_lanes * ld * kES;
    lead = (unsigned)(l.ry * ld * kES);
    off = lead + (unsigned)(l.vx * V * kES);
  }
  __device__ __forceinline__ const char* at(const Tile<U>& t) const { return base + t.index * U * step; }
  // step u < steps of the tile at `a`; in its last step a row lane without a row reads row lane 0's
  __device__ __forceinline__ Raw<DT, V> row(const char* a, const Tile<U>& t, int u, int ry) const {
    return load_raw<DT, V, NT>(a + u * step, off - (t.valid(u, ry) ? 0u : lead));
  }
  __device__ __forceinline__ void load(const Tile<U>& t, int ry, Raw<DT, V> (&raw)[U]) const {
    const char* a = at(t);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u < t.steps) raw[u] = row(a, t, u, ry);
  }
  __device__ __forceinline__ void store(const char* a, int u, const float (&f)[V]) const {
    store_vec<DT, V, NT>(const_cast<char*>(a) + u * step, off, f);
  }
};

// The mask of a thread's vector in the rows of a tile, u ascending from 0 in every tile.
template <int V> struct Mask {
  static constexpr bool kXor3 = V != 8;  // (philox7)
  const Drop& d;
  DropKey key;
  unsigned item;
  bool pairs;
  Draw<V> now, next;
  __device__ __forceinline__ Mask(const Drop& drop, const GnPlan& p, const Where& w, int channel)
      : d(drop), key(drop_key(drop)), item(drop.item0 + w.b), pairs(p.pairs) {
    if (d.per_channel) now = draw<V, kXor3>(d, key, item, channel);
  }
  // place: of the vector in row u; step: places between rows u and u + 1
  __device__ __forceinline__ void apply(float (&f)[V], int u, unsigned long long place, unsigned long long step) {
    if (!d.per_channel) {
      if constexpr (V == 4) {
        if (pairs) {
          if (u & 1) now = next;
          else draw_pair(d, key, item, place, step, now, next);
        } else now = draw<V>(d, key, item, place);
      } else now = draw<V, kXor3>(d, key, item, place);
    }
    drop_apply<V>(f, now, d);
  }
};
struct NoMask {
  template <typename... T> __device__ __forceinline__ NoMask(const T&...) {}
};

// Teams: the workgroup's threads, cut into teams of T lanes of one wave (T a power of two), one group each at a time.
struct Team { int T, id, lane, count; };
template <int THREADS = kBlock> __device__ __forceinline__ Team team_of(int ng) {
  int T = 64;
  while (T > 1 && THREADS / T < ng) T >>= 1;
  return {T, (int)threadIdx.x / T, (int)threadIdx.x & (T - 1), THREADS / T};
}
template <typename F> __device__ __forceinline__ F team_sum(F v, int T) {
  for (int o = T >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// f(k, value) for k = first, first + step, ... < n of src, K loads on their way at a time: partial sums have been written by
// workgroups all over the chip, a load of one takes about a microsecond, and one after the other they were most of a small pass
template <int K, typename F> __device__ __forceinline__ void each_partial(const float2* __restrict__ src, long long n, int first, int step, F&& f) {
  for (long long base = first; base < n; base += K * step) {
    float2 v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] = src[min(base + k * step, n - 1)];
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (base + k * step < n) f((int)(base + k * step), v[k]);
  }
}

// values that partial q of a group covers
__device__ __forceinline__ float part_count(const GnPlan& p, int q) {
  const int chunk = p.parts == 1 ? q : q / p.parts, part = q - chunk * p.parts;
  const float rows = (chunk < p.first.extra ? p.first.rows_more : p.first.rows) - (chunk == p.first.owner ? (float)(p.tile_rows - p.left) : 0.0f);
  return rows * (float)(p.parts == 1 ? p.cpg : min(p.cs, p.cpg - part * p.cs));
}

// dispatch on the type, the vector width, and how many adjacent channels of a vector are of one group (a power of two that divides
// both: a thread keeps one set of statistics for them): fn(DT, V, E) as integral constants
template <typename F> static void by_type(int dtype, const GnPlan& p, F&& fn) {
  using std::integral_constant;
  int one = p.V;
  while (p.cpg % one) one /= 2;
  auto width = [&](auto dt) {
    auto go = [&](auto v) {
      constexpr int V = decltype(v)::value;
      if constexpr (V >= 8) { if (one == 8) return fn(dt, v, integral_constant<int, 8>{}); }
      if constexpr (V >= 4) { if (one == 4) return fn(dt, v, integral_constant<int, 4>{}); }
      if constexpr (V >= 2) { if (one == 2) return fn(dt, v, integral_constant<int, 2>{}); }
      fn(dt, v, integral_constant<int, 1>{});
    };
    if constexpr (decltype(dt)::value != kF32) { if (p.V == 8) return go(integral_constant<int, 8>{}); }
    if (p.V == 4) return go(integral_constant<int, 4>{});
    if (p.V == 2) return go(integral_constant<int, 2>{});
    go(integral_constant<int, 1>{});
  };
  if (dtype == kF32) return width(integral_constant<int, kF32>{});
  if (dtype == kBF16) return width(integral_constant<int, kBF16>{});
  width(integral_constant<int, kF16>{});
}

// fn(DROP, FAR): nontemporal accesses come in the full width alone
template <int DT, int V, typename F> static void by_use(bool drop, bool away, F&& fn) {
  if constexpr (V * ElemBytes<DT>::value == 16) {
    if (away && drop) return fn(std::true_type{}, std::true_type{});
    if (away) return fn(std::false_type{}, std::true_type{});
  }
  if (drop) fn(std::true_type{}, std::false_type{});
  else fn(std::false_type{}, std::false_type{});
}

// rows of C elements of es bytes, ld elements apart
static bool rows_ok(const void* q, long long ld, int C, int es) { return q && ld >= C && ((uintptr_t)q & (es - 1)) == 0; }

// ld: the widest row stride of the call
static int gn_setup(long long B, long long N, int C, int G, int dtype, long long ld, bool backward, GnPlan& p, dim3& first,
                    dim3& last) {
  if (dtype < kF32 || dtype > kF16 || B < 1 || N < 1 || C < 1 || G < 1 || C % G || ld < C) return SFM_ERR_ARG;
  const int es = dtype == kF32 ? 4 : 2;
  // items are counted in 31 bits, elements in 60 with room for strides, the threads of a launch in 32 per dimension of the grid; the
  // rows that a workgroup takes at once lie within 31 bits of bytes of each other
  if (B > 0x7fffffffll || (__int128)B * N > ((__int128)1 << 40) || ld > 0x7fffffffll / es || !gn_plan(B, N, C, G, es, backward, p))
    return SFM_ERR_TOO_LARGE;
  gn_tiles(p, (int)std::min<long long>(p.row_lanes, 0x7fffffffll / (ld * es)));
  const __int128 blocks = (__int128)B * p.slabs * std::max(p.first.chunks, p.last.chunks);
  // (a launch's workgroups in one dimension, and with them those that sum the parameters' gradients; up to 1024 threads each)
  if (blocks + C > kMaxGrid || p.slabs > 65535) return SFM_ERR_TOO_LARGE;
  first = dim3((unsigned)B, p.first.chunks, p.slabs);
  last = dim3((unsigned)B, p.last.chunks, p.slabs);
  return SFM_OK;
}

}  // namespace
}  // namespace sfm
