// Shared parts of the windowed-attention kernels: which keys a query sees, how
// the keys of a work item are cut into blocks, and the operand types.
//
// Query t of batch b stands at position p = t + n - m and sees key j when
//   j <= p,  j < kv_len[b],  and  (j > p - window  or  j < n_first).
// Rows of a tile are (token, head) pairs of one kv head's group of G heads,
// token-major: row r is token tok0 + r / G, head r % G of the group, so every
// group size shares its keys within a tile and the keys that a tile reads are
// about the window plus the tile's few tokens.
//
// The keys of a work item are its first tokens [0, nf) and its window range
// [lo, hi), each cut into blocks of 32 keys; the blocks of both stand one
// after the other, so a few first tokens cost one block and not one whole
// chunk. When the two ranges touch they are one range from key 0.
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace dsa {
namespace win {

constexpr int kRows = 128;   // rows of a tile (TMEM lanes)
constexpr int kBlk = 32;     // keys of a block
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kBoxBytes = kRows * 128;  // one [128 rows x 64 columns] SW128 box

// 16-bit operand types: element format of tcgen05 kind::f16 and the rounding
// of two fp32 values into a packed pair (low half first). kNarrow: the exponent's range is
// smaller than fp32's, so values far from 1 have to be scaled before they are rounded.
struct Bf16 {
  static constexpr uint32_t kFmt = 1;
  static constexpr bool kNarrow = false;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
};
struct Fp16 {
  static constexpr uint32_t kFmt = 0;
  static constexpr bool kNarrow = true;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  static __device__ __forceinline__ float lo(uint32_t w) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(w & 0xFFFFu)));
  }
  static __device__ __forceinline__ float hi(uint32_t w) {
    return __half2float(__ushort_as_half(static_cast<unsigned short>(w >> 16)));
  }
};

// Instruction descriptor for kind::f16 with 16-bit A/B of one type and fp32 D
// (field layout: make_idesc_bf16_f32).
template <typename T>
__host__ __device__ constexpr uint32_t make_idesc(int M, int N, int b_mn_major) {
  return (1u << 4) | (T::kFmt << 7) | (T::kFmt << 10) |
         (static_cast<uint32_t>(b_mn_major) << 16) | (static_cast<uint32_t>(N >> 3) << 17) |
         (static_cast<uint32_t>(M >> 4) << 24);
}

// Registers of the executing warpgroup (all four warps execute it); the sum over
// the CTA's warpgroups must not exceed what the launch allotted.
template <int N>
__device__ __forceinline__ void set_max_regs_inc() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void set_max_regs_dec() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

struct Shape {
  int m, n;        // queries and keys per batch
  int h, hk, g;    // query heads, kv heads, heads per group (h / hk)
  int window, n_first;
  const int* kv_lens;  // [batch] valid keys, or null (= n)
};

// Valid keys of batch b, in [0, n].
__device__ __forceinline__ int kv_len_of(const Shape& s, int b) {
  if (s.kv_lens == nullptr) return s.n;
  return min(max(__ldg(s.kv_lens + b), 0), s.n);
}

// The key blocks that tokens [t0, t1) read (t1 > t0).
struct Range {
  int lo, hi;    // window range (from 0 when it touches the first tokens)
  int nf;        // first tokens that stand apart from the window range
  int nfb;       // their blocks
  int nblk;      // all blocks
  __device__ __forceinline__ int key(int i) const {  // first key of block i
    return i < nfb ? i * kBlk : lo + (i - nfb) * kBlk;
  }
};

__device__ __forceinline__ Range key_range(const Shape& s, int t0, int t1, int kv_len) {
  Range r;
  const int off = s.n - s.m;
  r.hi = max(min(t1 + off, kv_len), 0);
  r.lo = max(t0 + off - s.window + 1, 0);
  const int nf = min(s.n_first, r.hi);
  if (r.lo <= nf) {
    r.lo = 0;
    r.nf = 0;
  } else {
    r.nf = nf;
  }
  r.nfb = (r.nf + kBlk - 1) / kBlk;
  r.nblk = r.nfb + (r.hi > r.lo ? (r.hi - r.lo + kBlk - 1) / kBlk : 0);
  return r;
}

// Bits [a, b) of a 32-bit word (any a, b; empty when b <= a).
__device__ __forceinline__ uint32_t bits_between(int a, int b) {
  a = min(max(a, 0), 32);
  b = min(max(b, 0), 32);
  const uint32_t below_b = b == 32 ? 0xFFFFFFFFu : (1u << b) - 1u;
  const uint32_t below_a = a == 32 ? 0xFFFFFFFFu : (1u << a) - 1u;
  return below_b & ~below_a;
}

// Which keys of block i (bit c = key r.key(i) + c) the query at position pos sees.
__device__ __forceinline__ uint32_t seen_bits(const Shape& s, const Range& r, int i, int pos,
                                              int kv_len) {
  const int key = r.key(i);
  const int top = min(pos + 1, kv_len) - key;  // keys below it are causal and valid
  if (i < r.nfb) return bits_between(0, min(top, r.nf - key));
  const uint32_t near = bits_between(pos - s.window + 1 - key, top);
  return near | bits_between(0, min(top, s.n_first - key));
}

__device__ __forceinline__ void tmem_st_x16_nowait(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,"
      "%14,%15,%16};\n"
      :
      : "r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]),
        "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
        "r"(r[14]), "r"(r[15])
      : "memory");
}

// Work items of the kernels that walk the keys of fixed rows: two tiles of
// consecutive tokens of one (batch, kv head).
struct TileGrid {
  int tt;               // tokens of a tile
  int items_per_head;   // pairs of tiles
  int items;
};

// The item's keys are read in chunks of CB blocks (the last one may be shorter).
// Tile w sees keys of chunk c only if c <= last[w] and (c < head or c >= tail[w]):
// chunks with first tokens, and those from its own window's start on.
template <int CB>
struct Item {
  int b, kvh, kv_len;
  int t00, t10;      // first tokens of the tiles
  int t01, t11;      // past their last ones; a tile is empty when t_1 <= t_0
  Range r;
  int chunks, head;
  int tail0, tail1, last0, last1;

  __device__ __forceinline__ int t0(int w) const { return w ? t10 : t00; }
  __device__ __forceinline__ int t1(int w) const { return w ? t11 : t01; }
  __device__ __forceinline__ int last(int w) const { return w ? last1 : last0; }
  __device__ __forceinline__ int blocks(int c) const { return min(CB, r.nblk - c * CB); }
  __device__ __forceinline__ bool active(int w, int c) const {
    return c <= last(w) && (c < head || c >= (w ? tail1 : tail0));
  }
  __device__ __forceinline__ int first(int w) const { return head > 0 ? 0 : (w ? tail1 : tail0); }
};

template <int CB>
__device__ __forceinline__ void tile_span(const Shape& s, const Item<CB>& it, int t0, int t1,
                                          int* tail, int* last) {
  const int off = s.n - s.m;
  const int hi = min(t1 + off, it.kv_len);
  const int lo = t0 + off - s.window + 1;
  // blocks of the window range that lie below hi, and those wholly below lo
  const int below = max(hi - it.r.lo + kBlk - 1, 0) / kBlk;
  const int end = min(it.r.nfb + below, it.r.nblk);
  *tail = (it.r.nfb + max(lo - it.r.lo, 0) / kBlk) / CB;
  int l = t1 > t0 && hi > 0 && end > 0 ? (end - 1) / CB : -1;
  // a window that starts past the valid keys: first tokens only
  if (l >= it.head && l < *tail) l = it.head - 1;
  *last = l;
}

// The items of one CTA: blockIdx.x, blockIdx.x + gridDim.x, ... as (batch, kv head, pair
// of tiles), stepped without divisions.
struct ItemWalk {
  int item, b, kvh, pair;
  int step_bh, step_pair;
  __device__ __forceinline__ ItemWalk(const Shape& s, const TileGrid& g) {
    item = blockIdx.x;
    const int bh = item / g.items_per_head;
    pair = item - bh * g.items_per_head;
    b = bh / s.hk;
    kvh = bh - b * s.hk;
    step_bh = gridDim.x / g.items_per_head;
    step_pair = gridDim.x - step_bh * g.items_per_head;
  }
  __device__ __forceinline__ void next(const Shape& s, const TileGrid& g) {
    item += gridDim.x;
    pair += step_pair;
    kvh += step_bh;
    if (pair >= g.items_per_head) {
      pair -= g.items_per_head;
      ++kvh;
    }
    while (kvh >= s.hk) {
      kvh -= s.hk;
      ++b;
    }
  }
};

template <int CB>
__device__ __forceinline__ Item<CB> make_item(const Shape& s, const TileGrid& g, const ItemWalk& w) {
  Item<CB> it;
  const int t = w.pair * 2 * g.tt;
  it.b = w.b;
  it.kvh = w.kvh;
  it.kv_len = kv_len_of(s, it.b);
  it.t00 = t;
  it.t01 = it.t10 = min(t + g.tt, s.m);
  it.t11 = min(t + 2 * g.tt, s.m);
  it.r = key_range(s, it.t00, it.t11, it.kv_len);
  it.chunks = (it.r.nblk + CB - 1) / CB;
  // chunks with first tokens: of their own blocks, or of the one range from key 0
  const int heads = it.r.nfb > 0 ? it.r.nfb : (it.r.lo == 0 ? (s.n_first + kBlk - 1) / kBlk : 0);
  it.head = (heads + CB - 1) / CB;
  tile_span<CB>(s, it, it.t00, it.t01, &it.tail0, &it.last0);
  tile_span<CB>(s, it, it.t10, it.t11, &it.tail1, &it.last1);
  return it;
}

// Whether every row of the tile with tokens [t0, t1) sees all keys of chunk c.
template <int CB>
__device__ __forceinline__ bool chunk_full(const Shape& s, const Item<CB>& it, int t0, int t1, int c) {
  const int off = s.n - s.m;
  const int key = it.r.key(c * CB);
  const int end = key + it.blocks(c) * kBlk;
  return c * CB >= it.r.nfb && key > t1 - 1 + off - s.window && end <= t0 + off + 1 &&
         end <= it.kv_len;
}

// Stores 32 columns (16 packed words) of one row per lane to global memory: through
// 2 KB of the warp's own shared memory, so that each store instruction writes whole
// 64-byte pieces of 8 rows and not 16 bytes of 32. `row` is the lane's row (null: not
// stored).
__device__ __forceinline__ void store_rows(uint32_t stage, const uint32_t (&x)[16], uint16_t* row,
                                           int lane) {
#pragma unroll
  for (int j = 0; j < 4; ++j)
    st_shared_v4(stage + static_cast<uint32_t>(lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4)), x[4 * j],
                 x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2), j = lane & 3;
    const float4 v = ld_shared_f4(stage + static_cast<uint32_t>(r * 64 + ((j ^ ((r >> 1) & 3)) << 4)));
    const uint64_t at = __shfl_sync(0xFFFFFFFFu, reinterpret_cast<uint64_t>(row), r);
    if (at != 0) reinterpret_cast<float4*>(at)[j] = v;
  }
  __syncwarp();
}

}  // namespace win
}  // namespace dsa
