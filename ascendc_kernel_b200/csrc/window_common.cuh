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
// of two fp32 values into a packed pair (low half first).
struct Bf16 {
  static constexpr uint32_t kFmt = 1;
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) { return pack_bf16x2(lo, hi); }
  static __device__ __forceinline__ float lo(uint32_t w) { return __uint_as_float(w << 16); }
  static __device__ __forceinline__ float hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }
};
struct Fp16 {
  static constexpr uint32_t kFmt = 0;
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
  int64_t items;
};

inline TileGrid tile_grid(const Shape& s, int64_t batch) {
  TileGrid g;
  g.tt = kRows / s.g;
  g.items_per_head = ((s.m + g.tt - 1) / g.tt + 1) / 2;
  g.items = batch * s.hk * g.items_per_head;
  return g;
}

// The item's keys are read in chunks of CB blocks (the last one may be shorter).
struct Item {
  int b, kvh, kv_len;
  int t0[2], t1[2];  // tokens of each tile, empty when t1 <= t0
  Range r;

  template <int CB>
  __device__ __forceinline__ int chunks() const {
    return (r.nblk + CB - 1) / CB;
  }
  template <int CB>
  __device__ __forceinline__ int blocks(int c) const {
    return min(CB, r.nblk - c * CB);
  }
  // Whether any row of tile w sees a key of chunk c.
  template <int CB>
  __device__ __forceinline__ bool active(const Shape& s, int w, int c) const {
    if (t1[w] <= t0[w]) return false;
    const int off = s.n - s.m;
    const int hi = min(t1[w] + off, kv_len);
    const int lo = t0[w] + off - s.window + 1;
    const int nb = blocks<CB>(c);
    bool any = false;
    for (int i = 0; i < nb; ++i) {
      const int k = r.key(c * CB + i);
      any = any || (k < hi && (c * CB + i < r.nfb || k + kBlk > lo || k < s.n_first));
    }
    return any;
  }
  // First and last active chunk of tile w (last = -1 when none).
  template <int CB>
  __device__ __forceinline__ void span(const Shape& s, int w, int* first, int* last) const {
    int f = 0, l = chunks<CB>() - 1;
    while (l >= 0 && !active<CB>(s, w, l)) --l;
    while (f <= l && !active<CB>(s, w, f)) ++f;
    *first = f;
    *last = l;
  }
};

__device__ __forceinline__ Item make_item(const Shape& s, const TileGrid& g, int64_t item) {
  Item it;
  const int64_t bh = item / g.items_per_head;
  const int pair = static_cast<int>(item - bh * g.items_per_head);
  it.b = static_cast<int>(bh / s.hk);
  it.kvh = static_cast<int>(bh - static_cast<int64_t>(it.b) * s.hk);
  it.kv_len = kv_len_of(s, it.b);
  for (int w = 0; w < 2; ++w) {
    it.t0[w] = min((2 * pair + w) * g.tt, s.m);
    it.t1[w] = min((2 * pair + w + 1) * g.tt, s.m);
  }
  it.r = key_range(s, it.t0[0], max(it.t1[0], it.t1[1]), it.kv_len);
  return it;
}

}  // namespace win
}  // namespace dsa
