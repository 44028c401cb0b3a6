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

}  // namespace win
}  // namespace dsa
