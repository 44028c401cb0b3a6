// Host side shared by the windowed-attention entry points: argument checks and
// the tensor maps of strided q / k / v.
#pragma once

#include "host_util.h"
#include "window_common.cuh"

namespace dsa {
namespace win {

// Strides in elements of [batch, tokens, heads, head_dim] (head_dim contiguous).
struct Strides {
  int64_t b = 0, t = 0, h = 0;
};

struct Tensors {
  const void* q = nullptr;
  const void* k = nullptr;
  const void* v = nullptr;
  Strides qs, ks, vs;
};

inline bool same_strides(const Strides& a, const Strides& b) {
  return a.b == b.b && a.t == b.t && a.h == b.h;
}

// Strides given by the caller (null: contiguous). The stride of an extent of at
// most one element is never stepped over, so any value of it is replaced.
// DSA_ERR_MISALIGNED where a stride breaks the 16-byte rule of the tensor maps.
inline int read_strides(const int64_t* given, int64_t batch, int64_t tokens, int heads, int d,
                        Strides* out) {
  Strides s;
  s.h = d;
  s.t = static_cast<int64_t>(heads) * d;
  s.b = tokens * s.t;
  if (given != nullptr && batch > 0 && tokens > 0) {
    if (batch > 1) s.b = given[0];
    if (tokens > 1) s.t = given[1];
    if (heads > 1) s.h = given[2];
  }
  if (s.b <= 0) s.b = s.t;  // no token: nothing is stepped over
  for (const int64_t x : {s.b, s.t, s.h}) {
    if (x <= 0 || x >= (int64_t{1} << 38)) return DSA_ERR_UNSUPPORTED;
    if (x % 8 != 0) return DSA_ERR_MISALIGNED;
  }
  *out = s;
  return DSA_OK;
}

inline CUtensorMapDataType map_type(uint32_t fmt) {
  return fmt == Bf16::kFmt ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
}

// Box of `tt` tokens x `g` heads x 64 columns: the rows of a (token, head) tile.
inline int map_rows_by_head(CUtensorMap* tm, uint32_t fmt, const void* base, const Strides& s,
                            int64_t batch, int64_t tokens, int heads, int d, int g, int tt) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(heads),
                            static_cast<uint64_t>(tokens), static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {static_cast<uint64_t>(s.h) * 2, static_cast<uint64_t>(s.t) * 2,
                               static_cast<uint64_t>(s.b) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(g), static_cast<uint32_t>(tt), 1};
  return encode_tensor_map(tm, map_type(fmt), 4, base, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}

// Box of `rows` tokens of one head x 64 columns.
inline int map_head_by_rows(CUtensorMap* tm, uint32_t fmt, const void* base, const Strides& s,
                            int64_t batch, int64_t tokens, int heads, int d, int rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(tokens > 0 ? tokens : 1),
                            static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  const uint64_t strides[3] = {static_cast<uint64_t>(s.t) * 2, static_cast<uint64_t>(s.h) * 2,
                               static_cast<uint64_t>(s.b) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
  return encode_tensor_map(tm, map_type(fmt), 4, base, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}

// False when the items do not fit 31 bits.
inline bool tile_grid(const Shape& s, int64_t batch, TileGrid* g) {
  g->tt = kRows / s.g;
  g->items_per_head = ((s.m + g->tt - 1) / g->tt + 1) / 2;
  const int64_t items = batch * s.hk * g->items_per_head;
  g->items = static_cast<int>(items);
  return items <= 0x7FFFFF00;
}

// Checks shared by the forward and the backward; fills `x` and `s`.
inline int check_window_args(const void* q, const int64_t* q_strides, const void* k,
                             const int64_t* k_strides, const void* v, const int64_t* v_strides,
                             const int* kv_lens, int dtype, int64_t batch, int64_t m, int64_t n,
                             int n_heads, int n_kv_heads, int head_dim, int64_t window,
                             int64_t n_first, float softmax_scale, Tensors* x, Shape* s) {
  if (batch < 0 || m < 0 || n < 0 || n_heads < 1 || n_kv_heads < 1 || window < 1 || n_first < 0)
    return DSA_ERR_INVALID_ARGUMENT;
  if (n_heads % n_kv_heads != 0) return DSA_ERR_INVALID_ARGUMENT;
  if (!(softmax_scale > 0.f) || softmax_scale > 3.0e38f) return DSA_ERR_INVALID_ARGUMENT;
  if (dtype != DSA_DTYPE_BF16 && dtype != DSA_DTYPE_FP16) return DSA_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return DSA_ERR_UNSUPPORTED;
  if (n_heads / n_kv_heads > 128) return DSA_ERR_UNSUPPORTED;
  constexpr int64_t kMaxLen = int64_t{1} << 28;  // positions and their sums stay in 32 bits
  if (m > kMaxLen || n > kMaxLen || batch > (1 << 24) || n_heads > (1 << 20))
    return DSA_ERR_UNSUPPORTED;
  if (batch > 0 && m > 0 && (q == nullptr || (n > 0 && (k == nullptr || v == nullptr))))
    return DSA_ERR_INVALID_ARGUMENT;
  if (n == 0) k = v = q;  // nothing is read; the tensor maps want an address
  if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return DSA_ERR_MISALIGNED;
  x->q = q;
  x->k = k;
  x->v = v;
  int st = read_strides(q_strides, batch, m, n_heads, head_dim, &x->qs);
  if (st == DSA_OK) st = read_strides(k_strides, batch, n, n_kv_heads, head_dim, &x->ks);
  if (st == DSA_OK) st = read_strides(v_strides, batch, n, n_kv_heads, head_dim, &x->vs);
  if (st != DSA_OK) return st;
  s->m = static_cast<int>(m);
  s->n = static_cast<int>(n);
  s->h = n_heads;
  s->hk = n_kv_heads;
  s->g = n_heads / n_kv_heads;
  s->window = static_cast<int>(window < n ? window : (n > 0 ? n : 1));
  s->n_first = static_cast<int>(n_first < n ? n_first : n);
  s->kv_lens = kv_lens;
  return DSA_OK;
}

}  // namespace win
}  // namespace dsa
