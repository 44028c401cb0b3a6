// Writing new rows into a paged key-value cache, and eviction from it by
// accumulated attention weight, for sm_100a (layout: dsa_b200.h).
//
// Eviction keeps, of a sequence of len rows and a budget of B: all rows when len <= B;
// else the first n_first, the last n_recent, and of those between the
// B - n_first - n_recent with the largest weights, ties to the lowest index. The kept
// rows move in ascending order to rows 0, 1, ... of fresh pages: the old pages stay as
// they are (other sequences may share them), and nothing is read after it was
// overwritten.
//   evict_select_kernel  a block per sequence: radix select of the threshold over the
//                        32 bits of the orderable weight, then one ordered pass
//   evict_copy_kernel    rows and weights to their new slots, HBM bound
#include "host_util.h"

namespace dsa {
namespace cache {

struct Pool {
  uint8_t* k;
  uint8_t* v;            // null: one tensor for both
  int64_t ks[3], vs[3];  // (page, slot, head) strides in bytes
  float* weights;        // [num_pages, page] or null
  int64_t num_pages;
  int page, hk, row16;   // row16: 16-byte units of one head's row
  unsigned int* err;
};

__device__ __forceinline__ int lookup(const Pool& p, const int* table, int64_t max_pages, int64_t b,
                                      int64_t row) {
  const int page = __ldg(table + b * max_pages + row / p.page);
  return page >= 0 && page < p.num_pages ? page : -1;
}

// ------------------------------------------------------------------ append
struct AppendParams {
  Pool pool;
  const uint8_t* k;
  const uint8_t* v;
  int64_t ks[3], vs[3];  // (batch, token, head) strides in bytes
  const int* table;
  const int* start;
  int64_t max_pages;
  int64_t batch, t;
};

// A thread per 16-byte unit of a row; blockIdx.y: K or V.
__global__ void __launch_bounds__(256) cache_append_kernel(const AppendParams p) {
  const int units = p.pool.hk * p.pool.row16;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int64_t r = i / units;
  if (r >= p.batch * p.t) return;
  const int u = static_cast<int>(i - r * units);
  const int64_t b = r / p.t, t = r - b * p.t;
  const int64_t row = static_cast<int64_t>(__ldg(p.start + b)) + t;
  const bool room = row >= 0 && row < p.max_pages * p.pool.page;
  const int page = room ? lookup(p.pool, p.table, p.max_pages, b, row) : -1;
  if (page < 0) {
    if (u == 0) atomicOr(p.pool.err, DSA_DEVERR_CACHE);
    return;
  }
  const int slot = static_cast<int>(row % p.pool.page);
  const int head = u / p.pool.row16, x = u - head * p.pool.row16;
  const bool second = blockIdx.y == 1;
  const int64_t* ss = second ? p.vs : p.ks;
  const int64_t* ds = second ? p.pool.vs : p.pool.ks;
  const uint8_t* src = (second ? p.v : p.k) + b * ss[0] + t * ss[1] + head * ss[2] + x * 16;
  uint8_t* dst =
      (second ? p.pool.v : p.pool.k) + page * ds[0] + slot * ds[1] + head * ds[2] + x * 16;
  *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(src);
  if (u == 0 && !second && p.pool.weights != nullptr)
    p.pool.weights[static_cast<int64_t>(page) * p.pool.page + slot] = 0.f;
}

// ------------------------------------------------------------------ evict
struct EvictParams {
  Pool pool;
  const int* table;      // [batch, max_pages]
  const int* lens;       // [batch]
  const int* dst_table;  // [batch, dst_pages]
  int64_t max_pages, dst_pages;
  int budget, n_first, n_recent;
  int* kept;             // [batch, budget]: kept rows ascending, then -1
  int* new_lens;         // [batch]
};

constexpr int kSelThreads = 1024;
constexpr int kSelWarps = kSelThreads / 32;

// Orderable bits of a weight: larger weights have larger bits, NaN the largest.
__device__ __forceinline__ uint32_t order_bits(float w) {
  if (isnan(w)) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 and +0 are one value
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  __shared__ int hist[256];
  __shared__ int warp_gt[kSelWarps], warp_eq[kSelWarps];
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_need;
  const int b = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t room = p.max_pages * p.pool.page;
  int len = __ldg(p.lens + b);
  if (tid == 0 && (len < 0 || len > room)) atomicOr(p.pool.err, DSA_DEVERR_CACHE);
  len = max(len, 0);
  if (len > room) len = static_cast<int>(room);
  int* kept = p.kept + static_cast<int64_t>(b) * p.budget;
  const int left = min(len, p.budget);
  if (tid == 0) p.new_lens[b] = left;
  for (int i = left + tid; i < p.budget; i += kSelThreads) kept[i] = -1;
  if (len <= p.budget) {
    for (int i = tid; i < len; i += kSelThreads) kept[i] = i;
    return;
  }
  const int a = p.n_first, e = len - p.n_recent;  // the rows between, e - a > need >= 0
  for (int i = tid; i < a; i += kSelThreads) kept[i] = i;
  for (int i = tid; i < p.n_recent; i += kSelThreads) kept[p.budget - p.n_recent + i] = e + i;
  int need = p.budget - p.n_first - p.n_recent;
  if (need == 0) return;
  // an entry of the table that names no page: its rows rank below every weight
  auto bits_of = [&](int row) -> uint32_t {
    const int page = lookup(p.pool, p.table, p.max_pages, b, row);
    return page < 0 ? 0u
                    : order_bits(p.pool.weights[static_cast<int64_t>(page) * p.pool.page +
                                                row % p.pool.page]);
  };
  // ---- the need-th largest value, a byte a pass from the top
  uint32_t prefix = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < 256; i += kSelThreads) hist[i] = 0;
    __syncthreads();
    for (int i0 = a; i0 < e; i0 += kSelThreads) {
      const int row = i0 + tid;
      bool in = row < e;
      uint32_t u = 0;
      if (in) {
        u = bits_of(row);
        in = shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8));
      }
      const uint32_t live = __ballot_sync(0xFFFFFFFFu, in);
      if (in) {
        // one add per distinct byte of the warp: many weights are alike
        const uint32_t digit = (u >> shift) & 255u;
        const uint32_t same = __match_any_sync(live, digit);
        if (lane == __ffs(same) - 1) atomicAdd(&hist[digit], __popc(same));
      }
    }
    __syncthreads();
    if (warp == 0) {
      // lane l holds digits 255 - 8 l down to 248 - 8 l
      int c[8], sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        c[k] = hist[255 - 8 * lane - k];
        sum += c[k];
      }
      int incl = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, incl, o);
        if (lane >= o) incl += y;
      }
      int above = incl - sum;
      if (above < need && incl >= need) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          if (above < need && above + c[k] >= need) {
            sh_prefix = prefix | static_cast<uint32_t>(255 - 8 * lane - k) << shift;
            sh_need = need - above;
            above = need;  // found
          } else {
            above += c[k];
          }
        }
      }
    }
    __syncthreads();
    prefix = sh_prefix;
    need = sh_need;  // rows equal to the prefix that are still to be taken
  }
  // ---- rows above the threshold and the first `need` equal to it, in order: a warp a
  // contiguous stretch
  const int n = e - a;
  const int stretch = (n + kSelWarps - 1) / kSelWarps;
  const int w0 = min(warp * stretch, n), w1 = min(w0 + stretch, n);
  int gt = 0, eq = 0;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const bool in = i0 + lane < w1;
    const uint32_t u = in ? bits_of(a + i0 + lane) : 0u;
    gt += __popc(__ballot_sync(0xFFFFFFFFu, in && u > prefix));
    eq += __popc(__ballot_sync(0xFFFFFFFFu, in && u == prefix));
  }
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  gt = eq = 0;
  for (int i = 0; i < warp; ++i) {
    gt += warp_gt[i];
    eq += warp_eq[i];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const bool in = i0 + lane < w1;
    const uint32_t u = in ? bits_of(a + i0 + lane) : 0u;
    const uint32_t mg = __ballot_sync(0xFFFFFFFFu, in && u > prefix);
    const uint32_t me = __ballot_sync(0xFFFFFFFFu, in && u == prefix);
    const int g = gt + __popc(mg & below), q = eq + __popc(me & below);
    if (in && (u > prefix || (u == prefix && q < need))) kept[a + g + min(q, need)] = a + i0 + lane;
    gt += __popc(mg);
    eq += __popc(me);
  }
}

constexpr int kCopyThreads = 256;

// A block copies kCopyRows rows of a sequence's fresh pages, K and V, and their weights.
constexpr int kCopyRows = 16;

__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const EvictParams p) {
  __shared__ int64_t src_at[2][kCopyRows], dst_at[2][kCopyRows];  // byte offsets, -1: no copy
  const int b = blockIdx.y;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kCopyRows;
  const int left = p.new_lens[b];
  if (threadIdx.x < kCopyRows) {
    const int64_t row = r0 + threadIdx.x;
    int64_t s[2] = {-1, -1}, d[2] = {-1, -1};
    if (row < p.dst_pages * p.pool.page) {
      const int dp = lookup(p.pool, p.dst_table, p.dst_pages, b, row);
      const int ds = static_cast<int>(row % p.pool.page);
      float weight = 0.f;
      int sp = -1;
      if (row < left) {
        const int from = p.kept[static_cast<int64_t>(b) * p.budget + row];
        sp = lookup(p.pool, p.table, p.max_pages, b, from);
        const int ss = from % p.pool.page;
        if (sp < 0 || dp < 0) {
          atomicOr(p.pool.err, DSA_DEVERR_CACHE);
        } else {
          s[0] = sp * p.pool.ks[0] + ss * p.pool.ks[1];
          s[1] = sp * p.pool.vs[0] + ss * p.pool.vs[1];
          d[0] = dp * p.pool.ks[0] + ds * p.pool.ks[1];
          d[1] = dp * p.pool.vs[0] + ds * p.pool.vs[1];
          weight = p.pool.weights[static_cast<int64_t>(sp) * p.pool.page + ss];
        }
      }
      if (dp >= 0) p.pool.weights[static_cast<int64_t>(dp) * p.pool.page + ds] = weight;
    }
    for (int k = 0; k < 2; ++k) {
      src_at[k][threadIdx.x] = s[k];
      dst_at[k][threadIdx.x] = d[k];
    }
  }
  __syncthreads();
  const int units = p.pool.hk * p.pool.row16;
  const int kinds = p.pool.v == nullptr ? 1 : 2;
  constexpr int kAhead = 8;  // loads in flight per thread
  const int total = kinds * kCopyRows * units;
  for (int i0 = threadIdx.x; i0 < total; i0 += kCopyThreads * kAhead) {
    uint4 x[kAhead];
    uint8_t* to[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kCopyThreads;
      to[k] = nullptr;
      if (i < total) {
        const int kind = i / (kCopyRows * units);
        const int y = i - kind * kCopyRows * units;
        const int row = y / units, u = y - row * units;
        const int head = u / p.pool.row16;
        const int64_t at = (kind ? p.pool.vs[2] : p.pool.ks[2]) * head + (u - head * p.pool.row16) * 16;
        uint8_t* base = kind ? p.pool.v : p.pool.k;
        if (src_at[kind][row] >= 0) {
          x[k] = *reinterpret_cast<const uint4*>(base + src_at[kind][row] + at);
          to[k] = base + dst_at[kind][row] + at;
        }
      }
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k)
      if (to[k] != nullptr) *reinterpret_cast<uint4*>(to[k]) = x[k];
  }
}

// ------------------------------------------------------------------ host
// Byte strides of a [a, b, heads, d] tensor of 2-byte elements; `given` in elements.
inline int byte_strides(const int64_t* given, int64_t a, int64_t b, int heads, int d, int64_t* out) {
  int64_t s[3] = {b * heads * d, static_cast<int64_t>(heads) * d, d};
  if (given != nullptr) {
    if (a > 1) s[0] = given[0];
    if (b > 1) s[1] = given[1];
    if (heads > 1) s[2] = given[2];
  }
  for (int i = 0; i < 3; ++i) {
    if (s[i] < 0 || s[i] >= (int64_t{1} << 38)) return DSA_ERR_UNSUPPORTED;
    if (s[i] % 8 != 0) return DSA_ERR_MISALIGNED;
    out[i] = s[i] * 2;
  }
  return DSA_OK;
}

inline int make_pool(void* k, const int64_t* k_strides, void* v, const int64_t* v_strides,
                     float* weights, int64_t num_pages, int64_t page, int heads, int d, Pool* p) {
  if (num_pages < 1 || page < 1 || heads < 1) return DSA_ERR_INVALID_ARGUMENT;
  if (d < 8 || d % 8 != 0 || d > 1024 || heads > 4096 || page > (1 << 20) || num_pages > 0x7FFFFFFF)
    return DSA_ERR_UNSUPPORTED;
  if (!aligned16(k) || !aligned16(v)) return DSA_ERR_MISALIGNED;
  p->k = static_cast<uint8_t*>(k);
  p->v = static_cast<uint8_t*>(v);
  int st = byte_strides(k_strides, num_pages, page, heads, d, p->ks);
  if (st == DSA_OK) st = byte_strides(v != nullptr ? v_strides : k_strides, num_pages, page, heads, d, p->vs);
  if (st != DSA_OK) return st;
  p->weights = weights;
  p->num_pages = num_pages;
  p->page = static_cast<int>(page);
  p->hk = heads;
  p->row16 = d / 8;
  return DSA_OK;
}

}  // namespace cache
}  // namespace dsa

extern "C" int dsa_cache_append(const void* k, const int64_t* k_strides, const void* v,
                                const int64_t* v_strides, void* k_pages, const int64_t* kp_strides,
                                void* v_pages, const int64_t* vp_strides, float* weights,
                                const int* block_table, const int* start, int64_t batch, int64_t t,
                                int n_kv_heads, int head_dim, int64_t num_pages, int64_t page_size,
                                int64_t max_pages, void* stream) {
  using namespace dsa;
  using namespace dsa::cache;
  if (batch < 0 || t < 0 || max_pages < 1) return DSA_ERR_INVALID_ARGUMENT;
  if ((v == nullptr) != (v_pages == nullptr)) return DSA_ERR_INVALID_ARGUMENT;
  AppendParams p;
  int st = make_pool(k_pages, kp_strides, v_pages, vp_strides, weights, num_pages, page_size,
                     n_kv_heads, head_dim, &p.pool);
  if (st != DSA_OK) return st;
  if (batch == 0 || t == 0) return DSA_OK;
  if (k == nullptr || k_pages == nullptr || block_table == nullptr || start == nullptr)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(k) || !aligned16(v)) return DSA_ERR_MISALIGNED;
  st = byte_strides(k_strides, batch, t, n_kv_heads, head_dim, p.ks);
  if (st == DSA_OK)
    st = byte_strides(v != nullptr ? v_strides : k_strides, batch, t, n_kv_heads, head_dim, p.vs);
  if (st != DSA_OK) return st;
  if (batch > (1 << 28) || t > (1 << 28) || max_pages > (int64_t{1} << 28))
    return DSA_ERR_UNSUPPORTED;
  const int64_t work = batch * t * n_kv_heads * (head_dim / 8);
  const int64_t blocks = (work + 255) / 256;
  if (blocks > 0x7FFFFFFF) return DSA_ERR_UNSUPPORTED;
  p.k = static_cast<const uint8_t*>(k);
  p.v = static_cast<const uint8_t*>(v);
  p.table = block_table;
  p.start = start;
  p.max_pages = max_pages;
  p.batch = batch;
  p.t = t;
  st = device_error_word(&p.pool.err);
  if (st != DSA_OK) return st;
  cache_append_kernel<<<dim3(static_cast<unsigned>(blocks), v != nullptr ? 2 : 1), 256, 0,
                        static_cast<cudaStream_t>(stream)>>>(p);
  return cuda_status(cudaGetLastError());
}

extern "C" int dsa_cache_evict(void* k_pages, const int64_t* kp_strides, void* v_pages,
                               const int64_t* vp_strides, float* weights, const int* block_table,
                               const int* lens, const int* dst_table, int* kept, int* new_lens,
                               int64_t batch, int n_kv_heads, int head_dim, int64_t num_pages,
                               int64_t page_size, int64_t max_pages, int64_t dst_pages,
                               int64_t budget, int64_t n_first, int64_t n_recent, void* stream) {
  using namespace dsa;
  using namespace dsa::cache;
  if (batch < 0 || max_pages < 1 || dst_pages < 1 || budget < 1 || n_first < 0 || n_recent < 0 ||
      n_first > budget || n_recent > budget - n_first)
    return DSA_ERR_INVALID_ARGUMENT;
  EvictParams p;
  int st = make_pool(k_pages, kp_strides, v_pages, vp_strides, weights, num_pages, page_size,
                     n_kv_heads, head_dim, &p.pool);
  if (st != DSA_OK) return st;
  if (max_pages > (int64_t{1} << 28) || dst_pages > (int64_t{1} << 28) ||
      max_pages * page_size > (int64_t{1} << 28) || dst_pages * page_size > (int64_t{1} << 28) ||
      batch > 65535)
    return DSA_ERR_UNSUPPORTED;
  if (budget > dst_pages * page_size) return DSA_ERR_INVALID_ARGUMENT;  // the kept rows do not fit
  if (batch == 0) return DSA_OK;
  if (k_pages == nullptr || weights == nullptr || block_table == nullptr || lens == nullptr ||
      dst_table == nullptr || kept == nullptr || new_lens == nullptr)
    return DSA_ERR_INVALID_ARGUMENT;
  p.table = block_table;
  p.lens = lens;
  p.dst_table = dst_table;
  p.max_pages = max_pages;
  p.dst_pages = dst_pages;
  p.budget = static_cast<int>(budget);
  p.n_first = static_cast<int>(n_first);
  p.n_recent = static_cast<int>(n_recent);
  p.kept = kept;
  p.new_lens = new_lens;
  st = device_error_word(&p.pool.err);
  if (st != DSA_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  evict_select_kernel<<<static_cast<unsigned>(batch), kSelThreads, 0, cs>>>(p);
  st = cuda_status(cudaGetLastError());
  if (st != DSA_OK) return st;
  const int64_t blocks = (dst_pages * page_size + kCopyRows - 1) / kCopyRows;
  evict_copy_kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(batch)), kCopyThreads,
                      0, cs>>>(p);
  return cuda_status(cudaGetLastError());
}
