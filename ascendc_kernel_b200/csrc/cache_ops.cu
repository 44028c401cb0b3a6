// Writing new rows into a paged key-value cache, and eviction from it by
// accumulated attention weight, for sm_100a (layout: dsa_b200.h).
//
// Eviction keeps, of a sequence of len rows and a budget of B: all rows when len <= B;
// else the first n_first, the last n_recent, and of those between the
// B - n_first - n_recent with the largest weights, ties to the lowest index. The kept
// rows move in ascending order to rows 0, 1, ... of fresh pages: the old pages stay as
// they are (other sequences may share them), and nothing is read after it was
// overwritten.
//   evict_select_kernel  a cluster per sequence: radix select of the threshold over the
//                        32 bits of the orderable weight, then one ordered pass
//   evict_copy_kernel    rows and weights to their new slots, HBM bound
//
// Measured (bf16, 8 kv heads of 128, K and V): evicting 32 sequences of up to 16,384 rows
// to 4,096 each takes 188 us for 1.04 GB, select 19 and copy 168 (6.2 TB/s, 0.95 of a
// copy); one sequence of 2,600 rows of one head to 1,024, 19 us, of which the GPU works
// for 12. Appending 4 x 4096 rows: 24 us for 134 MB (5.6 TB/s; each launch's start and end
// are 4 us of it); one row each of 64 sequences: 3 us on the GPU, 12 with the call.
#include <cooperative_groups.h>

#include "common.cuh"
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

// ------------------------------------------------------------------ row copies
constexpr int kCopyThreads = 256;
constexpr int kAhead = 8;       // 16-byte loads in flight per thread
constexpr int kCopyRows = 16;   // rows of a block, at most

// Byte offsets of one row's source and target in K and V; -1: the row is not copied.
struct RowPlan {
  int64_t src[2][kCopyRows], dst[2][kCopyRows];
};

struct RowCopy {
  const uint8_t* src[2];  // K, V
  uint8_t* dst[2];
  int64_t src_head[2], dst_head[2];  // bytes from head to head
  int kinds, rows;        // tensors; rows of the block
  int units, row16;       // 16-byte units of a row (all heads) and of a head
  uint32_t magic_units, magic_row16;  // floor(2^32 / x) + 1
};

// i / x for i * x < 2^32, from magic = floor(2^32 / x) + 1 (x > 1; x = 1: magic 0)
__host__ __device__ __forceinline__ uint32_t div_magic(uint32_t x) {
  return x == 1 ? 0u : 0xFFFFFFFFu / x + 1u;
}
__device__ __forceinline__ uint32_t div_by(uint32_t i, uint32_t magic) {
  return magic == 0u ? i : __umulhi(i, magic);
}

// The block's rows, a thread 16 bytes at a time with kAhead loads in flight, units of a
// row on neighbouring threads. Flat: a row's heads follow one another without a gap on
// both sides, so a unit's offset is its number.
template <bool Flat>
__device__ __forceinline__ void copy_rows(const RowCopy& c, const RowPlan& plan) {
  const int total = c.rows * c.units;
  for (int kind = 0; kind < c.kinds; ++kind) {
    const uint8_t* src = c.src[kind];
    uint8_t* dst = c.dst[kind];
    for (int i0 = threadIdx.x; i0 < total; i0 += kCopyThreads * kAhead) {
      uint4 x[kAhead];
      int64_t to[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int i = i0 + k * kCopyThreads;
        to[k] = -1;
        if (i < total) {
          const int row = static_cast<int>(div_by(i, c.magic_units));
          const int u = i - row * c.units;
          const int64_t from = plan.src[kind][row];
          if (from >= 0) {
            int64_t a = u * 16, b = u * 16;
            if (!Flat) {
              const int head = static_cast<int>(div_by(u, c.magic_row16));
              a = head * c.src_head[kind] + (u - head * c.row16) * 16;
              b = head * c.dst_head[kind] + (u - head * c.row16) * 16;
            }
            x[k] = __ldcs(reinterpret_cast<const uint4*>(src + from + a));
            to[k] = plan.dst[kind][row] + b;
          }
        }
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k)
        if (to[k] >= 0) *reinterpret_cast<uint4*>(dst + to[k]) = x[k];
    }
  }
}

// Rows of a block: few enough that the call fills the thread slots of a full GPU (148 SMs of 8
// blocks) about twice, one at least.
inline int rows_per_block(int64_t rows) {
  const int64_t r = rows / (2 * 148 * 8);
  return static_cast<int>(r < 1 ? 1 : (r > kCopyRows ? kCopyRows : r));
}

// ------------------------------------------------------------------ append
struct AppendParams {
  Pool pool;
  RowCopy copy;
  int64_t ks[2], vs[2];  // (batch, token) strides of the new rows in bytes
  const int* table;
  const int* start;
  int64_t max_pages;
  int64_t batch, t;
};

template <bool Flat>
__global__ void __launch_bounds__(kCopyThreads) cache_append_kernel(const AppendParams p) {
  __shared__ RowPlan plan;
  if (threadIdx.x < p.copy.rows) {
    const int64_t r = static_cast<int64_t>(blockIdx.x) * p.copy.rows + threadIdx.x;
    int64_t s[2] = {-1, -1}, d[2] = {-1, -1};
    if (r < p.batch * p.t) {
      const int64_t b = r / p.t, t = r - b * p.t;
      const int64_t row = static_cast<int64_t>(__ldg(p.start + b)) + t;
      const bool room = row >= 0 && row < p.max_pages * p.pool.page;
      const int64_t page = room ? lookup(p.pool, p.table, p.max_pages, b, row) : -1;
      if (page < 0) {
        atomicOr(p.pool.err, DSA_DEVERR_CACHE);
      } else {
        const int64_t slot = row % p.pool.page;
        s[0] = b * p.ks[0] + t * p.ks[1];
        s[1] = b * p.vs[0] + t * p.vs[1];
        d[0] = page * p.pool.ks[0] + slot * p.pool.ks[1];
        d[1] = page * p.pool.vs[0] + slot * p.pool.vs[1];
        if (p.pool.weights != nullptr) p.pool.weights[page * p.pool.page + slot] = 0.f;
      }
    }
    for (int k = 0; k < 2; ++k) {
      plan.src[k][threadIdx.x] = s[k];
      plan.dst[k][threadIdx.x] = d[k];
    }
  }
  __syncthreads();
  copy_rows<Flat>(p.copy, plan);
}

// ------------------------------------------------------------------ evict
struct EvictParams {
  Pool pool;
  RowCopy copy;
  const int* table;      // [batch, max_pages]
  const int* lens;       // [batch]
  const int* dst_table;  // [batch, dst_pages]
  int64_t max_pages, dst_pages;
  int budget, n_first, n_recent;
  int* kept;             // [batch, budget]: kept rows ascending, then -1
  int* new_lens;         // [batch]
  int staged;            // rows of the select kernel's shared memory
};

constexpr int kSelThreads = 512;
constexpr int kSelWarps = kSelThreads / 32;
constexpr int kSelMaxCluster = 8;
constexpr int kSelStaged = 48 * 1024;  // rows of a block whose weights fit in shared memory

// Orderable bits of a weight: larger weights have larger bits, NaN the largest.
__device__ __forceinline__ uint32_t order_bits(float w) {
  if (isnan(w)) return 0xFFFFFFFFu;
  const uint32_t u = __float_as_uint(w + 0.0f);  // -0 and +0 are one value
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// A cluster of 1, 2, 4 or 8 blocks per sequence (select_cluster), each with a contiguous
// stretch of its rows. Latency bound: the weights are read once through the table and
// staged; each pass is a few shared-memory atomics per thread, one cluster barrier and
// the sum of the blocks' 256 counts over distributed shared memory.
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictParams p) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  __shared__ int hist[2][256];  // passes alternate, so one barrier a pass is enough
  __shared__ int total[256];
  __shared__ int warp_gt[kSelWarps], warp_eq[kSelWarps];
  __shared__ int block_gt, block_eq;
  __shared__ uint32_t sh_prefix;
  __shared__ int sh_need;
  extern __shared__ uint32_t staged[];
  const int blocks = static_cast<int>(cluster.num_blocks());
  const int rank = static_cast<int>(cluster.block_rank());
  const int b = blockIdx.x / blocks;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int ctid = rank * kSelThreads + tid, cthreads = blocks * kSelThreads;
  const int64_t room = p.max_pages * p.pool.page;
  int len = __ldg(p.lens + b);
  if (ctid == 0 && (len < 0 || len > room)) atomicOr(p.pool.err, DSA_DEVERR_CACHE);
  len = max(len, 0);
  if (len > room) len = static_cast<int>(room);
  int* kept = p.kept + static_cast<int64_t>(b) * p.budget;
  const int left = min(len, p.budget);
  if (ctid == 0) p.new_lens[b] = left;
  for (int i = left + ctid; i < p.budget; i += cthreads) kept[i] = -1;
  if (len <= p.budget) {
    for (int i = ctid; i < len; i += cthreads) kept[i] = i;
    return;
  }
  const int e = len - p.n_recent;  // rows [n_first, e) compete; more than need >= 0
  for (int i = ctid; i < p.n_first; i += cthreads) kept[i] = i;
  for (int i = ctid; i < p.n_recent; i += cthreads) kept[p.budget - p.n_recent + i] = e + i;
  int need = p.budget - p.n_first - p.n_recent;
  if (need == 0) return;
  // this block's rows: [a, a + n)
  const int64_t all = e - p.n_first;
  const int a = p.n_first + static_cast<int>(all * rank / blocks);
  const int n = p.n_first + static_cast<int>(all * (rank + 1) / blocks) - a;
  // an entry of the table that names no page: its rows rank below every weight
  auto read = [&](int i) -> uint32_t {
    const int row = a + i;
    const int page = lookup(p.pool, p.table, p.max_pages, b, row);
    return page < 0 ? 0u
                    : order_bits(p.pool.weights[static_cast<int64_t>(page) * p.pool.page +
                                                row % p.pool.page]);
  };
  // the weights are read once through the table, and the passes below run on the copy; a
  // stretch that does not fit is read again in each pass
  const bool whole = n <= p.staged;
  if (whole) {
    for (int i0 = tid; i0 < n; i0 += 8 * kSelThreads) {
      uint32_t u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = i0 + k * kSelThreads < n ? read(i0 + k * kSelThreads) : 0u;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (i0 + k * kSelThreads < n) staged[i0 + k * kSelThreads] = u[k];
    }
  }
  auto bits_of = [&](int i) -> uint32_t { return whole ? staged[i] : read(i); };
  for (int i = tid; i < 512; i += kSelThreads) (&hist[0][0])[i] = 0;
  __syncthreads();
  // ---- the need-th largest value, a byte a pass from the top
  uint32_t prefix = 0;
  for (int shift = 24, pass = 0; shift >= 0; shift -= 8, ++pass) {
    int* mine = hist[pass & 1];
    for (int i0 = 0; i0 < n; i0 += kSelThreads) {
      const int i = i0 + tid;
      bool in = i < n;
      uint32_t u = 0;
      if (in) {
        u = bits_of(i);
        in = shift == 24 || (u >> (shift + 8)) == (prefix >> (shift + 8));
      }
      const uint32_t live = __ballot_sync(0xFFFFFFFFu, in);
      if (in) {
        // many weights are alike: a warp whose rows share the byte adds once
        const uint32_t digit = (u >> shift) & 255u;
        int same;
        __match_all_sync(live, digit, &same);
        if (!same)
          atomicAdd(&mine[digit], 1);
        else if (lane == __ffs(live) - 1)
          atomicAdd(&mine[digit], __popc(live));
      }
    }
    cluster.sync();
    for (int i = tid; i < 256; i += kSelThreads) {
      int sum = 0;
      for (int r = 0; r < blocks; ++r) sum += cluster.map_shared_rank(mine, r)[i];
      total[i] = sum;
      // the other buffer was read before this barrier; the next pass counts into it
      hist[(pass & 1) ^ 1][i] = 0;
    }
    __syncthreads();
    if (warp == 0) {
      // lane l holds digits 255 - 8 l down to 248 - 8 l
      int c[8], sum = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        c[k] = total[255 - 8 * lane - k];
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
  const int stretch = (n + kSelWarps - 1) / kSelWarps;
  const int w0 = min(warp * stretch, n), w1 = min(w0 + stretch, n);
  int gt = 0, eq = 0;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const bool in = i0 + lane < w1;
    const uint32_t u = in ? bits_of(i0 + lane) : 0u;
    gt += __popc(__ballot_sync(0xFFFFFFFFu, in && u > prefix));
    eq += __popc(__ballot_sync(0xFFFFFFFFu, in && u == prefix));
  }
  if (lane == 0) {
    warp_gt[warp] = gt;
    warp_eq[warp] = eq;
  }
  __syncthreads();
  if (warp == 0) {
    const int g = __reduce_add_sync(0xFFFFFFFFu, lane < kSelWarps ? warp_gt[lane] : 0);
    const int q = __reduce_add_sync(0xFFFFFFFFu, lane < kSelWarps ? warp_eq[lane] : 0);
    if (lane == 0) {
      block_gt = g;
      block_eq = q;
    }
  }
  cluster.sync();
  gt = eq = 0;
  for (int r = 0; r < rank; ++r) {
    gt += *cluster.map_shared_rank(&block_gt, r);
    eq += *cluster.map_shared_rank(&block_eq, r);
  }
  for (int i = 0; i < warp; ++i) {
    gt += warp_gt[i];
    eq += warp_eq[i];
  }
  const uint32_t below = (1u << lane) - 1u;
  for (int i0 = w0; i0 < w1; i0 += 32) {
    const bool in = i0 + lane < w1;
    const uint32_t u = in ? bits_of(i0 + lane) : 0u;
    const uint32_t mg = __ballot_sync(0xFFFFFFFFu, in && u > prefix);
    const uint32_t me = __ballot_sync(0xFFFFFFFFu, in && u == prefix);
    const int g = gt + __popc(mg & below), q = eq + __popc(me & below);
    if (in && (u > prefix || (u == prefix && q < need)))
      kept[p.n_first + g + min(q, need)] = a + i0 + lane;
    gt += __popc(mg);
    eq += __popc(me);
  }
  cluster.sync();  // no block leaves while another reads its counts
}

// Blocks of a sequence's cluster: a block per 1024 rows of the table's room, as long as
// all clusters fit the GPU (2 blocks an SM) at once.
inline int select_cluster(int64_t batch, int64_t room) {
  int c = 1;
  while (c < kSelMaxCluster && room > 1024 * c && batch * 2 * c <= 2 * 148) c *= 2;
  return c;
}

// A block copies copy.rows rows of a sequence's fresh pages, K and V, and their weights.
template <bool Flat>
__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const EvictParams p) {
  __shared__ RowPlan plan;
  const int b = blockIdx.y;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * p.copy.rows;
  grid_dependency_wait();
  if (threadIdx.x < p.copy.rows) {
    const int left = p.new_lens[b];
    const int64_t row = r0 + threadIdx.x;
    int64_t s[2] = {-1, -1}, d[2] = {-1, -1};
    if (row < p.dst_pages * p.pool.page) {
      const int64_t dp = lookup(p.pool, p.dst_table, p.dst_pages, b, row);
      const int64_t ds = row % p.pool.page;
      float weight = 0.f;
      if (row < left) {
        const int from = p.kept[static_cast<int64_t>(b) * p.budget + row];
        const int64_t sp = lookup(p.pool, p.table, p.max_pages, b, from);
        const int64_t ss = from % p.pool.page;
        if (sp < 0 || dp < 0) {
          atomicOr(p.pool.err, DSA_DEVERR_CACHE);
        } else {
          s[0] = sp * p.pool.ks[0] + ss * p.pool.ks[1];
          s[1] = sp * p.pool.vs[0] + ss * p.pool.vs[1];
          d[0] = dp * p.pool.ks[0] + ds * p.pool.ks[1];
          d[1] = dp * p.pool.vs[0] + ds * p.pool.vs[1];
          weight = p.pool.weights[sp * p.pool.page + ss];
        }
      }
      if (dp >= 0) p.pool.weights[dp * p.pool.page + ds] = weight;
    }
    for (int k = 0; k < 2; ++k) {
      plan.src[k][threadIdx.x] = s[k];
      plan.dst[k][threadIdx.x] = d[k];
    }
  }
  __syncthreads();
  copy_rows<Flat>(p.copy, plan);
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
  // rows of at most 16383 units keep the divisions of copy_rows exact
  if (d < 8 || d % 8 != 0 || d > 1024 || static_cast<int64_t>(heads) * (d / 8) > 16383 || page > (1 << 20) || num_pages > 0x7FFFFFFF)
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

// The pool's side of a copy of `rows` rows; the source is the caller's to fill in.
inline RowCopy row_copy(const Pool& p, int64_t rows) {
  RowCopy c;
  c.dst[0] = p.k;
  c.dst[1] = p.v;
  c.dst_head[0] = p.ks[2];
  c.dst_head[1] = p.vs[2];
  c.kinds = p.v != nullptr ? 2 : 1;
  c.rows = rows_per_block(rows);
  c.row16 = p.row16;
  c.units = p.hk * p.row16;
  c.magic_units = div_magic(c.units);
  c.magic_row16 = div_magic(c.row16);
  return c;
}

inline bool flat_rows(const RowCopy& c) {
  for (int k = 0; k < c.kinds; ++k)
    if (c.units != c.row16 && (c.src_head[k] != c.row16 * 16 || c.dst_head[k] != c.row16 * 16))
      return false;
  return true;
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
  int64_t ks[3], vs[3];
  st = byte_strides(k_strides, batch, t, n_kv_heads, head_dim, ks);
  if (st == DSA_OK)
    st = byte_strides(v != nullptr ? v_strides : k_strides, batch, t, n_kv_heads, head_dim, vs);
  if (st != DSA_OK) return st;
  if (batch > (1 << 28) || t > (1 << 28) || max_pages > (int64_t{1} << 28))
    return DSA_ERR_UNSUPPORTED;
  for (int i = 0; i < 2; ++i) {
    p.ks[i] = ks[i];
    p.vs[i] = vs[i];
  }
  p.copy = row_copy(p.pool, batch * t);
  p.copy.src[0] = static_cast<const uint8_t*>(k);
  p.copy.src[1] = static_cast<const uint8_t*>(v);
  p.copy.src_head[0] = ks[2];
  p.copy.src_head[1] = vs[2];
  const int64_t blocks = (batch * t + p.copy.rows - 1) / p.copy.rows;
  if (blocks > 0x7FFFFFFF) return DSA_ERR_UNSUPPORTED;
  p.table = block_table;
  p.start = start;
  p.max_pages = max_pages;
  p.batch = batch;
  p.t = t;
  st = device_error_word(&p.pool.err);
  if (st != DSA_OK) return st;
  auto kernel = flat_rows(p.copy) ? cache_append_kernel<true> : cache_append_kernel<false>;
  kernel<<<static_cast<unsigned>(blocks), kCopyThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
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
  const int64_t room = max_pages * page_size;
  const int cluster = select_cluster(batch, room);
  const int64_t stretch = (room + cluster - 1) / cluster;
  p.staged = static_cast<int>(stretch < kSelStaged ? stretch : kSelStaged);
  st = set_max_dynamic_smem(reinterpret_cast<const void*>(evict_select_kernel), kSelStaged * 4);
  if (st != DSA_OK) return st;
  {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>(batch * cluster));
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = static_cast<size_t>(p.staged) * 4;
    cfg.stream = cs;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = static_cast<unsigned>(cluster);
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    st = cuda_status(cudaLaunchKernelEx(&cfg, evict_select_kernel, p));
  }
  if (st != DSA_OK) return st;
  p.copy = row_copy(p.pool, batch * dst_pages * page_size);
  p.copy.src[0] = p.pool.k;
  p.copy.src[1] = p.pool.v;
  p.copy.src_head[0] = p.pool.ks[2];
  p.copy.src_head[1] = p.pool.vs[2];
  const int64_t blocks = (dst_pages * page_size + p.copy.rows - 1) / p.copy.rows;
  auto kernel = flat_rows(p.copy) ? evict_copy_kernel<true> : evict_copy_kernel<false>;
  return launch_dependent(kernel, dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(batch)),
                          dim3(kCopyThreads), 0, cs, p);
}
