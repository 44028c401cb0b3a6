// Attention of one new token per sequence over a paged key-value cache, for
// sm_100a: split over the cache's length and joined.
//
//   s_j = scale q.k_j over the keys the token sees: all of its sequence, or the
//   last `window` and the first n_first of them
//   out = sum_j e^(s_j) v_j / (sum_j e^(s_j) + e^(sink_h))
//   weights[slot of j] += sum_h e^(s_j - lse_h)          (optional)
//
// Bound by the cache's bytes: every visible K and V row is read once for all
// heads of its group. The keys of a (sequence, kv head) are cut into chunks of
// 128; all chunks of the batch form one line, and each CTA (one per SM,
// persistent) takes an equal stretch of it, so ragged lengths balance. A stretch
// may end one sequence and start another: each (CTA, sequence) piece leaves a
// partial (maximum, sum, output) per softmax warpgroup, which paged_join_kernel
// joins in a fixed order.
//
// Heads are the N side of the products (S^T = K Q^T, O^T += V^T P^T): a group of
// 8 heads costs a few columns and not a 128-row tile, and a thread owns one KEY:
// its visibility is one flag, its weights of all heads lie in its registers.
//   warps 0, 3  TMA: pages -> rings of 128-row slots, K and q by warp 0, V by warp 3 (one
//               ring for both when they are one tensor), in granules of 8, 16 or 32
//               rows that never cross a page
//   warps 1, 2  tcgen05 issuers: S^T and O^T
//   warps 4..11 softmax: warpgroup w takes the chunks of parity w, with its own
//               accumulator, reference and sums; S^T products run up to four chunks ahead
// The reference of a head is the score of a warpgroup's first visible key of a
// piece and moves (O and the sums are rescaled) only when a score exceeds it by more
// than 2^14, so the common chunk needs one vote and no reduction over keys; the sums
// stay per thread until the piece ends. P is rounded to the operands' type
// (relative 2^-8 at most for bf16, 2^-11 for fp16 and below its normal range 2^-25 of the row's
// largest P: the size of the output's own rounding); sums are fp32.
// TMEM: kSBufs S^T buffers of NM columns, then O^T of the two warpgroups.
//
// Measured (bf16, head_dim 128):
//   64 sequences of up to 8192 rows, 32 heads on 8, with weights: 221 us for 1.21 GB;
//   the split kernel 202 us, 6.0 TB/s (DRAM 76 % active), the weights 12, the join 8.
//   8 sequences of up to 131,072 rows, 64 heads on one kv head (K is V): split 52 us,
//   172 MB at 3.3 TB/s. Bound by the softmax: 8,192 exponentials a chunk, about 3,450
//   cycles for a warpgroup with two of them in turn; DRAM 37 %.
//   One sequence of 333 rows, 64 heads: split 9 us, join 4.4: the launches' and a
//   chunk's latency.
//   One copy warp for all rings and one issuer for S^T and O^T: 242, 71 and 41 us.
#include "host_util.h"
#include "window_common.cuh"
#include "window_host.h"

namespace dsa {
namespace paged {

using win::Bf16;
using win::Fp16;
using win::kLn2;
using win::kLog2e;

constexpr int kThreads = 384;
constexpr int kRegsAux = 88;        // 128 x 88 + 256 x 208 = 384 x 168 at launch
constexpr int kRegsSoftmax = 208;
constexpr int kKeys = 128;          // keys of a chunk
constexpr int kBox = kKeys * 128;   // one [128 keys x 64 columns] SW128 box
constexpr float kRescaleLog2 = 14.0f;  // P <= 2^14 fits fp16
constexpr int kMaxSmem = 232448;
constexpr float kNone = -1.0e30f;   // reference of a piece without a visible key

template <int D, int NM>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kSlotBytes = kKeys * D * 2;
  static constexpr int kSlots = (NM == 128 ? 3 : 5) * (128 / D);
  static constexpr int kSBufs = NM == 128 ? 2 : 4;  // S^T products that may run ahead
  static constexpr int kSlotsK = kSlots / 2;        // of them K's; V has the others
  static constexpr int kSlotsV = kSlots - kSlotsK;
  static constexpr int kQBytes = NM * D * 2;
  static constexpr int kPBytes = kKeys * (NM < 64 ? 64 : NM) * 2;  // [128 keys x 64 heads] boxes
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = kOffQ + kQBytes;
  // the second 64-column half of V^T that a 64-wide head lacks is read from the
  // next slot, past the last one from P: rows 64.. of O^T are not used
  static constexpr int kOffP = kOffKV + kSlots * kSlotBytes;
  static constexpr int kOffMax = kOffP + 2 * kPBytes;         // [2][4 warps][NM] f32
  static constexpr int kOffRef = kOffMax + 2 * 4 * NM * 4;    // [2][2: reference, step][NM]
  static constexpr int kOffMeta = kOffRef + 2 * 2 * NM * 4;   // [16 chunks][16] granule states
  static constexpr int kOffBar = kOffMeta + 16 * 16 * 4;
  static constexpr int kNumBars = 2 + 2 * kSlots + 2 * kSBufs + 2 + 2 + 2 + 2 + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 48 + 1024;
  static constexpr int kColsO = kSBufs * NM;                  // TMEM: S^T buffers, then O^T
  static constexpr uint32_t kTmemCols = kColsO + 2 * NM <= 256 ? 256 : 512;
};

struct Params {
  int batch, h, hk, g;
  int page, max_pages;        // page size, table width
  int gran, gshift;           // rows of a granule, a power of two
  int64_t num_pages;
  int window, n_first;        // window 0: the whole sequence
  const int* table;           // [batch, max_pages]
  const int* lens;            // [batch]
  float scale_log2;
  const float* sink;          // [h] or null
  int shared;
  float* part_o;              // [piece][2][g][D]
  float2* part_ml;            // [piece][2][g]
  float* scores;              // [chunk][128][g] log2-scaled, or null
  float* lse2;                // [batch, h] log2-scaled lse
  void* out;                  // [batch, h, D]
  float* lse;                 // [batch, h] or null
  float* weights;             // [num_pages, page] or null
  int units;                  // CTAs of the split kernel
  unsigned int* err;
};

// The visible rows of one sequence, as granules of `gran` rows: those of the first
// tokens, then those of the window range.
struct Seq {
  int len, lo, nf;   // window range [lo, len); first tokens [0, nf) that stand apart
  int start;         // first row of the window's granules
  int nfg, chunks;
};

__device__ __forceinline__ Seq make_seq(const Params& p, int b) {
  Seq s;
  const int64_t room = static_cast<int64_t>(p.max_pages) * p.page;
  s.len = max(__ldg(p.lens + b), 0);
  if (s.len > room) s.len = static_cast<int>(room);
  s.lo = p.window > 0 ? max(s.len - p.window, 0) : 0;
  s.nf = min(p.n_first, s.len);
  if (s.lo <= s.nf) s.lo = s.nf = 0;
  s.start = s.lo & -p.gran;
  s.nfg = (s.nf + p.gran - 1) >> p.gshift;
  const int n = s.nfg + ((s.len - s.start + p.gran - 1) >> p.gshift);
  s.chunks = ((n << p.gshift) + kKeys - 1) / kKeys;
  return s;
}
__device__ __forceinline__ int seq_chunks(const Params& p, int b) { return make_seq(p, b).chunks; }

// First row of granule i (may lie at or past len in the last chunk).
__device__ __forceinline__ int gran_row(const Params& p, const Seq& s, int i) {
  return i < s.nfg ? i * p.gran : s.start + (i - s.nfg) * p.gran;
}
__device__ __forceinline__ bool row_seen(const Seq& s, int gran, int row) {
  return gran < s.nfg ? row < s.nf : (row >= s.lo && row < s.len);
}
// Page of a row and whether the table names one that exists.
__device__ __forceinline__ int page_of(const Params& p, int b, int row) {
  const int page = __ldg(p.table + static_cast<int64_t>(b) * p.max_pages + row / p.page);
  return page >= 0 && page < p.num_pages ? page : -1;
}

// The line of all chunks cut into `units` stretches whose lengths differ by one at
// most: the first `more` have each + 1 chunks.
struct Line {
  int each, more;
  __device__ __forceinline__ Line(int all, int units) : each(all / units), more(all - each * units) {}
  __device__ __forceinline__ int start(int u) const { return u * each + min(u, more); }
  __device__ __forceinline__ int owner(int chunk) const {
    const int longer = more * (each + 1);
    return chunk < longer ? chunk / (each + 1) : more + (chunk - longer) / each;
  }
};

// Chunks (of one kv head) of all sequences before b and of the whole batch, summed by
// one warp.
__device__ __forceinline__ void chunk_sums(const Params& p, int b, int* before, int* all) {
  int x = 0, y = 0;
  for (int i = threadIdx.x & 31; i < p.batch; i += 32) {
    const int n = seq_chunks(p, i);
    y += n;
    if (i < b) x += n;
  }
  *before = __reduce_add_sync(0xFFFFFFFFu, x);
  *all = __reduce_add_sync(0xFFFFFFFFu, y);
}

// A CTA's stretch, walked piece by piece. The line orders the chunks by (sequence,
// kv head, chunk).
struct Walk {
  int b, kvh, c0, c1;   // the piece: chunks [c0, c1) of (b, kvh)
  int left;             // chunks of the stretch after this piece
  Seq s;
};

__device__ __forceinline__ bool walk_take(const Params& p, Walk& w) {
  // (b, kvh, c0) is the next chunk, w.left what the stretch still holds
  while (w.left > 0) {
    if (w.b >= p.batch) return false;
    w.s = make_seq(p, w.b);
    if (w.c0 >= w.s.chunks) {  // an empty sequence, or a finished head
      w.c0 = 0;
      if (w.s.chunks == 0 || ++w.kvh == p.hk) {
        w.kvh = 0;
        ++w.b;
      }
      continue;
    }
    w.c1 = w.c0 + min(w.s.chunks - w.c0, w.left);
    w.left -= w.c1 - w.c0;
    return true;
  }
  return false;
}
__device__ __forceinline__ void walk_next(Walk& w) { w.c0 = w.c1; }

// Reduces 32 values of each lane over the lanes: lane k gets the result of a[k]. Each
// step halves the values a lane carries, so it takes 31 shuffles and not 160.
template <typename Op>
__device__ __forceinline__ float warp_transposed(float (&a)[32], int lane, Op op) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = (lane & o) != 0;
#pragma unroll
    for (int k = 0; k < o; ++k) {
      const float send = up ? a[k] : a[k + o];
      const float keep = up ? a[k + o] : a[k];
      a[k] = op(keep, __shfl_xor_sync(0xFFFFFFFFu, send, o));
    }
  }
  return a[0];
}

static_assert(Cfg<128, 32>::kSmemBytes <= kMaxSmem && Cfg<128, 64>::kSmemBytes <= kMaxSmem &&
                  Cfg<128, 128>::kSmemBytes <= kMaxSmem && Cfg<64, 32>::kSmemBytes <= kMaxSmem &&
                  Cfg<64, 64>::kSmemBytes <= kMaxSmem && Cfg<64, 128>::kSmemBytes <= kMaxSmem,
              "227 KB of shared memory a CTA");

template <typename T, int D, int NM>
__global__ void __launch_bounds__(kThreads, 1)
    paged_split_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                       const __grid_constant__ CUtensorMap tm_v, const Params p) {
  using C = Cfg<D, NM>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;                    // rows of q -> MMA
  uint64_t* q_empty = q_full + 1;             // last S^T of the piece done -> TMA
  uint64_t* kv_full = q_empty + 1;            // [kSlots]
  uint64_t* kv_empty = kv_full + C::kSlots;   // [kSlots]
  uint64_t* s_full = kv_empty + C::kSlots;    // [kSBufs] S^T of a chunk in TMEM
  uint64_t* s_empty = s_full + C::kSBufs;     // [kSBufs] its scores are read (128 arrivals)
  uint64_t* p_full = s_empty + C::kSBufs;     // [2] P written (128 arrivals)
  uint64_t* o_done = p_full + 2;              // [2] O^T product of a chunk completed
  uint64_t* o_empty = o_done + 2;             // [2] O^T read at a piece's end (128 arrivals)
  uint64_t* v_ready = o_empty + 2;            // [2] V of the warpgroup's chunk has arrived
  uint64_t* drain_bar = v_ready + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);
  int* walk_s = reinterpret_cast<int*>(smem + C::kOffMisc + 8);  // b, kvh, chunk, left
  int* meta = reinterpret_cast<int*>(smem + C::kOffMeta);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int npad = (p.g + 31) & ~31;
  const int gpc = kKeys >> p.gshift;  // granules of a chunk

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int i = 0; i < C::kSBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&s_empty[i], 128);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&p_full[w], 128);
      mbar_init(&o_done[w], 1);
      mbar_init(&o_empty[w], 128);
      mbar_init(&v_ready[w], 1);
    }
    mbar_init(drain_bar, 2);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // rows of q past the group stay 0: their scores are 0, their columns are not used
  if (p.g < npad) {
    for (int i = threadIdx.x; i < C::kQBytes / 16; i += kThreads)
      st_shared_v4(smem_u32(smem + C::kOffQ + i * 16), 0u, 0u, 0u, 0u);
    fence_proxy_async_smem();
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == 2) {
    // where this CTA's stretch [first, last) of the line starts
    int unused, all;
    chunk_sums(p, 0, &unused, &all);
    const Line line(all * p.hk, p.units);
    const int first = line.start(blockIdx.x), last = line.start(blockIdx.x + 1);
    int base = 0;  // chunks before the 32 sequences that the lanes hold
    int b = p.batch, kvh = 0, c = 0;
    bool found = first >= last;
    for (int i0 = 0; i0 < p.batch && !found; i0 += 32) {
      const int mine = i0 + lane < p.batch ? seq_chunks(p, i0 + lane) * p.hk : 0;
      int sum = mine;  // inclusive prefix over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t hit = __ballot_sync(0xFFFFFFFFu, first < base + sum && mine > 0);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        const int begin = base + __shfl_sync(0xFFFFFFFFu, sum - mine, l);
        const int n = __shfl_sync(0xFFFFFFFFu, mine, l) / p.hk;
        b = i0 + l;
        kvh = (first - begin) / n;
        c = (first - begin) - kvh * n;
        found = true;
      }
      base += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    if (lane == 0) {
      walk_s[0] = b;
      walk_s[1] = kvh;
      walk_s[2] = c;
      walk_s[3] = last - first;
    }
  }
  if (warp == 3 && blockIdx.x == 0) {
    // lengths outside the table's room are clamped and reported
    for (int i = lane; i < p.batch; i += 32) {
      const int n = __ldg(p.lens + i);
      if (n < 0 || n > static_cast<int64_t>(p.max_pages) * p.page) atomicOr(p.err, DSA_DEVERR_CACHE);
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  grid_launch_dependents();
  const uint32_t tmem = *tmem_holder;
  Walk wk;
  wk.b = walk_s[0];
  wk.kvh = walk_s[1];
  wk.c0 = walk_s[2];
  wk.left = walk_s[3];
  // slots of the ring that chunks take in turn: K's (or both), and V's behind them
  const int ring_k = p.shared ? C::kSlots : C::kSlotsK;

  if (warp < 4) {
    win::set_max_regs_dec<kRegsAux>();
    if (warp == 0 || (warp == 3 && !p.shared)) {
      // ---------------------------------------------------------- producers: K (and q), V
      const bool is_v = warp == 3;
      const CUtensorMap* tm = is_v ? &tm_v : &tm_k;
      const int slot0 = is_v ? C::kSlotsK : 0, slots = is_v ? C::kSlotsV : ring_k;
      Ring<0> at;
      int gc = 0, pieces = 0;
      bool ok = true;
      // a lane per granule of the next `ahead` chunks: their pages are looked up while the
      // copies of the chunks before them are waited for
      const int ahead = 32 / gpc;
      const int sub = lane / gpc, gi = lane - sub * gpc;
      for (; ok && walk_take(p, wk); walk_next(wk), ++pieces) {
        if (!is_v) {
          ok = mbar_wait_warp(q_empty, (pieces & 1) ^ 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
          if (!ok) break;
          if (lane == 0) {
            mbar_arrive_expect_tx(q_full, static_cast<uint32_t>(p.g * D * 2));
#pragma unroll
            for (int half = 0; half < C::kHalves; ++half)
              tma_load_3d(smem + C::kOffQ + half * NM * 128, &tm_q, half * 64, wk.kvh * p.g, wk.b,
                          q_full);
          }
        }
        int page = -1, row = 0, next_page = -1, next_row = 0;
        auto look = [&](int c) {
          const int r = gran_row(p, wk.s, (c + sub) * gpc + gi);
          const int i = r / p.page;
          next_row = r - i * p.page;
          next_page = c + sub < wk.c1 && r < wk.s.len
                          ? __ldg(p.table + static_cast<int64_t>(wk.b) * p.max_pages + i)
                          : -2;  // nothing to read
        };
        look(wk.c0);
        for (int c = wk.c0, turn = 0; c < wk.c1; ++c, ++gc, turn = turn + 1 == ahead ? 0 : turn + 1) {
          if (turn == 0) {
            page = next_page;
            row = next_row;
            if (page != -2 && (page < 0 || page >= p.num_pages)) {
              atomicOr(p.err, DSA_DEVERR_CACHE);
              page = -1;
            }
            look(c + ahead);
          }
          const bool mine = sub == turn;
          const bool live = mine && page >= 0;
          const int bytes = __popc(__ballot_sync(0xFFFFFFFFu, live)) * p.gran * D * 2;
          const int s = slot0 + at.slot;
          ok = mbar_wait_warp(&kv_empty[s], at.parity ^ 1u, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
          if (!ok) break;
          // the granules' states: the ring of 16 is longer than any chunk is ahead
          if (mine && !is_v) meta[(gc & 15) * 16 + gi] = live ? 1 : 0;
          __syncwarp();
          if (lane == 0) mbar_arrive_expect_tx(&kv_full[s], static_cast<uint32_t>(bytes));
          __syncwarp();
          if (live) {
            uint8_t* dst = smem + C::kOffKV + s * C::kSlotBytes + gi * p.gran * 128;
#pragma unroll
            for (int half = 0; half < C::kHalves; ++half)
              tma_load_4d(dst + half * kBox, tm, half * 64, row, wk.kvh, page, &kv_full[s]);
          }
          at.next(slots);
        }
      }
      // copies in flight land before the CTA's shared memory goes away
      for (int i = max(gc - slots, 0); i < gc; ++i)
        mbar_drain(&kv_full[slot0 + i % slots], static_cast<uint32_t>((i / slots) & 1));
      if (!is_v && pieces > 0) mbar_drain(q_full, (pieces - 1) & 1);
    } else if (warp == 1 || warp == 2) {
      // ---------------------------------------------------------- MMA issuers: S^T, O^T
      // The whole warp walks and waits; one elected lane issues.
      const uint32_t idesc_s = win::make_idesc<T>(128, 0, 0) | (static_cast<uint32_t>(npad / 8) << 17);
      const uint32_t idesc_o = win::make_idesc<T>(128, 0, 1) | (1u << 15) |
                               (static_cast<uint32_t>(npad / 8) << 17);
      const uint64_t dq = make_smem_desc(smem_u32(smem + C::kOffQ), 16u, 1024u, kLayoutSW128);
      const uint32_t hi = static_cast<uint32_t>(dq >> 32);
      const uint32_t q_lo = static_cast<uint32_t>(dq);
      const uint32_t k_lo = q_lo + static_cast<uint32_t>((C::kOffKV - C::kOffQ) >> 4);
      const uint32_t v_lo = static_cast<uint32_t>(make_smem_desc(
          smem_u32(smem + C::kOffKV), static_cast<uint32_t>(kBox), 1024u, kLayoutSW128));
      const uint32_t p_lo = static_cast<uint32_t>(make_smem_desc(
          smem_u32(smem + C::kOffP), static_cast<uint32_t>(kBox), 1024u, kLayoutSW128));
      Ring<0> at;
      int gc = 0, pieces = 0;
      int drained[2] = {0, 0};  // pieces of the warpgroup whose O^T was to be read
      bool ok = true;
      auto wait_warp = [&](uint64_t* b, uint32_t parity) -> bool {
        return mbar_wait_warp(b, parity, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
      };
      // S^T runs ahead of the softmax by up to kSBufs chunks
      auto issue_s = [&](bool end) -> bool {
        const int s = at.slot;
        const uint32_t buf = static_cast<uint32_t>(gc) % C::kSBufs;
        if (!wait_warp(&kv_full[s], at.parity) ||
            !wait_warp(&s_empty[buf], ((static_cast<uint32_t>(gc) / C::kSBufs) & 1u) ^ 1u))
          return false;
        at.next(ring_k);
        tc_fence_after();
        const uint32_t ka = k_lo + static_cast<uint32_t>(s * (C::kSlotBytes >> 4));
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t ao = static_cast<uint32_t>(((k >> 2) * kBox + (k & 3) * 32) >> 4);
            const uint32_t bo = static_cast<uint32_t>(((k >> 2) * NM * 128 + (k & 3) * 32) >> 4);
            umma_bf16(tmem + buf * NM, desc_from_words(ka + ao, hi), desc_from_words(q_lo + bo, hi),
                      idesc_s, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[buf]);
          if (!p.shared) umma_commit(&kv_empty[s]);
          if (end) umma_commit(q_empty);
        }
        __syncwarp();
        return true;
      };
      auto issue_o = [&](bool fresh) -> bool {
        const int w = gc & 1;
        const int s = p.shared ? at.slot : C::kSlotsK + at.slot;
        // shared: the slot's data is there, since the chunk's P is made of its S^T
        if (!p.shared && !wait_warp(&kv_full[s], at.parity)) return false;
        if (elect_one()) mbar_arrive(&v_ready[w]);  // the softmax may clear its hidden rows
        __syncwarp();
        at.next(p.shared ? ring_k : C::kSlotsV);
        if (!wait_warp(&p_full[w], (gc >> 1) & 1)) return false;
        if (fresh) {
          const int d = w ? drained[1]++ : drained[0]++;
          if (d > 0 && !wait_warp(&o_empty[w], (d - 1) & 1)) return false;
        }
        tc_fence_after();
        const uint32_t va = v_lo + static_cast<uint32_t>(s * (C::kSlotBytes >> 4));
        const uint32_t pb = p_lo + static_cast<uint32_t>(w * (C::kPBytes >> 4));
        const uint32_t d = tmem + static_cast<uint32_t>(C::kColsO + w * NM);
        if (elect_one()) {
#pragma unroll
          for (int st = 0; st < kKeys / 16; ++st)
            umma_bf16(d, desc_from_words(va + static_cast<uint32_t>(st * 128), hi),
                      desc_from_words(pb + static_cast<uint32_t>(st * 128), hi), idesc_o,
                      (fresh && st == 0) ? 0u : 1u);
          umma_commit(&o_done[w]);
          umma_commit(&kv_empty[s]);
        }
        __syncwarp();
        return true;
      };
      for (; ok && walk_take(p, wk); walk_next(wk), ++pieces) {
        const int n = wk.c1 - wk.c0;
        if (warp == 1) {
          ok = wait_warp(q_full, pieces & 1);
          for (int j = 0; ok && j < n; ++j, ++gc) ok = issue_s(j == n - 1);
        } else {
          // the first chunk of each warpgroup in the piece starts its sum anew
          for (int j = 0; ok && j < n; ++j, ++gc) ok = issue_o(j < 2);
        }
      }
      if (elect_one()) umma_commit(drain_bar);
      __syncwarp();
      mbar_drain(drain_bar, 0);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax
    // After a wait that ran out the abort flag makes every later wait return at once: the
    // loops run to their end, so that no thread misses a named barrier, on values that
    // the error word declares void.
    win::set_max_regs_inc<kRegsSoftmax>();
    const int w = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int key = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t od = tmem + lane_off + static_cast<uint32_t>(C::kColsO + w * NM);
    const uint32_t bar = 1 + static_cast<uint32_t>(w);
    // shared-memory addresses of the warpgroup's per-warp maxima [4][NM], the heads'
    // negative references [NM] and their last steps [NM]
    const uint32_t wmax = smem_u32(smem + C::kOffMax) + static_cast<uint32_t>(w * 4 * NM * 4);
    const uint32_t nref = smem_u32(smem + C::kOffRef) + static_cast<uint32_t>(w * 2 * NM * 4);
    const uint32_t move = nref + NM * 4;
    const int gi = key >> p.gshift;  // the key's granule of a chunk and row of it
    const int gr = key & (p.gran - 1);
    const uint32_t prow = smem_u32(smem + C::kOffP) + static_cast<uint32_t>(w * C::kPBytes + key * 128);
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    int gc = 0, gw = 0;
    uint32_t sp = 0;  // the chunk's S^T
    auto wait = [&](uint64_t* b, uint32_t parity) {  // whole warps
      mbar_wait(b, parity, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
      __syncwarp();
    };
    // 32 scores of the key relative to their heads' references, log2-scaled
    auto load_scores = [&](int q, uint64_t (&d)[16]) {
      uint32_t v[32];
      tmem_ld_32x32b_x32(sp + static_cast<uint32_t>(q * 32), v);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float4 r = ld_shared_f4(nref + static_cast<uint32_t>(q * 128 + k * 16));
        d[2 * k] = f2_fma(f2_pack(__uint_as_float(v[4 * k]), __uint_as_float(v[4 * k + 1])), scale2,
                          f2_pack(r.x, r.y));
        d[2 * k + 1] = f2_fma(f2_pack(__uint_as_float(v[4 * k + 2]), __uint_as_float(v[4 * k + 3])),
                              scale2, f2_pack(r.z, r.w));
      }
    };
    for (; walk_take(p, wk); walk_next(wk)) {
      uint64_t l2[NM / 2];  // sums of the key's weights, two heads a register pair
#pragma unroll
      for (int k = 0; k < NM / 2; ++k) l2[k] = 0ull;
      const int n = wk.c1 - wk.c0;
      bool fresh = true;  // no chunk of the piece yet
      bool unset = true;  // no visible key yet: the references stand at 0
      if (key < npad) st_shared_f32(nref + key * 4, 0.f);
      named_bar_sync(bar, 128);
      for (int j = 0; j < n; ++j, ++gc) {
        if ((gc & 1) != w) continue;
        const int c = wk.c0 + j;
        const int row = gran_row(p, wk.s, c * gpc + gi) + gr;
        const uint32_t buf = static_cast<uint32_t>(gc) % C::kSBufs;
        sp = tmem + lane_off + buf * NM;
        wait(&s_full[buf], (static_cast<uint32_t>(gc) / C::kSBufs) & 1u);
        tc_fence_after();
        const bool valid = row_seen(wk.s, c * gpc + gi, row) && meta[(gc & 15) * 16 + gi] != 0;
        // up to 64 heads the scores stay in registers; beyond, they are loaded again
        constexpr bool kHold = NM <= 64;
        uint64_t d[kHold ? NM / 32 : 1][16];
#pragma unroll
        for (int q = 0; q < NM / 32; ++q)
          if (kHold && q * 32 < npad) load_scores(q, d[q]);
        if (unset) {
          // the references are the scores of the first visible key: any key does, as long
          // as the vote below moves a reference that others exceed by far
          const uint32_t seen = __ballot_sync(0xFFFFFFFFu, valid);
          if (lane == 0) st_shared_f32(wmax + quarter * 4, __uint_as_float(seen));
          named_bar_sync(bar, 128);
          int owner = -1;
#pragma unroll
          for (int i = 3; i >= 0; --i)
            if (__float_as_uint(ld_shared_f32(wmax + i * 4)) != 0u) owner = i;
          if (owner >= 0) {
            const bool mine = quarter == owner && lane == __ffs(seen) - 1;
#pragma unroll
            for (int q = 0; q < NM / 32; ++q) {
              if (q * 32 < npad) {
                uint64_t(&x)[16] = d[kHold ? q : 0];
                if (!kHold) {
                  named_bar_sync(bar, 128);  // all warps read the references of 0
                  load_scores(q, x);
                }
                if (mine) {
#pragma unroll
                  for (int k = 0; k < 16; ++k) {
                    float a, b;
                    f2_unpack(x[k], a, b);
                    st_shared_f32(nref + static_cast<uint32_t>((q * 32 + 2 * k) * 4), -a);
                    st_shared_f32(nref + static_cast<uint32_t>((q * 32 + 2 * k) * 4 + 4), -b);
                  }
                }
              }
            }
            named_bar_sync(bar, 128);
#pragma unroll
            for (int q = 0; q < NM / 32; ++q)
              if (kHold && q * 32 < npad) load_scores(q, d[q]);
            unset = false;
          }
        }
        float excess = -INFINITY;
#pragma unroll
        for (int q = 0; q < NM / 32; ++q) {
          if (q * 32 < npad) {
            uint64_t(&x)[16] = d[kHold ? q : 0];
            if (!kHold) load_scores(q, x);
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float a, b;
              f2_unpack(x[k], a, b);
              excess = fmax3(excess, a, b);
            }
          }
        }
        // does any score exceed its head's reference by more than 2^14? Rare: the code is
        // kept short (rolled loops), so that it does not push the common path out of the
        // instruction cache
        if (named_bar_or(bar, 128, valid && excess > kRescaleLog2)) {
          // the heads' maxima over the chunk's keys: warps, then the warpgroup
#pragma unroll 1
          for (int q = 0; q * 32 < npad; ++q) {
            uint64_t x[16];
            load_scores(q, x);
            float a[32];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              f2_unpack(x[k], a[2 * k], a[2 * k + 1]);
              a[2 * k] = valid ? a[2 * k] : kNone;
              a[2 * k + 1] = valid ? a[2 * k + 1] : kNone;
            }
            const float m = warp_transposed(a, lane, [](float u, float v) { return fmaxf(u, v); });
            st_shared_f32(wmax + static_cast<uint32_t>((quarter * NM + q * 32 + lane) * 4), m);
          }
          named_bar_sync(bar, 128);
          if (key < npad) {
            float m = ld_shared_f32(wmax + key * 4);
#pragma unroll
            for (int i = 1; i < 4; ++i)
              m = fmaxf(m, ld_shared_f32(wmax + static_cast<uint32_t>((i * NM + key) * 4)));
            const float step = m > kRescaleLog2 ? m : 0.f;
            st_shared_f32(nref + key * 4, ld_shared_f32(nref + key * 4) - step);
            st_shared_f32(move + key * 4, ex2_approx(-step));
          }
          named_bar_sync(bar, 128);
          if (!fresh) {
            wait(&o_done[w], (gw - 1) & 1);
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q * 32 < npad; ++q) {
              uint32_t v[32];
              tmem_ld_32x32b_x32(od + static_cast<uint32_t>(q * 32), v);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float4 f = ld_shared_f4(move + static_cast<uint32_t>(q * 128 + k * 16));
                v[4 * k] = __float_as_uint(__uint_as_float(v[4 * k]) * f.x);
                v[4 * k + 1] = __float_as_uint(__uint_as_float(v[4 * k + 1]) * f.y);
                v[4 * k + 2] = __float_as_uint(__uint_as_float(v[4 * k + 2]) * f.z);
                v[4 * k + 3] = __float_as_uint(__uint_as_float(v[4 * k + 3]) * f.w);
              }
              tmem_st_32x32b_x32(od + static_cast<uint32_t>(q * 32), v);
            }
#pragma unroll
            for (int k = 0; k < NM / 4; ++k) {
              if (4 * k < npad) {
                const float4 f = ld_shared_f4(move + static_cast<uint32_t>(k * 16));
                l2[2 * k] = f2_mul(l2[2 * k], f2_pack(f.x, f.y));
                l2[2 * k + 1] = f2_mul(l2[2 * k + 1], f2_pack(f.z, f.w));
              }
            }
          }
#pragma unroll
          for (int q = 0; q < NM / 32; ++q)
            if (kHold && q * 32 < npad) load_scores(q, d[q]);
        }
        // ---- P = 2^(z - reference), the key's weights of all heads
        if (gw > 0) wait(&o_done[w], (gw - 1) & 1);  // the previous product has read P
        float* zrow = nullptr;
        if (p.scores != nullptr) {
          // chunks of this sequence lie [kv head][chunk] at max_chunks of the table
          const int64_t cap = (static_cast<int64_t>(p.max_pages) * p.page + kKeys - 1) / kKeys + 2;
          zrow = p.scores +
                 (((static_cast<int64_t>(wk.b) * p.hk + wk.kvh) * cap + c) * kKeys + key) * p.g;
        }
        const bool some = !__all_sync(0xFFFFFFFFu, valid);
#pragma unroll
        for (int q = 0; q < NM / 32; ++q) {
          if (q * 32 < npad) {
            uint64_t(&x)[16] = d[kHold ? q : 0];
            if (!kHold) load_scores(q, x);
            if (some && !valid) {
#pragma unroll
              for (int k = 0; k < 16; ++k) x[k] = f2_pack(-INFINITY, -INFINITY);
            }
            if (zrow != nullptr) {
#pragma unroll
              for (int k = 0; k < 16; ++k) {
                float a, b;
                f2_unpack(x[k], a, b);
                const int i = q * 32 + 2 * k;
                if (i < p.g) zrow[i] = a - ld_shared_f32(nref + i * 4);
                if (i + 1 < p.g) zrow[i + 1] = b - ld_shared_f32(nref + i * 4 + 4);
              }
            }
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float a, b;
              f2_unpack(x[k], a, b);
              a = ex2_approx(a);
              b = ex2_approx(b);
              l2[q * 16 + k] = f2_add(l2[q * 16 + k], f2_pack(a, b));
              pk[k] = T::pack(a, b);
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint32_t c16 = static_cast<uint32_t>((q & 1) * 4 + k);
              st_shared_v4(prow + static_cast<uint32_t>((q >> 1) * kBox) +
                               ((c16 ^ static_cast<uint32_t>(key & 7)) << 4),
                           pk[4 * k], pk[4 * k + 1], pk[4 * k + 2], pk[4 * k + 3]);
            }
          }
        }
        if (!valid) {
          // a hidden V row may hold anything, and 0 x NaN is NaN: it is cleared. The issuer
          // of O^T, which waits for V's slots in their order, says when it is there
          const int sv = p.shared ? gc % C::kSlots : C::kSlotsK + gc % C::kSlotsV;
          mbar_wait(&v_ready[w], gw & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
          uint8_t* vr = smem + C::kOffKV + sv * C::kSlotBytes + key * 128;
#pragma unroll
          for (int x = 0; x < C::kHalves * 8; ++x)
            st_shared_v4(smem_u32(vr + (x >> 3) * kBox + (x & 7) * 16), 0u, 0u, 0u, 0u);
        }
        __syncwarp();
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&s_empty[buf]);
        mbar_arrive(&p_full[w]);
        ++gw;
        fresh = false;
      }
      // ---- the piece's partial of this warpgroup
      const int64_t piece = static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(wk.b) * p.hk + wk.kvh;
      float2* ml = p.part_ml + (piece * 2 + w) * p.g;
      if (fresh) {  // it had no chunk
        if (key < p.g) ml[key] = make_float2(kNone, 0.f);
        continue;
      }
      wait(&o_done[w], (gw - 1) & 1);
      tc_fence_after();
#pragma unroll
      for (int q = 0; q < NM / 32; ++q) {
        if (q * 32 < npad) {
          // sums over the warp's 32 keys of 32 heads
          float a[32];
#pragma unroll
          for (int k = 0; k < 16; ++k) f2_unpack(l2[q * 16 + k], a[2 * k], a[2 * k + 1]);
          const float sum = warp_transposed(a, lane, [](float u, float v) { return u + v; });
          st_shared_f32(wmax + static_cast<uint32_t>((quarter * NM + q * 32 + lane) * 4), sum);
          uint32_t v[32];
          tmem_ld_32x32b_x32(od + static_cast<uint32_t>(q * 32), v);
          if (key < D) {
            float* dst = p.part_o + ((piece * 2 + w) * p.g + q * 32) * D + key;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (q * 32 + k < p.g) dst[k * D] = __uint_as_float(v[k]);
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&o_empty[w]);
      named_bar_sync(bar, 128);
      if (key < p.g) {
        float sum = ld_shared_f32(wmax + key * 4);
#pragma unroll
        for (int i = 1; i < 4; ++i) sum += ld_shared_f32(wmax + static_cast<uint32_t>((i * NM + key) * 4));
        // chunks of absent pages leave no reference: the join must not take their 0 for one
        ml[key] = make_float2(unset ? kNone : -ld_shared_f32(nref + key * 4), sum);
      }
      named_bar_sync(bar, 128);  // the next piece writes the references and maxima
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::kTmemCols);
  }
}

// Joins the pieces of one (sequence, head): a block of D threads, a column each. The
// pieces' maxima and sums are read at once, then the outputs eight at a time; latency
// bound (a few MB at most).
template <typename T, int D>
__global__ void __launch_bounds__(D) paged_join_kernel(const Params p) {
  extern __shared__ float weight[];  // [2 (units + 1)]
  __shared__ float red[2][D / 32];
  const int head = blockIdx.x % p.h;
  const int b = blockIdx.x / p.h;
  const int kvh = head / p.g, gi = head - kvh * p.g;
  const int x = threadIdx.x, warp = x >> 5;
  int before, all;
  chunk_sums(p, b, &before, &all);
  const int n = seq_chunks(p, b);
  const Line line(all * p.hk, p.units);
  const float sink2 = p.sink != nullptr ? __ldg(p.sink + head) * kLog2e : -INFINITY;
  int u0 = 0, parts = 0;  // two (warpgroups) per piece, none of which is empty
  if (n > 0) {
    const int first = before * p.hk + kvh * n;
    u0 = line.owner(first);
    parts = (line.owner(first + n - 1) - u0 + 1) * 2;
  }
  grid_dependency_wait();
  // piece u of (sequence, kv head) is number u + b hk + kvh
  const int64_t piece = (static_cast<int64_t>(u0) + static_cast<int64_t>(b) * p.hk + kvh) * 2;
  auto part = [&](int i) -> float2 {
    return p.part_ml[(piece + i) * p.g + gi];
  };
  float top = kNone;
  for (int i = x; i < parts; i += D) top = fmaxf(top, part(i).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, o));
  if ((x & 31) == 0) red[0][warp] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < D / 32; ++i) top = fmaxf(top, red[0][i]);
  top = fmaxf(top, sink2);
  float sum = 0.f;
  for (int i = x; i < parts; i += D) {
    const float2 ml = part(i);
    // a part without a visible key (sum 0) is not read below
    const float f = ml.y == 0.f ? 0.f : ex2_approx(ml.x - top);
    weight[i] = f;
    sum += ml.y * f;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
  if ((x & 31) == 0) red[1][warp] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i) sum += red[1][i];
  float acc = 0.f;
  const float* o = p.part_o + (piece * p.g + gi) * D + x;
#pragma unroll 8
  for (int i = 0; i < parts; ++i)
    if (weight[i] != 0.f) acc = fmaf(o[static_cast<int64_t>(i) * p.g * D], weight[i], acc);
  const float total = sum + (p.sink != nullptr ? ex2_approx(sink2 - top) : 0.f);
  const float v = total == 0.f ? 0.f : acc / total;
  const uint32_t bits = T::pack(v, 0.f);
  static_cast<uint16_t*>(p.out)[static_cast<int64_t>(blockIdx.x) * D + x] =
      static_cast<uint16_t>(bits & 0xFFFFu);
  if (x == 0) {
    const float lse2 = total == 0.f ? -INFINITY : top + log2f(total);
    p.lse2[blockIdx.x] = lse2;
    if (p.lse != nullptr) p.lse[blockIdx.x] = lse2 * kLn2;
  }
}

// weights[slot of key] += sum over heads of 2^(z - lse): a thread a key, heads in order,
// four at a time where the group's size and the scores' rows allow. lse is the join's
// result, so it is read with ordinary loads: a read-only load is not held back by the wait.
__global__ void __launch_bounds__(kKeys) paged_weights_kernel(const Params p) {
  const int b = blockIdx.y, c = blockIdx.x;
  const Seq s = make_seq(p, b);
  int row = 0, page = -1;
  if (c < s.chunks) {
    const int per = kKeys >> p.gshift;
    const int gi = threadIdx.x >> p.gshift;
    row = gran_row(p, s, c * per + gi) + (threadIdx.x & (p.gran - 1));
    if (row_seen(s, c * per + gi, row)) page = page_of(p, b, row);
  }
  // every block waits, also those without a visible row: the launch after this one counts on
  // the join being done once this grid is
  grid_dependency_wait();
  if (page < 0) return;
  const int64_t cap = (static_cast<int64_t>(p.max_pages) * p.page + kKeys - 1) / kKeys + 2;
  const float* lse = p.lse2 + static_cast<int64_t>(b) * p.h;
  const float* z = p.scores + ((static_cast<int64_t>(b) * p.hk * cap + c) * kKeys + threadIdx.x) * p.g;
  const int64_t step = cap * kKeys * p.g;  // to the next kv head
  float sum = 0.f;
  if (p.g % 4 == 0) {
    const int n4 = p.h / 4, g4 = p.g / 4;
#pragma unroll 8
    for (int i = 0; i < n4; ++i) {
      const int kvh = i / g4;
      const float4 a = *reinterpret_cast<const float4*>(z + kvh * step + (i - kvh * g4) * 4);
      const float4 m = reinterpret_cast<const float4*>(lse)[i];
      sum += (ex2_approx(a.x - m.x) + ex2_approx(a.y - m.y)) +
             (ex2_approx(a.z - m.z) + ex2_approx(a.w - m.w));
    }
  } else {
    for (int kvh = 0; kvh < p.hk; ++kvh)
      for (int k = 0; k < p.g; ++k)
        sum += ex2_approx(z[kvh * step + k] - lse[kvh * p.g + k]);
  }
  // one add per slot; pages that sequences share get one from each
  atomicAdd(p.weights + static_cast<int64_t>(page) * p.page + row % p.page, sum);
}

// ------------------------------------------------------------------ host
struct Plan {
  int units;
  size_t off_ml, off_lse, off_scores, bytes;
};

inline int64_t max_chunks(int64_t max_pages, int64_t page) {
  // first-token and window ranges each end in a partly used granule
  return (max_pages * page + kKeys - 1) / kKeys + 2;
}

// One CTA per SM of a full GPU (148, also on a part of one: the pieces and with them the bits
// stay the same, and no CTA waits for another), fewer when the batch cannot have that many
// chunks.
inline Plan plan_paged(int64_t batch, int h, int hk, int d, int64_t max_pages, int64_t page,
                       bool weights) {
  Plan pl;
  const int64_t bound = batch * hk * max_chunks(max_pages, page);
  pl.units = static_cast<int>(bound < 148 ? bound : 148);
  const auto pad = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  const size_t pieces = static_cast<size_t>(pl.units) + static_cast<size_t>(batch) * hk;
  const size_t g = static_cast<size_t>(h / hk);
  pl.off_ml = pad(pieces * 2 * g * d * sizeof(float));
  pl.off_lse = pl.off_ml + pad(pieces * 2 * g * sizeof(float2));
  pl.off_scores = pl.off_lse + pad(static_cast<size_t>(batch) * h * sizeof(float));
  pl.bytes = pl.off_scores +
             (weights ? static_cast<size_t>(bound) * kKeys * g * sizeof(float) : 0);
  return pl;
}

// Rows that a copy may take at once without crossing a page: the largest of 32,
// 16 and 8 that divides the page size.
inline int granule(int64_t page) { return page % 32 == 0 ? 32 : (page % 16 == 0 ? 16 : 8); }

template <typename T, int D, int NM>
int launch_split(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Params& p,
                 cudaStream_t stream) {
  using C = Cfg<D, NM>;
  auto kernel = paged_split_kernel<T, D, NM>;
  int st = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), C::kSmemBytes);
  if (st != DSA_OK) return st;
  kernel<<<p.units, kThreads, C::kSmemBytes, stream>>>(q, k, v, p);
  return cuda_status(cudaGetLastError());
}

template <typename T, int D>
int launch(const CUtensorMap& q, const CUtensorMap& k, const CUtensorMap& v, const Params& p,
           cudaStream_t stream) {
  int st = p.g <= 32   ? launch_split<T, D, 32>(q, k, v, p, stream)
           : p.g <= 64 ? launch_split<T, D, 64>(q, k, v, p, stream)
                       : launch_split<T, D, 128>(q, k, v, p, stream);
  if (st != DSA_OK) return st;
  st = launch_dependent(paged_join_kernel<T, D>, dim3(static_cast<unsigned>(p.batch * p.h)), dim3(D),
                        2 * (p.units + 1) * sizeof(float), stream, p);
  if (st != DSA_OK || p.weights == nullptr) return st;
  return launch_dependent(paged_weights_kernel,
                          dim3(static_cast<unsigned>(max_chunks(p.max_pages, p.page)),
                               static_cast<unsigned>(p.batch)),
                          dim3(kKeys), 0, stream, p);
}

// Pages [num_pages, page, heads, d]: a box of `rows` slots of one page and head.
inline int map_pages(CUtensorMap* tm, uint32_t fmt, const void* base, const int64_t* given,
                     int64_t num_pages, int64_t page, int heads, int d, int rows) {
  int64_t s[3] = {page * heads * d, static_cast<int64_t>(heads) * d, d};
  if (given != nullptr) {
    if (num_pages > 1) s[0] = given[0];
    s[1] = given[1];
    if (heads > 1) s[2] = given[2];
  }
  for (const int64_t x : s) {
    if (x <= 0 || x >= (int64_t{1} << 38)) return DSA_ERR_UNSUPPORTED;
    if (x % 8 != 0) return DSA_ERR_MISALIGNED;
  }
  const uint64_t dims[4] = {static_cast<uint64_t>(d), static_cast<uint64_t>(page),
                            static_cast<uint64_t>(heads), static_cast<uint64_t>(num_pages)};
  const uint64_t strides[3] = {static_cast<uint64_t>(s[1]) * 2, static_cast<uint64_t>(s[2]) * 2,
                               static_cast<uint64_t>(s[0]) * 2};
  const uint32_t box[4] = {64, static_cast<uint32_t>(rows), 1, 1};
  return encode_tensor_map(tm, win::map_type(fmt), 4, base, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
}

}  // namespace paged
}  // namespace dsa

extern "C" size_t dsa_paged_attn_workspace_bytes(int64_t batch, int n_heads, int n_kv_heads,
                                                 int head_dim, int64_t max_pages, int64_t page_size,
                                                 int want_weights) {
  if (batch < 1 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 || max_pages < 1 ||
      page_size < 1 || head_dim < 1)
    return 0;
  return dsa::paged::plan_paged(batch, n_heads, n_kv_heads, head_dim, max_pages, page_size,
                                want_weights != 0)
      .bytes;
}

extern "C" int dsa_paged_attn_fwd(const void* q, const int64_t* q_strides, const void* k_pages,
                                  const int64_t* k_strides, const void* v_pages,
                                  const int64_t* v_strides, const int* block_table, const int* lens,
                                  const float* sink, void* out, float* lse, float* weights, int dtype,
                                  int64_t batch, int n_heads, int n_kv_heads, int head_dim,
                                  int64_t num_pages, int64_t page_size, int64_t max_pages,
                                  int64_t window, int64_t n_first, float softmax_scale,
                                  void* workspace, size_t workspace_bytes, void* stream) {
  using namespace dsa;
  using namespace dsa::paged;
  if (batch < 0 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads != 0 || num_pages < 1 ||
      page_size < 1 || max_pages < 1 || window < 0 || n_first < 0)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!(softmax_scale > 0.f) || softmax_scale > 3.0e38f) return DSA_ERR_INVALID_ARGUMENT;
  if (dtype != DSA_DTYPE_BF16 && dtype != DSA_DTYPE_FP16) return DSA_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return DSA_ERR_UNSUPPORTED;
  const int g = n_heads / n_kv_heads;
  if (g > 128 || page_size % 8 != 0 || page_size > (1 << 20) || num_pages > 0x7FFFFFFF ||
      max_pages > (int64_t{1} << 28) || max_pages * page_size > (int64_t{1} << 28) ||
      batch > 65535 || batch * n_heads > (int64_t{1} << 28) ||
      batch * n_kv_heads * max_chunks(max_pages, page_size) > 0x7FFFFFFF)
    return DSA_ERR_UNSUPPORTED;
  if (batch == 0) return DSA_OK;
  if (q == nullptr || k_pages == nullptr || v_pages == nullptr || block_table == nullptr ||
      lens == nullptr || out == nullptr)
    return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(q) || !aligned16(k_pages) || !aligned16(v_pages) || !aligned16(out))
    return DSA_ERR_MISALIGNED;
  const Plan pl = plan_paged(batch, n_heads, n_kv_heads, head_dim, max_pages, page_size,
                             weights != nullptr);
  if (workspace == nullptr || workspace_bytes < pl.bytes) return DSA_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return DSA_ERR_MISALIGNED;
  DeviceInfo di;
  int st = current_device_info(&di);
  if (st != DSA_OK) return st;
  if (di.max_smem_optin < kMaxSmem) return DSA_ERR_UNSUPPORTED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Params p;
  p.batch = static_cast<int>(batch);
  p.h = n_heads;
  p.hk = n_kv_heads;
  p.g = g;
  p.page = static_cast<int>(page_size);
  p.max_pages = static_cast<int>(max_pages);
  p.gran = granule(page_size);
  p.gshift = p.gran == 32 ? 5 : (p.gran == 16 ? 4 : 3);
  p.num_pages = num_pages;
  const int64_t room = max_pages * page_size;
  p.window = static_cast<int>(window < room ? window : 0);  // at least the room: everything
  p.n_first = static_cast<int>(n_first < room ? n_first : room);
  p.table = block_table;
  p.lens = lens;
  p.scale_log2 = softmax_scale * kLog2e;
  p.sink = sink;
  p.shared = v_pages == k_pages;
  for (int i = 0; i < 3 && p.shared; ++i) {
    const bool a = k_strides == nullptr, b = v_strides == nullptr;
    p.shared = (a && b) || (!a && !b && k_strides[i] == v_strides[i]);
  }
  p.part_o = reinterpret_cast<float*>(ws);
  p.part_ml = reinterpret_cast<float2*>(ws + pl.off_ml);
  p.lse2 = reinterpret_cast<float*>(ws + pl.off_lse);
  p.scores = weights != nullptr ? reinterpret_cast<float*>(ws + pl.off_scores) : nullptr;
  p.out = out;
  p.lse = lse;
  p.weights = weights;
  p.units = pl.units;
  st = device_error_word(&p.err);
  if (st != DSA_OK) return st;
  const uint32_t fmt = dtype == DSA_DTYPE_BF16 ? win::Bf16::kFmt : win::Fp16::kFmt;
  CUtensorMap tm_q, tm_k, tm_v;
  {
    int64_t s[2] = {static_cast<int64_t>(n_heads) * head_dim, head_dim};
    if (q_strides != nullptr) {
      if (batch > 1) s[0] = q_strides[0];
      if (n_heads > 1) s[1] = q_strides[1];
    }
    for (const int64_t x : s) {
      if (x <= 0 || x >= (int64_t{1} << 38)) return DSA_ERR_UNSUPPORTED;
      if (x % 8 != 0) return DSA_ERR_MISALIGNED;
    }
    const uint64_t dims[3] = {static_cast<uint64_t>(head_dim), static_cast<uint64_t>(n_heads),
                              static_cast<uint64_t>(batch)};
    const uint64_t strides[2] = {static_cast<uint64_t>(s[1]) * 2, static_cast<uint64_t>(s[0]) * 2};
    const uint32_t box[3] = {64, static_cast<uint32_t>(g), 1};
    st = encode_tensor_map(&tm_q, win::map_type(fmt), 3, q, dims, strides, box,
                           CU_TENSOR_MAP_SWIZZLE_128B);
  }
  if (st == DSA_OK)
    st = map_pages(&tm_k, fmt, k_pages, k_strides, num_pages, page_size, n_kv_heads, head_dim, p.gran);
  if (st == DSA_OK)
    st = map_pages(&tm_v, fmt, v_pages, v_strides, num_pages, page_size, n_kv_heads, head_dim, p.gran);
  if (st != DSA_OK) return st;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    return dtype == DSA_DTYPE_BF16 ? launch<Bf16, 128>(tm_q, tm_k, tm_v, p, cs)
                                   : launch<Fp16, 128>(tm_q, tm_k, tm_v, p, cs);
  return dtype == DSA_DTYPE_BF16 ? launch<Bf16, 64>(tm_q, tm_k, tm_v, p, cs)
                                 : launch<Fp16, 64>(tm_q, tm_k, tm_v, p, cs);
}
