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
//   warp 0      TMA: pages -> ring of 128-row slots (K, V; one slot a chunk when they
//               are one tensor), in granules of 8, 16 or 32 rows that never cross a
//               page; rows of q
//   warp 1      tcgen05 issuer
//   warps 4..11 softmax: warpgroup w takes the chunks of parity w, with its own
//               accumulator, reference and sums
// The reference of a head is set by a warpgroup's first chunk of a piece and
// moves (O and the sums are rescaled) only when a score exceeds it by more than
// 2^8, so the common chunk needs one vote and no reduction over keys; the sums
// stay per thread until the piece ends. P is rounded to the operands' type
// (relative 2^-8 at most for bf16, the size of the output's own rounding); sums are fp32.
// TMEM: S^T of warpgroup w [w NM, +NM), O^T [2 NM + w NM, +NM).
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
constexpr float kRescaleLog2 = 8.0f;
constexpr float kNone = -1.0e30f;   // reference of a piece without a visible key

template <int D, int NM>
struct Cfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kSlotBytes = kKeys * D * 2;
  static constexpr int kSlots = (NM == 128 ? 3 : 4) * (128 / D);
  static constexpr int kQBufs = NM == 128 ? 1 : 2;
  static constexpr int kQBytes = NM * D * 2;
  static constexpr int kPBytes = kKeys * NM * 2;
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = kOffQ + kQBufs * kQBytes;
  // the second 64-column half of V^T that a 64-wide head lacks is read from the
  // next slot, past the last one from P: rows 64.. of O^T are not used
  static constexpr int kOffP = kOffKV + kSlots * kSlotBytes;
  static constexpr int kOffMax = kOffP + 2 * kPBytes;         // [2][4 warps][NM] f32
  static constexpr int kOffRef = kOffMax + 2 * 4 * NM * 4;    // [2][2: reference, factor][NM]
  static constexpr int kOffMeta = kOffRef + 2 * 2 * NM * 4;   // [slot][16] granule states
  static constexpr int kOffBar = kOffMeta + kSlots * 16 * 4;
  static constexpr int kNumBars = 2 * kQBufs + 2 * kSlots + 2 + 2 + 2 + 2 + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 48 + 1024;
  static constexpr uint32_t kTmemCols = 4 * NM;
};

struct Params {
  int batch, h, hk, g;
  int page, max_pages, gran;  // page size, table width, rows of a granule
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
  s.start = s.lo - s.lo % p.gran;
  s.nfg = (s.nf + p.gran - 1) / p.gran;
  const int per = kKeys / p.gran;
  const int n = s.nfg + (s.len - s.start + p.gran - 1) / p.gran;
  s.chunks = (n + per - 1) / per;
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

// Chunks of all sequences before b and of the whole batch, summed by one warp.
__device__ __forceinline__ void chunk_sums(const Params& p, int b, int64_t* before, int64_t* all) {
  int64_t x = 0, y = 0;
  for (int i = threadIdx.x & 31; i < p.batch; i += 32) {
    const int n = seq_chunks(p, i);
    y += n;
    if (i < b) x += n;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
    y += __shfl_xor_sync(0xFFFFFFFFu, y, o);
  }
  *before = x;
  *all = y;
}

// A CTA's stretch, walked piece by piece. The line orders the chunks by (sequence,
// kv head, chunk).
struct Walk {
  int b, kvh, c0, c1;   // the piece: chunks [c0, c1) of (b, kvh)
  int64_t left;         // chunks of the stretch after this piece
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
    const int64_t n = w.s.chunks - w.c0;
    w.c1 = w.c0 + static_cast<int>(n < w.left ? n : w.left);
    w.left -= w.c1 - w.c0;
    return true;
  }
  return false;
}
__device__ __forceinline__ void walk_next(Walk& w) { w.c0 = w.c1; }

// max over the warp of a float (NaN is ignored)
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

static_assert(Cfg<128, 64>::kSmemBytes <= 232448 && Cfg<128, 128>::kSmemBytes <= 232448 &&
                  Cfg<64, 64>::kSmemBytes <= 232448 && Cfg<64, 128>::kSmemBytes <= 232448,
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
  uint64_t* q_full = bars;                    // [kQBufs]
  uint64_t* q_empty = q_full + C::kQBufs;     // [kQBufs]
  uint64_t* kv_full = q_empty + C::kQBufs;    // [kSlots]
  uint64_t* kv_empty = kv_full + C::kSlots;   // [kSlots]
  uint64_t* s_full = kv_empty + C::kSlots;    // [2] S^T of a chunk in TMEM
  uint64_t* p_full = s_full + 2;              // [2] P written (128 arrivals)
  uint64_t* o_done = p_full + 2;              // [2] O^T product of a chunk completed
  uint64_t* o_empty = o_done + 2;             // [2] O^T read at a piece's end (128 arrivals)
  uint64_t* drain_bar = o_empty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);
  int* walk_s = reinterpret_cast<int*>(smem + C::kOffMisc + 8);  // b, kvh, chunk, left (2 words)
  int* meta = reinterpret_cast<int*>(smem + C::kOffMeta);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int per = p.shared ? 1 : 2;
  const int npad = (p.g + 31) & ~31;
  const int gpc = kKeys / p.gran;  // granules of a chunk

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kQBufs; ++i) {
      mbar_init(&q_full[i], 1);
      mbar_init(&q_empty[i], 1);
    }
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&p_full[w], 128);
      mbar_init(&o_done[w], 1);
      mbar_init(&o_empty[w], 128);
    }
    mbar_init(drain_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // rows of q past the group stay 0: their scores are 0, their columns are not used
  for (int i = threadIdx.x; i < C::kQBufs * C::kQBytes / 16; i += kThreads)
    st_shared_v4(smem_u32(smem + C::kOffQ + i * 16), 0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  if (warp == 1) {
    tmem_alloc(tmem_holder, C::kTmemCols);
    tmem_relinquish();
  }
  if (warp == 2) {
    // where this CTA's stretch [first, last) of the line starts
    int64_t unused, all;
    chunk_sums(p, 0, &unused, &all);
    all *= p.hk;
    const int64_t first = all * blockIdx.x / p.units;
    const int64_t last = all * (blockIdx.x + 1) / p.units;
    int64_t base = 0;  // chunks before the 32 sequences that the lanes hold
    int b = p.batch, kvh = 0, c = 0;
    bool found = first >= last;
    for (int i0 = 0; i0 < p.batch && !found; i0 += 32) {
      const int64_t mine =
          i0 + lane < p.batch ? static_cast<int64_t>(seq_chunks(p, i0 + lane)) * p.hk : 0;
      int64_t sum = mine;  // inclusive prefix over the lanes
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xFFFFFFFFu, sum, o);
        if (lane >= o) sum += y;
      }
      const uint32_t hit = __ballot_sync(0xFFFFFFFFu, first < base + sum && mine > 0);
      if (hit != 0) {
        const int l = __ffs(hit) - 1;
        const int64_t begin = base + __shfl_sync(0xFFFFFFFFu, sum - mine, l);
        const int64_t n = __shfl_sync(0xFFFFFFFFu, mine, l) / p.hk;
        b = i0 + l;
        kvh = static_cast<int>((first - begin) / n);
        c = static_cast<int>((first - begin) - static_cast<int64_t>(kvh) * n);
        found = true;
      }
      base += __shfl_sync(0xFFFFFFFFu, sum, 31);
    }
    if (lane == 0) {
      walk_s[0] = b;
      walk_s[1] = kvh;
      walk_s[2] = c;
      *reinterpret_cast<int64_t*>(walk_s + 4) = last > first ? last - first : 0;
      if (blockIdx.x == 0) {
        // lengths outside the table's room are clamped and reported
        bool bad = false;
        for (int i = 0; i < p.batch; ++i) {
          const int n = __ldg(p.lens + i);
          bad = bad || n < 0 || n > static_cast<int64_t>(p.max_pages) * p.page;
        }
        if (bad) atomicOr(p.err, DSA_DEVERR_CACHE);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  Walk wk;
  wk.b = walk_s[0];
  wk.kvh = walk_s[1];
  wk.c0 = walk_s[2];
  wk.left = *reinterpret_cast<const int64_t*>(walk_s + 4);

  if (warp < 4) {
    win::set_max_regs_dec<kRegsAux>();
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      int seq = 0, pieces = 0;
      bool ok = true;
      for (; ok && walk_take(p, wk); walk_next(wk), ++pieces) {
        const int qb = pieces % C::kQBufs;
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&q_empty[qb], ((pieces / C::kQBufs) & 1) ^ 1,
                                               abort_flag, p.err, DSA_DEVERR_WIN_WAIT));
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&q_full[qb], static_cast<uint32_t>(p.g * D * 2));
#pragma unroll
          for (int half = 0; half < C::kHalves; ++half)
            tma_load_3d(smem + C::kOffQ + qb * C::kQBytes + half * NM * 128, &tm_q, half * 64,
                        wk.kvh * p.g, wk.b, &q_full[qb]);
        }
        for (int c = wk.c0; ok && c < wk.c1; ++c) {
          // a lane per granule: its page, looked up while the slots are still in use
          const int i = c * gpc + lane;
          const int row = gran_row(p, wk.s, i);
          int page = -1;
          if (lane < gpc && row < wk.s.len) {
            page = page_of(p, wk.b, row);
            if (page < 0) atomicOr(p.err, DSA_DEVERR_CACHE);
          }
          const uint32_t live = __ballot_sync(0xFFFFFFFFu, page >= 0);
          const uint32_t bytes = static_cast<uint32_t>(__popc(live) * p.gran * D * 2);
          for (int kind = 0; kind < per; ++kind, ++seq) {
            const int s = seq % C::kSlots;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&kv_empty[s], ((seq / C::kSlots) & 1) ^ 1,
                                                   abort_flag, p.err, DSA_DEVERR_WIN_WAIT));
            if (!ok) break;
            if (lane < 16) meta[s * 16 + lane] = page >= 0 ? 1 : 0;
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(&kv_full[s], bytes);
            __syncwarp();
            if (page >= 0) {
              const CUtensorMap* tm = kind == 0 ? &tm_k : &tm_v;
              uint8_t* dst = smem + C::kOffKV + s * C::kSlotBytes + lane * p.gran * 128;
#pragma unroll
              for (int half = 0; half < C::kHalves; ++half)
                tma_load_4d(dst + half * kBox, tm, half * 64, row % p.page, wk.kvh, page, &kv_full[s]);
            }
          }
        }
      }
      // copies in flight land before the CTA's shared memory goes away
      for (int i = (seq > C::kSlots ? seq - C::kSlots : 0); i < seq; ++i)
        mbar_drain(&kv_full[i % C::kSlots], (i / C::kSlots) & 1);
      for (int i = (pieces > C::kQBufs ? pieces - C::kQBufs : 0); i < pieces; ++i)
        mbar_drain(&q_full[i % C::kQBufs], (i / C::kQBufs) & 1);
    } else if (warp == 1 && lane == 0) {
      // ---------------------------------------------------------- MMA issuer
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
      int gc = 0, pieces = 0;
      int gp[2] = {0, 0};       // O^T products issued per warpgroup
      int drained[2] = {0, 0};  // pieces of the warpgroup whose O^T was to be read
      int prev = -1;            // chunk whose O^T product is not yet issued
      bool prev_fresh = false;
      bool ok = true;
      auto issue_o = [&](int i, bool fresh) -> bool {
        const int w = i & 1;
        const int s = (i * per + per - 1) % C::kSlots;
        if (!mbar_wait(&kv_full[s], ((i * per + per - 1) / C::kSlots) & 1, abort_flag, p.err,
                       DSA_DEVERR_WIN_WAIT) ||
            !mbar_wait(&p_full[w], gp[w] & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT))
          return false;
        if (fresh) {
          if (drained[w] > 0 && !mbar_wait(&o_empty[w], (drained[w] - 1) & 1, abort_flag, p.err,
                                           DSA_DEVERR_WIN_WAIT))
            return false;
          ++drained[w];
        }
        tc_fence_after();
        const uint32_t va = v_lo + static_cast<uint32_t>(s * (C::kSlotBytes >> 4));
        const uint32_t pb = p_lo + static_cast<uint32_t>(w * (C::kPBytes >> 4));
        const uint32_t d = tmem + static_cast<uint32_t>((2 + w) * NM);
#pragma unroll
        for (int st = 0; st < kKeys / 16; ++st)
          umma_bf16(d, desc_from_words(va + static_cast<uint32_t>(st * 128), hi),
                    desc_from_words(pb + static_cast<uint32_t>(st * 128), hi), idesc_o,
                    (fresh && st == 0) ? 0u : 1u);
        umma_commit(&o_done[w]);
        umma_commit(&kv_empty[s]);
        ++gp[w];
        return true;
      };
      for (; ok && walk_take(p, wk); walk_next(wk), ++pieces) {
        const int qb = pieces % C::kQBufs;
        ok = mbar_wait(&q_full[qb], (pieces / C::kQBufs) & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        const int n = wk.c1 - wk.c0;
        for (int j = 0; ok && j < n; ++j, ++gc) {
          // S^T(i) while the softmax of chunk i - 1 runs. Its columns held S^T(i - 2),
          // whose readers arrived before O^T(i - 2) was issued
          const int w = gc & 1;
          const int s = (gc * per) % C::kSlots;
          ok = mbar_wait(&kv_full[s], ((gc * per) / C::kSlots) & 1, abort_flag, p.err,
                         DSA_DEVERR_WIN_WAIT);
          if (!ok) break;
          tc_fence_after();
          const uint32_t ka = k_lo + static_cast<uint32_t>(s * (C::kSlotBytes >> 4));
          const uint32_t qa = q_lo + static_cast<uint32_t>(qb * (C::kQBytes >> 4));
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t ao = static_cast<uint32_t>(((k >> 2) * kBox + (k & 3) * 32) >> 4);
            const uint32_t bo = static_cast<uint32_t>(((k >> 2) * NM * 128 + (k & 3) * 32) >> 4);
            umma_bf16(tmem + static_cast<uint32_t>(w * NM), desc_from_words(ka + ao, hi),
                      desc_from_words(qa + bo, hi), idesc_s, k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[w]);
          if (!p.shared) umma_commit(&kv_empty[s]);
          if (j == n - 1) umma_commit(&q_empty[qb]);
          if (prev >= 0) ok = issue_o(prev, prev_fresh);
          prev = gc;
          prev_fresh = j < 2;
        }
      }
      if (ok && prev >= 0) issue_o(prev, prev_fresh);
      umma_commit(drain_bar);
      mbar_drain(drain_bar, 0);
    }
  } else {
    // ------------------------------------------------------------ softmax
    win::set_max_regs_inc<kRegsSoftmax>();
    const int w = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int key = quarter * 32 + lane;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t sp = tmem + lane_off + static_cast<uint32_t>(w * NM);
    const uint32_t od = tmem + lane_off + static_cast<uint32_t>((2 + w) * NM);
    const uint32_t bar = 1 + static_cast<uint32_t>(w);
    float* wmax = reinterpret_cast<float*>(smem + C::kOffMax) + w * 4 * NM;
    float* ref = reinterpret_cast<float*>(smem + C::kOffRef) + w * 2 * NM;
    float* fac = ref + NM;
    const uint32_t prow = smem_u32(smem + C::kOffP) + static_cast<uint32_t>(w * C::kPBytes + key * 128);
    int gc = 0, gw = 0;
    bool ok = true;
    // a warpgroup leaves together: it meets at named barriers
    auto wait_all = [&](uint64_t* b, uint32_t parity) -> bool {
      return named_bar_and(bar, 128, mbar_wait(b, parity, abort_flag, p.err, DSA_DEVERR_WIN_WAIT));
    };
    for (; ok && walk_take(p, wk); walk_next(wk)) {
      float l[NM];
#pragma unroll
      for (int k = 0; k < NM; ++k) l[k] = 0.f;
      const int n = wk.c1 - wk.c0;
      bool fresh = true;
      for (int j = 0; j < n; ++j, ++gc) {
        if ((gc & 1) != w) continue;
        ok = wait_all(&s_full[w], gw & 1);
        if (!ok) break;
        const int c = wk.c0 + j;
        const int sv = (gc * per + per - 1) % C::kSlots;
        const int gi = key / p.gran;
        const int row = gran_row(p, wk.s, c * gpc + gi) + (key - gi * p.gran);
        // the granules' states are read from the V slot, which stays until this chunk's
        // weights are used (the K slot is given back as soon as S^T is done)
        ok = wait_all(&kv_full[sv], ((gc * per + per - 1) / C::kSlots) & 1);
        if (!ok) break;
        const bool valid = row_seen(wk.s, c * gpc + gi, row) && meta[sv * 16 + gi] != 0;
        tc_fence_after();
        // ---- does any score exceed its head's reference by more than 2^8?
        bool over = fresh;
        if (!fresh) {
          float excess = -INFINITY;
#pragma unroll
          for (int q = 0; q < NM / 32; ++q) {
            if (q * 32 < npad) {
              uint32_t v[32];
              tmem_ld_32x32b_x32(sp + static_cast<uint32_t>(q * 32), v);
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float4 r = reinterpret_cast<const float4*>(ref)[q * 8 + k];
                excess = fmax3(excess, fmaf(__uint_as_float(v[4 * k]), p.scale_log2, -r.x),
                               fmaf(__uint_as_float(v[4 * k + 1]), p.scale_log2, -r.y));
                excess = fmax3(excess, fmaf(__uint_as_float(v[4 * k + 2]), p.scale_log2, -r.z),
                               fmaf(__uint_as_float(v[4 * k + 3]), p.scale_log2, -r.w));
              }
            }
          }
          over = valid && excess > kRescaleLog2;
        }
        if (named_bar_or(bar, 128, over)) {
          // the heads' maxima over the chunk's keys: warps, then the warpgroup
#pragma unroll 1
          for (int q = 0; q * 32 < npad; ++q) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(sp + static_cast<uint32_t>(q * 32), v);
            float mine = 0.f;
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float m = warp_max(valid ? __uint_as_float(v[k]) * p.scale_log2 : kNone);
              if (lane == k) mine = m;
            }
            wmax[quarter * NM + q * 32 + lane] = mine;
          }
          named_bar_sync(bar, 128);
          if (key < npad) {
            const float m = fmaxf(fmaxf(wmax[key], wmax[NM + key]),
                                  fmaxf(wmax[2 * NM + key], wmax[3 * NM + key]));
            const float old = fresh ? m : ref[key];
            const float now = m > old + kRescaleLog2 ? m : old;
            ref[key] = now;
            fac[key] = ex2_approx(old - now);
          }
          named_bar_sync(bar, 128);
          if (!fresh) {
            ok = wait_all(&o_done[w], (gw - 1) & 1);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int q = 0; q < NM / 32; ++q) {
              if (q * 32 < npad) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(od + static_cast<uint32_t>(q * 32), v);
#pragma unroll
                for (int k = 0; k < 32; ++k) {
                  const float f = fac[q * 32 + k];
                  l[q * 32 + k] *= f;
                  v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                }
                tmem_st_32x32b_x32(od + static_cast<uint32_t>(q * 32), v);
              }
            }
          }
        }
        // ---- P = 2^(z - reference), the key's weights of all heads
        if (gw > 0) {  // the warpgroup's previous product has read P
          ok = wait_all(&o_done[w], (gw - 1) & 1);
          if (!ok) break;
        }
        float* zrow = nullptr;
        if (p.scores != nullptr) {
          // chunks of this sequence lie [kv head][chunk] at max_chunks of the table
          const int64_t cap = (static_cast<int64_t>(p.max_pages) * p.page + kKeys - 1) / kKeys + 2;
          zrow = p.scores +
                 (((static_cast<int64_t>(wk.b) * p.hk + wk.kvh) * cap + c) * kKeys + key) * p.g;
        }
#pragma unroll
        for (int q = 0; q < NM / 32; ++q) {
          if (q * 32 < npad) {
            uint32_t v[32];
            tmem_ld_32x32b_x32(sp + static_cast<uint32_t>(q * 32), v);
            if (zrow != nullptr) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (q * 32 + k < p.g)
                  zrow[q * 32 + k] = valid ? __uint_as_float(v[k]) * p.scale_log2 : -INFINITY;
            }
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float4 r = reinterpret_cast<const float4*>(ref)[q * 8 + k];
              const float e0 = valid ? ex2_approx(fmaf(__uint_as_float(v[4 * k]), p.scale_log2, -r.x)) : 0.f;
              const float e1 = valid ? ex2_approx(fmaf(__uint_as_float(v[4 * k + 1]), p.scale_log2, -r.y)) : 0.f;
              const float e2 = valid ? ex2_approx(fmaf(__uint_as_float(v[4 * k + 2]), p.scale_log2, -r.z)) : 0.f;
              const float e3 = valid ? ex2_approx(fmaf(__uint_as_float(v[4 * k + 3]), p.scale_log2, -r.w)) : 0.f;
              l[q * 32 + 4 * k] += e0;
              l[q * 32 + 4 * k + 1] += e1;
              l[q * 32 + 4 * k + 2] += e2;
              l[q * 32 + 4 * k + 3] += e3;
              pk[2 * k] = T::pack(e0, e1);
              pk[2 * k + 1] = T::pack(e2, e3);
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
          // a hidden V row may hold anything, and 0 x NaN is NaN: it is cleared
          uint8_t* vr = smem + C::kOffKV + sv * C::kSlotBytes + key * 128;
#pragma unroll
          for (int x = 0; x < C::kHalves * 8; ++x)
            st_shared_v4(smem_u32(vr + (x >> 3) * kBox + (x & 7) * 16), 0u, 0u, 0u, 0u);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&p_full[w]);
        ++gw;
        fresh = false;
      }
      if (!ok) break;
      // ---- the piece's partial of this warpgroup
      const int64_t piece = static_cast<int64_t>(blockIdx.x) + static_cast<int64_t>(wk.b) * p.hk + wk.kvh;
      float2* ml = p.part_ml + (piece * 2 + w) * p.g;
      if (fresh) {  // it had no chunk
        for (int x = key; x < p.g; x += 128) ml[x] = make_float2(kNone, 0.f);
        continue;
      }
      ok = wait_all(&o_done[w], (gw - 1) & 1);
      if (!ok) break;
      tc_fence_after();
#pragma unroll
      for (int q = 0; q < NM / 32; ++q) {
        if (q * 32 < npad) {
          // sums over the warp's 32 keys of 32 heads: lane k ends with head k
          float a[32];
#pragma unroll
          for (int k = 0; k < 32; ++k) a[k] = l[q * 32 + k];
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) {
            const bool up = (lane & o) != 0;
#pragma unroll
            for (int k = 0; k < o; ++k) {
              const float send = up ? a[k] : a[k + o];
              a[k] = (up ? a[k + o] : a[k]) + __shfl_xor_sync(0xFFFFFFFFu, send, o);
            }
          }
          wmax[quarter * NM + q * 32 + lane] = a[0];
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
      if (key < p.g)
        ml[key] = make_float2(ref[key], (wmax[key] + wmax[NM + key]) +
                                            (wmax[2 * NM + key] + wmax[3 * NM + key]));
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

// Joins the pieces of one (sequence, head): a block of D threads, a column each.
template <typename T, int D>
__global__ void __launch_bounds__(D) paged_join_kernel(const Params p) {
  const int head = blockIdx.x % p.h;
  const int b = blockIdx.x / p.h;
  const int kvh = head / p.g, gi = head - kvh * p.g;
  const int x = threadIdx.x;
  int64_t before, all;
  chunk_sums(p, b, &before, &all);
  const int64_t n = seq_chunks(p, b);
  const int64_t first = before * p.hk + kvh * n, last = first + n;
  all *= p.hk;
  const float sink2 = p.sink != nullptr ? __ldg(p.sink + head) * kLog2e : -INFINITY;
  float top = sink2, sum = 0.f, acc = 0.f;
  if (n > 0) {
    // CTA u takes chunks [all u / units, all (u + 1) / units)
    int64_t u0 = first * p.units / all;
    while (u0 > 0 && all * u0 / p.units > first) --u0;
    while (all * (u0 + 1) / p.units <= first) ++u0;
    int64_t u1 = u0;
    while (all * (u1 + 1) / p.units < last) ++u1;
    const int64_t bh = static_cast<int64_t>(b) * p.hk + kvh;
    for (int64_t u = u0; u <= u1; ++u) {
      if (all * u / p.units == all * (u + 1) / p.units) continue;  // an empty stretch
      for (int w = 0; w < 2; ++w) {
        const int64_t at = ((u + bh) * 2 + w) * p.g + gi;
        const float2 ml = p.part_ml[at];
        if (ml.y == 0.f) continue;  // no visible key
        const float o = p.part_o[at * D + x];
        const float now = fmaxf(top, ml.x);
        const float f = top == now ? 1.f : ex2_approx(top - now), g = ex2_approx(ml.x - now);
        acc = acc * f + o * g;
        sum = sum * f + ml.y * g;
        top = now;
      }
    }
  }
  const float ref = top == -INFINITY ? 0.f : top;
  const float total = sum + (p.sink != nullptr ? ex2_approx(sink2 - ref) : 0.f);
  const float v = total == 0.f ? 0.f : acc / total;
  const uint32_t bits = T::pack(v, 0.f);
  static_cast<uint16_t*>(p.out)[static_cast<int64_t>(blockIdx.x) * D + x] =
      static_cast<uint16_t>(bits & 0xFFFFu);
  if (x == 0) {
    const float l2 = ref + log2f(total);
    p.lse2[blockIdx.x] = l2;
    if (p.lse != nullptr) p.lse[blockIdx.x] = l2 * kLn2;
  }
}

// weights[slot of key] += sum over heads of 2^(z - lse): a thread a key, heads in order.
__global__ void __launch_bounds__(kKeys) paged_weights_kernel(const Params p) {
  const int b = blockIdx.y, c = blockIdx.x;
  const Seq s = make_seq(p, b);
  if (c >= s.chunks) return;
  const int per = kKeys / p.gran;
  const int gi = threadIdx.x / p.gran;
  const int row = gran_row(p, s, c * per + gi) + (threadIdx.x - gi * p.gran);
  if (!row_seen(s, c * per + gi, row)) return;
  const int page = page_of(p, b, row);
  if (page < 0) return;
  const int64_t cap = (static_cast<int64_t>(p.max_pages) * p.page + kKeys - 1) / kKeys + 2;
  const float* lse = p.lse2 + static_cast<int64_t>(b) * p.h;
  float sum = 0.f;
  for (int kvh = 0; kvh < p.hk; ++kvh) {
    const float* z = p.scores +
                     (((static_cast<int64_t>(b) * p.hk + kvh) * cap + c) * kKeys + threadIdx.x) * p.g;
    for (int k = 0; k < p.g; ++k) sum += ex2_approx(z[k] - __ldg(lse + kvh * p.g + k));
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

// One CTA per SM of a full GPU, fewer when the batch cannot have that many chunks.
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
  int st = p.g <= 64 ? launch_split<T, D, 64>(q, k, v, p, stream)
                     : launch_split<T, D, 128>(q, k, v, p, stream);
  if (st != DSA_OK) return st;
  paged_join_kernel<T, D><<<static_cast<unsigned>(p.batch * p.h), D, 0, stream>>>(p);
  st = cuda_status(cudaGetLastError());
  if (st != DSA_OK || p.weights == nullptr) return st;
  paged_weights_kernel<<<dim3(static_cast<unsigned>(max_chunks(p.max_pages, p.page)),
                              static_cast<unsigned>(p.batch)),
                         kKeys, 0, stream>>>(p);
  return cuda_status(cudaGetLastError());
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
      batch > 65535 || batch * n_heads > (int64_t{1} << 28))
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
  const int need = g <= 64 ? (head_dim == 128 ? Cfg<128, 64>::kSmemBytes : Cfg<64, 64>::kSmemBytes)
                           : (head_dim == 128 ? Cfg<128, 128>::kSmemBytes : Cfg<64, 128>::kSmemBytes);
  if (di.max_smem_optin < need) return DSA_ERR_UNSUPPORTED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  Params p;
  p.batch = static_cast<int>(batch);
  p.h = n_heads;
  p.hk = n_kv_heads;
  p.g = g;
  p.page = static_cast<int>(page_size);
  p.max_pages = static_cast<int>(max_pages);
  p.gran = granule(page_size);
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
