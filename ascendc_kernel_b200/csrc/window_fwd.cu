// Attention with a sliding window and a few first tokens that stay visible,
// forward, for sm_100a.
//
//   s_j = scale q.k_j over the keys a row sees (window_common.cuh)
//   out = sum_j e^(s_j) v_j / (sum_j e^(s_j) + e^(sink_h)),  lse = log of the divisor
// A row that sees no key and has no sink gets out = 0 and lse = -inf.
//
// One pass over the keys with a running reference (maximum) and sum in fp32.
// Per CTA (one per SM, persistent, 384 threads), a work item is two 128-row
// tiles (consecutive tokens, all heads of a group) that share every key chunk of
// up to 64 keys:
//   warp 0      TMA: q tiles, K and V chunks into a ring of stages (twice as many when
//               K and V are the same tensor and a stage holds it once).
//   warps 1, 2  tcgen05 issuers, one per tile: S = Q K^T, then O += P V with P read
//               from TMEM.
//   warps 4..11 softmax: a warpgroup per tile, a thread per row: no exchange
//               between threads for the row's maximum and sum.
// Each tile has two S buffers (P overwrites its S): PV(c) is followed by S(c + 2) into
// the buffer that it frees while the softmax is at chunk c + 1, so the scores are there
// when the softmax gets to them. One issuer for both tiles was the bottleneck: its
// waits and commits took 2,000 of the 3,400 cycles of a chunk.
// P is rounded to the operands' 16-bit type for the second product (its sum is
// taken before the rounding, in fp32): a relative 2^-8 (2^-11 for fp16, below its normal range
// 2^-25 of the row's largest P) a term at most, the size of the output's own rounding. The
// reference moves, and O is rescaled,
// only when a row's maximum exceeds it by more than 2^8, so P stays within fp16.
// TMEM per tile w: S/P buffers [256w, +64), [256w+64, +64), O [256w+128, +D).
//
// Measured (bf16, head_dim 128):
//   8 x 2600 tokens, 64 heads on one kv head, window 128 + 4: 233 us, 2.9 TB/s of q and
//   out (0.45 of a copy). An item is 4 tokens: 131 keys of the window and 4 first ones, 6
//   blocks, 3 chunks; with its start (q, the first scores) and its end (O to HBM) it takes
//   6.5 us where its bytes take 3.0; the tensor pipe is active 27 % of the time.
//   16,384 tokens, 32 heads on 8, window 4096 + 4: 1,090-1,110 us, 870 TFLOP/s (0.52 of a
//   library GEMM's burst). Tensor pipe 44 %, exponentials 45 %, issue slots 45 %: no
//   unit is full; the chain S -> maximum -> 2^x -> P -> O of a chunk is what a row's
//   thread waits for, and two tiles (all that TMEM and registers hold) hide half of it.
//   128-key chunks with one S buffer a tile, one issuer for both: 349 and 1,581 us.
#include "host_util.h"
#include "window_common.cuh"
#include "window_host.h"

namespace dsa {
namespace win {

constexpr int kThreads = 384;
// The launch holds 384 x 168 registers; the softmax warpgroups, whose threads keep
// a chunk's scores and their row's results, take 208 each and the warpgroup of TMA and MMA keeps 88:
// 128 x 88 + 256 x 208 = 384 x 168.
constexpr int kRegsAux = 88;
constexpr int kRegsSoftmax = 208;
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleLog2 = 8.0f;
constexpr int kCB = 2;  // key blocks of a chunk
constexpr int kHalfBox = kCB * kBlk * 128;  // one [64 keys x 64 columns] SW128 box

template <int D>
struct FwdCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kRows * D * 2;
  static constexpr int kSlotBytes = kCB * kBlk * D * 2;
  static constexpr int kSlots = 6;  // 6 stages of one slot (K = V) or 3 of two (K, V)
  static constexpr int kOffQ = 0;
  static constexpr int kOffKV = 2 * kTileBytes;
  static constexpr int kOffStage = kOffKV + kSlots * kSlotBytes;  // [2] tiles of results
  static constexpr int kOffBar = kOffStage + 2 * kTileBytes;
  static constexpr int kNumBars = 2 + 2 + 2 * kSlots + 4 + 4 + 4 + 2 + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 16 + 1024;
};

struct FwdParams {
  Shape s;
  TileGrid grid;
  float scale_log2;
  const float* sink;    // [h] or null
  float* lse;           // [batch, m, h] or null
  int shared;           // K and V are one tensor
  unsigned int* err;
};

template <typename T, int D>
__global__ void __launch_bounds__(kThreads, 1)
    window_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ CUtensorMap tm_out,
                      const FwdParams p) {
  using C = FwdCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;                  // [2] TMA -> MMA
  uint64_t* q_empty = q_full + 2;           // [2] last S of the tile done -> TMA
  uint64_t* kv_full = q_empty + 2;          // [stages]
  uint64_t* kv_empty = kv_full + C::kSlots; // [stages] both issuers
  uint64_t* s_full = kv_empty + C::kSlots;  // [2 tiles][2] S of a chunk in TMEM
  uint64_t* p_full = s_full + 4;            // [2 tiles][2] P written (128 arrivals)
  uint64_t* o_done = p_full + 4;            // [2 tiles][2] PV of a chunk completed
  uint64_t* o_empty = o_done + 4;           // [2] O read by the epilogue (128 arrivals)
  uint64_t* drain_bar = o_empty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int stages = p.shared ? C::kSlots : C::kSlots / 2;
  const int stage_bytes = p.shared ? C::kSlotBytes : 2 * C::kSlotBytes;

  if (threadIdx.x == 0) {
    for (int w = 0; w < 2; ++w) {
      mbar_init(&q_full[w], 1);
      mbar_init(&q_empty[w], 1);
      for (int i = 0; i < 2; ++i) {
        mbar_init(&s_full[2 * w + i], 1);
        mbar_init(&p_full[2 * w + i], 128);
        mbar_init(&o_done[2 * w + i], 1);
      }
      mbar_init(&o_empty[w], 128);
    }
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 2);
    }
    mbar_init(drain_bar, 2);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
    tma_prefetch_desc(&tm_out);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp < 4) {
    set_max_regs_dec<kRegsAux>();
  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (lane == 0) {
      Ring<0> at;
      int loads = 0;
      int uses0 = 0, uses1 = 0;
      bool ok = true;
      auto load = [&](const Item<kCB>& it, int c) -> bool {
        if (!mbar_wait(&kv_empty[at.slot], at.parity ^ 1u, abort_flag, p.err, DSA_DEVERR_WIN_WAIT))
          return false;
        const int nb = it.blocks(c);
        uint8_t* dst = smem + C::kOffKV + at.slot * stage_bytes;
        mbar_arrive_expect_tx(&kv_full[at.slot],
                              static_cast<uint32_t>(nb * kBlk * D * 2 * (p.shared ? 1 : 2)));
        for (int kind = 0; kind < (p.shared ? 1 : 2); ++kind) {
          const CUtensorMap* tm = kind == 0 ? &tm_k : &tm_v;
          for (int i = 0; i < nb; ++i) {
            const int key = it.r.key(c * kCB + i);
#pragma unroll
            for (int half = 0; half < C::kHalves; ++half)
              tma_load_4d(dst + kind * C::kSlotBytes + half * kHalfBox + i * kBlk * 128, tm, half * 64,
                          key, it.kvh, it.b, &kv_full[at.slot]);
          }
        }
        at.next(stages);
        ++loads;
        return true;
      };
      auto load_q = [&](const Item<kCB>& it, int w, int& uses) -> bool {
        if (it.last(w) < 0) return true;
        if (!mbar_wait(&q_empty[w], (uses & 1) ^ 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT))
          return false;
        uint8_t* qs = smem + C::kOffQ + w * C::kTileBytes;
        mbar_arrive_expect_tx(&q_full[w], static_cast<uint32_t>(p.grid.tt * p.s.g * D * 2));
#pragma unroll
        for (int half = 0; half < C::kHalves; ++half)
          tma_load_4d(qs + half * kBoxBytes, &tm_q, half * 64, it.kvh * p.s.g, it.t0(w), it.b,
                      &q_full[w]);
        ++uses;
        return true;
      };
      for (ItemWalk wk(p.s, p.grid); ok && wk.item < p.grid.items; wk.next(p.s, p.grid)) {
        const Item<kCB> it = make_item<kCB>(p.s, p.grid, wk);
        if (it.chunks > 0) ok = load(it, 0);
        ok = ok && load_q(it, 0, uses0) && load_q(it, 1, uses1);
        for (int c = 1; c < it.chunks && ok; ++c) ok = load(it, c);
      }
      // copies in flight land before the CTA's shared memory goes away
      for (int i = max(loads - stages, 0); i < loads; ++i)
        mbar_drain(&kv_full[i % stages], (i / stages) & 1);
      if (uses0 > 0) mbar_drain(&q_full[0], (uses0 - 1) & 1);
      if (uses1 > 0) mbar_drain(&q_full[1], (uses1 - 1) & 1);
    }
  } else if (warp == 1 || warp == 2) {
    // ------------------------------------------------------------ MMA issuers
    // the whole warp walks and waits; one elected lane issues
    {
      const int w = warp - 1;
      constexpr uint32_t idesc_o = make_idesc<T>(128, D, 1);
      const uint64_t dq = make_smem_desc(smem_u32(smem + C::kOffQ), 16u, 1024u, kLayoutSW128);
      const uint64_t dk = make_smem_desc(smem_u32(smem + C::kOffKV), 16u, 1024u, kLayoutSW128);
      const uint32_t hi = static_cast<uint32_t>(dk >> 32);
      const uint32_t q_lo = static_cast<uint32_t>(dq);
      const uint32_t k_lo = static_cast<uint32_t>(dk);
      const uint32_t v_lo = static_cast<uint32_t>(make_smem_desc(
          smem_u32(smem + C::kOffKV), static_cast<uint32_t>(kHalfBox), 1024u, kLayoutSW128));
      Ring<0> at;  // the next stage
      bool ok = true;
      auto wait_warp = [&](uint64_t* b, uint32_t parity) -> bool {
        return mbar_wait_warp(b, parity, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
      };
      auto commit = [&](uint64_t* b) {
        if (elect_one()) umma_commit(b);
        __syncwarp();
      };
      // waits for the next stage and returns its number
      auto take = [&]() -> int {
        const int s = at.slot;
        ok = ok && wait_warp(&kv_full[s], at.parity);
        at.next(stages);
        return s;
      };
      int gs = 0, go = 0, uses = 0;  // S and PV products issued, items
      auto issue_s = [&](const Item<kCB>& it, int c, int slot) {
        if (!ok || !it.active(w, c)) return;
        // the buffer's P was read by the PV product before the last one
        const int buf = 2 * w + (gs & 1);
        if (gs >= 2) ok = wait_warp(&o_done[buf], ((gs - 2) >> 1) & 1);
        if (!ok) return;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(w * 256 + (gs & 1) * 64);
        const uint32_t qa = q_lo + static_cast<uint32_t>(w * (C::kTileBytes >> 4));
        const uint32_t kb = k_lo + static_cast<uint32_t>(slot * (stage_bytes >> 4));
        const uint32_t idesc_s =
            make_idesc<T>(128, 0, 0) | (static_cast<uint32_t>(it.blocks(c) * kBlk / 8) << 17);
        const bool end = c == it.last(w);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t ao = static_cast<uint32_t>(((k >> 2) * kBoxBytes + (k & 3) * 32) >> 4);
            const uint32_t bo = static_cast<uint32_t>(((k >> 2) * kHalfBox + (k & 3) * 32) >> 4);
            umma_bf16(d, desc_from_words(qa + ao, hi), desc_from_words(kb + bo, hi), idesc_s,
                      k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[buf]);
          if (end) umma_commit(&q_empty[w]);
        }
        __syncwarp();
        ++gs;
      };
      // PV of chunk c; the stage is given back
      auto issue_pv = [&](const Item<kCB>& it, int c, int slot) {
        if (!ok) return;
        if (!it.active(w, c)) {
          commit(&kv_empty[slot]);
          return;
        }
        const bool fresh = c == it.first(w);
        const int buf = 2 * w + (go & 1);
        ok = wait_warp(&p_full[buf], (go >> 1) & 1);
        if (ok && fresh && uses > 1) ok = wait_warp(&o_empty[w], (uses - 2) & 1);
        if (!ok) return;
        tc_fence_after();
        const uint32_t sp = tmem + static_cast<uint32_t>(w * 256 + (go & 1) * 64);
        const uint32_t od = tmem + static_cast<uint32_t>(w * 256 + 128);
        const uint32_t vb =
            v_lo + static_cast<uint32_t>((slot * stage_bytes + stage_bytes - C::kSlotBytes) >> 4);
        const int nb = it.blocks(c);
        const uint32_t more = fresh ? 0u : 1u;
        if (elect_one()) {
#pragma unroll
          for (int st = 0; st < kCB * 2; ++st)  // 16 keys a step, 8 TMEM columns of P
            if (st < nb * 2)
              umma_bf16_tmem_a(od, sp + static_cast<uint32_t>(st * 8),
                               desc_from_words(vb + static_cast<uint32_t>(st * 128), hi), idesc_o,
                               st > 0 ? 1u : more);
          umma_commit(&o_done[buf]);
          umma_commit(&kv_empty[slot]);
        }
        __syncwarp();
        ++go;
      };
      // V rows at or past kv_len may hold anything, and 0 x NaN is NaN: they are
      // cleared before the product that reads them (by both issuers, to the same zeros)
      auto clear_tail = [&](const Item<kCB>& it, int c, int slot) {
        uint8_t* base = smem + C::kOffKV + slot * stage_bytes + stage_bytes - C::kSlotBytes;
        bool wrote = false;
        for (int i = 0; i < it.blocks(c); ++i) {
          const int key = it.r.key(c * kCB + i);
          for (int r = max(it.kv_len - key, 0); r < kBlk; ++r) {
            wrote = true;
            if (int x = lane; x < C::kHalves * 8)
              st_shared_v4(smem_u32(base + (x >> 3) * kHalfBox + (i * kBlk + r) * 128 + (x & 7) * 16),
                           0u, 0u, 0u, 0u);
          }
        }
        if (wrote) fence_proxy_async_smem();
        __syncwarp();
      };
      for (ItemWalk wk(p.s, p.grid); ok && wk.item < p.grid.items; wk.next(p.s, p.grid)) {
        const Item<kCB> it = make_item<kCB>(p.s, p.grid, wk);
        const int n = it.chunks;
        if (n == 0) continue;
        // stages of chunks c, c + 1 and c + 2; the other issuer takes the same
        int s0 = take(), s1 = 0, s2 = 0;
        if (it.last(w) >= 0) ok = ok && wait_warp(&q_full[w], uses++ & 1);
        issue_s(it, 0, s0);
        if (n > 1) {
          s1 = take();
          issue_s(it, 1, s1);
        }
        for (int c = 0; c < n && ok; ++c) {
          if (p.s.kv_lens != nullptr) clear_tail(it, c, s0);
          issue_pv(it, c, s0);
          if (c + 2 < n) {
            s2 = take();
            issue_s(it, c + 2, s2);
          }
          s0 = s1;
          s1 = s2;
        }
      }
      commit(drain_bar);
      mbar_drain(drain_bar, 0);
      __syncwarp();
    }
  }
  } else {
    // ------------------------------------------------------------ softmax
    set_max_regs_inc<kRegsSoftmax>();
    const int w = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int tok = row / p.s.g;
    const int head = row - tok * p.s.g;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t st = tmem + lane_off + static_cast<uint32_t>(w * 256);
    const uint32_t od = st + 128u;
    uint8_t* stage = smem + C::kOffStage + w * C::kTileBytes;
    const uint32_t stage_row = smem_u32(stage) + static_cast<uint32_t>(row * 128);
    const uint32_t bar = 1 + static_cast<uint32_t>(w);
    const bool leader = quarter == 0 && lane == 0;  // issues the tile's stores
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    int gc = 0;  // chunks processed (all items)
    bool ok = true;
    for (ItemWalk wk(p.s, p.grid); wk.item < p.grid.items; wk.next(p.s, p.grid)) {
      const Item<kCB> it = make_item<kCB>(p.s, p.grid, wk);
      const int first = it.first(w), last = it.last(w);
      const int t = it.t0(w) + tok;
      const bool valid = tok < p.grid.tt && t < it.t1(w);
      // rows past the tile's tokens follow its last one: their values are not used
      const int pos = min(t, it.t1(w) - 1) + p.s.n - p.s.m;
      const int gh = it.kvh * p.s.g + head;
      float m = -INFINITY, l = 0.f;
      for (int c = first; c <= last; ++c) {
        if (!it.active(w, c)) continue;
        const int nb = it.blocks(c);
        const uint32_t buf = static_cast<uint32_t>(gc) & 1u;
        ok = mbar_wait_warp(&s_full[2 * w + buf], (gc >> 1) & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        tc_fence_after();
        const uint32_t sp = st + buf * 64u;
        uint32_t v[kCB][32];
#pragma unroll
        for (int i = 0; i < kCB; ++i)
          if (i < nb) tmem_ld_32x32b_x32_nowait(sp + static_cast<uint32_t>(i * kBlk), v[i]);
        const bool full = chunk_full<kCB>(p.s, it, it.t0(w), it.t1(w), c);
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < kCB; ++i) {
          if (i < nb) {
            tmem_wait_ld_dep(v[i]);
            if (!full) {
              const uint32_t seen = seen_bits(p.s, it.r, c * kCB + i, pos, it.kv_len);
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!((seen >> k) & 1u)) v[i][k] = 0xFF800000u;
            }
            float a[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
              a[k] = fmaxf(__uint_as_float(v[i][k]), __uint_as_float(v[i][k + 4]));
#pragma unroll
            for (int k = 8; k < 32; k += 8) {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                a[j] = fmax3(a[j], __uint_as_float(v[i][k + j]), __uint_as_float(v[i][k + j + 4]));
            }
            mx = fmax3(mx, fmaxf(a[0], a[1]), fmaxf(a[2], a[3]));
          }
        }
        const float mz = mx * p.scale_log2;
        if (c == first) {
          m = fmaxf(m, mz);  // nothing accumulated yet
        } else {
          float factor = 1.f;
          if (mz > m + kRescaleLog2) {  // m = -inf: l and O are 0
            factor = ex2_approx(m - mz);
            m = mz;
            l *= factor;
          }
          if (__any_sync(0xFFFFFFFFu, factor != 1.f)) {
            // O holds the previous chunk's product once that completed (the one before
            // it completed before this chunk's S was issued)
            ok = mbar_wait_warp(&o_done[2 * w + (buf ^ 1u)], ((gc - 1) >> 1) & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int q = 0; q < D / 32; ++q) {
              uint32_t ov[32];
              tmem_ld_32x32b_x32(od + static_cast<uint32_t>(q * 32), ov);
#pragma unroll
              for (int k = 0; k < 32; ++k) ov[k] = __float_as_uint(__uint_as_float(ov[k]) * factor);
              tmem_st_32x32b_x32(od + static_cast<uint32_t>(q * 32), ov);
            }
          }
        }
        const float ref = m == -INFINITY ? 0.f : m;
        const uint64_t neg2 = f2_pack(-ref, -ref);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int i = 0; i < kCB; ++i) {
          if (i < nb) {
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float d0, d1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(v[i][2 * k]), __uint_as_float(v[i][2 * k + 1])),
                               scale2, neg2),
                        d0, d1);
              const float e0 = ex2_approx(d0), e1 = ex2_approx(d1);
              sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(e0, e1));
              pk[k] = T::pack(e0, e1);
            }
            tmem_st_x16_nowait(sp + static_cast<uint32_t>(i * 16), pk);
          }
        }
        float a0, a1, b0, b1;
        f2_unpack(sum2[0], a0, a1);
        f2_unpack(sum2[1], b0, b1);
        l += (a0 + a1) + (b0 + b1);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[2 * w + buf]);
        ++gc;
      }
      // ---- epilogue. The previous item's rows have left the staging buffer; a warpgroup
      // leaves together, since it meets at barriers
      if (leader) bulk_wait_group_read<0>();
      if (!named_bar_and(bar, 128, ok)) break;
      if (last >= 0) {
        // a wait that runs out here ends the loop at the next item's barrier
        ok = mbar_wait_warp(&o_done[2 * w + ((gc - 1) & 1)], ((gc - 1) >> 1) & 1, abort_flag, p.err,
                            DSA_DEVERR_WIN_WAIT);
        tc_fence_after();
      }
      // O / (l + sink term), both relative to the larger of the reference and the sink
      const float sink2 =
          p.sink != nullptr && tok < p.grid.tt ? __ldg(p.sink + gh) * kLog2e : -INFINITY;
      const float top = fmaxf(m, sink2);
      const float ref = top == -INFINITY ? 0.f : top;
      const float mine = ex2_approx(m - ref);  // 0 when no key was seen
      const float total = fmaf(l, mine, ex2_approx(sink2 - ref));
      const float inv = total == 0.f ? 0.f : mine / total;
#pragma unroll
      for (int half = 0; half < C::kHalves; ++half) {
        uint32_t ov[2][32];
        if (last >= 0) {
          tmem_ld_32x32b_x32_nowait(od + static_cast<uint32_t>(half * 64), ov[0]);
          tmem_ld_32x32b_x32_nowait(od + static_cast<uint32_t>(half * 64 + 32), ov[1]);
          tmem_wait_ld_dep(ov[0]);
          tmem_wait_ld_dep(ov[1]);
          if (half == C::kHalves - 1) {
            tc_fence_before();
            mbar_arrive(&o_empty[w]);
          }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          uint32_t x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int k = (j & 3) * 8 + 2 * u;
            x[u] = last < 0 ? 0u
                            : T::pack(__uint_as_float(ov[j >> 2][k]) * inv,
                                      __uint_as_float(ov[j >> 2][k + 1]) * inv);
          }
          st_shared_v4(stage_row + static_cast<uint32_t>(half * kBoxBytes) +
                           ((static_cast<uint32_t>(j) ^ static_cast<uint32_t>(row & 7)) << 4),
                       x[0], x[1], x[2], x[3]);
        }
      }
      fence_proxy_async_smem();
      named_bar_sync(bar, 128);
      if (leader && it.t1(w) > it.t0(w)) {
#pragma unroll
        for (int half = 0; half < C::kHalves; ++half)
          tma_store_4d(&tm_out, stage + half * kBoxBytes, half * 64, it.kvh * p.s.g, it.t0(w), it.b);
        bulk_commit_group();
      }
      if (valid && p.lse != nullptr)
        p.lse[(static_cast<int64_t>(it.b) * p.s.m + t) * p.s.h + gh] = (ref + log2f(total)) * kLn2;
    }
    if (leader) bulk_wait_group<0>();
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemCols);
  }
}

template <typename T, int D>
int launch_fwd(const Tensors& x, const Shape& s, int64_t batch, float scale, const float* sink,
               void* out, float* lse, cudaStream_t stream) {
  using C = FwdCfg<D>;
  DeviceInfo di;
  int st = current_device_info(&di);
  if (st != DSA_OK) return st;
  if (di.max_smem_optin < C::kSmemBytes) return DSA_ERR_UNSUPPORTED;
  unsigned int* err = nullptr;
  st = device_error_word(&err);
  if (st != DSA_OK) return st;
  FwdParams p;
  p.s = s;
  if (!tile_grid(s, batch, &p.grid)) return DSA_ERR_UNSUPPORTED;
  p.scale_log2 = scale * kLog2e;
  p.sink = sink;
  p.lse = lse;
  p.shared = x.v == x.k && same_strides(x.vs, x.ks);
  p.err = err;
  CUtensorMap tm_q, tm_k, tm_v, tm_out;
  st = map_rows_by_head(&tm_q, T::kFmt, x.q, x.qs, batch, s.m, s.h, D, s.g, p.grid.tt);
  if (st == DSA_OK) st = map_head_by_rows(&tm_k, T::kFmt, x.k, x.ks, batch, s.n, s.hk, D, kBlk);
  if (st == DSA_OK) st = map_head_by_rows(&tm_v, T::kFmt, x.v, x.vs, batch, s.n, s.hk, D, kBlk);
  if (st == DSA_OK) {
    Strides os;
    os.h = D;
    os.t = static_cast<int64_t>(s.h) * D;
    os.b = os.t * s.m;
    st = map_rows_by_head(&tm_out, T::kFmt, out, os, batch, s.m, s.h, D, s.g, p.grid.tt);
  }
  if (st != DSA_OK) return st;
  auto kernel = window_fwd_kernel<T, D>;
  st = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), C::kSmemBytes);
  if (st != DSA_OK) return st;
  const int grid = p.grid.items < di.num_sms ? p.grid.items : di.num_sms;
  kernel<<<static_cast<unsigned>(grid), kThreads, C::kSmemBytes, stream>>>(tm_q, tm_k, tm_v, tm_out,
                                                                              p);
  return cuda_status(cudaGetLastError());
}

}  // namespace win
}  // namespace dsa

extern "C" int dsa_window_attn_fwd(const void* q, const int64_t* q_strides, const void* k,
                                   const int64_t* k_strides, const void* v,
                                   const int64_t* v_strides, const float* sink, const int* kv_lens,
                                   void* out, float* lse, int dtype, int64_t batch, int64_t m,
                                   int64_t n, int n_heads, int n_kv_heads, int head_dim,
                                   int64_t window, int64_t n_first, float softmax_scale,
                                   void* stream) {
  using namespace dsa;
  using namespace dsa::win;
  Tensors x;
  Shape s;
  const int st = check_window_args(q, q_strides, k, k_strides, v, v_strides, kv_lens, dtype, batch,
                                   m, n, n_heads, n_kv_heads, head_dim, window, n_first,
                                   softmax_scale, &x, &s);
  if (st != DSA_OK) return st;
  if (batch == 0 || m == 0) return DSA_OK;
  if (out == nullptr) return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(out)) return DSA_ERR_MISALIGNED;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (head_dim == 128)
    return dtype == DSA_DTYPE_BF16
               ? launch_fwd<Bf16, 128>(x, s, batch, softmax_scale, sink, out, lse, cs)
               : launch_fwd<Fp16, 128>(x, s, batch, softmax_scale, sink, out, lse, cs);
  return dtype == DSA_DTYPE_BF16
             ? launch_fwd<Bf16, 64>(x, s, batch, softmax_scale, sink, out, lse, cs)
             : launch_fwd<Fp16, 64>(x, s, batch, softmax_scale, sink, out, lse, cs);
}
