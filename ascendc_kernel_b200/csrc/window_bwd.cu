// Attention with a sliding window and a few first tokens, backward, for sm_100a.
//
// With P_j = e^(s_j - lse) over the keys a row sees (window_common.cuh), D =
// rowsum(dout * out) and dS_j = P_j (dout.v_j - D):
//   dq = scale sum_j dS_j k_j      dk_j = scale sum_rows dS_j q      dv_j = sum_rows P_j dout
//   dsink_h = -sum_rows e^(sink_h - lse) D       (v the same tensor as k: dk + dv in one)
//
// Deterministic without atomics (but maxima, whose order does not matter), in up to five
// launches:
//   window_stat_kernel  per row -lse log2(e) and -D, HBM bound (out and dout read once)
//   window_dkv_kernel   a key tile stays, the rows that see it stream by (4 products)
//   window_join_kernel  sums the fp32 parts of key tiles whose rows were split
//   window_dq_kernel    a row tile stays, its keys stream by (3 products); S and dout V^T
//                       are computed again, which costs 2 products of 7 and keeps dq out of
//                       atomics, whose order would change results from run to run
//   window_dsink_*      the rows' sink terms summed in a fixed order
// P and dS are rounded to the operands' 16-bit type for the products that sum
// over them (relative 2^-8 at most for bf16, the size of the gradients' own rounding);
// every sum is fp32. D comes from the rounded out; the sink's gradient, an fp32
// output, uses the unrounded D = sum_j P_j (dout.v_j) that the dq kernel sees.
//
// fp16 is normal from 2^-14 to 2^16 only, where P has 1 / keys and dS the upstream gradient's
// size in it. Both are scaled by powers of two before they are rounded and the sums scaled back
// in fp32: P by 2^14, dP - D by the power of two that brings its bound below 1,
//   |dP - D| <= |dout| |v| + |D|
// (dk: this key's |v| and the largest |dout| and |D| of the kv head's rows; dq: this row's
// |dout| and D and the largest |v|). The scale belongs to the accumulator's row, so it leaves
// the sum. |dS| stays below 2^14, and no dS is off by more than 2^-38 of the bound. It costs
// 3 % of the gradients' time in the first case below and 9 % in the second (752 against 728
// and 394 against 362 us); unscaled, dk of an upstream gradient of 1e-5 was lost.
//
// Measured (bf16, head_dim 128), in us:
//   2 x 4096 tokens, 32 heads on 8, window 1024 + 4: dk/dv 368, dq 316, statistics 22,
//   join 9; the five products the formulas need run at 440 TFLOP/s, the seven done at
//   613. Tensor pipe 45 % (dk/dv) and 32 % (dq), issue slots 34 % and 27 %, DRAM below 8 %:
//   bound by the chain S, dP -> P, dS -> products of a tile, of which two are in flight
//   (dk/dv fills TMEM with two accumulators and two pairs of S and dP; dq has one pair a tile,
//   so that its next scores wait for the product of this chunk), and by the 64-wide products,
//   which read shared memory faster than they compute.
//   2 x 2600 tokens, 64 heads on one kv head, window 128 + 4: dk/dv 200, dq 96, statistics
//   31, join 12, dsink 6.
#include "host_util.h"
#include "window_common.cuh"
#include "window_host.h"

namespace dsa {
namespace win {

constexpr int kBwdThreads = 384;
constexpr int kBwdRegsAux = 88;       // 128 x 88 + 256 x 208 = 384 x 168 at launch
constexpr int kBwdRegsSoftmax = 208;
constexpr uint32_t kBwdTmemCols = 512;
constexpr int kCB = 2;                // key blocks of a chunk (dq), 64 keys
constexpr int kStream = 64;           // rows of a streamed tile (dkv)
constexpr int kHalfBox = kStream * 128;  // one [64 rows x 64 columns] SW128 box

// ------------------------------------------------------------------ scales (fp16)
constexpr float kPUp = 14.f;                // P is rounded as 2^kPUp P
constexpr float kPDown = 1.f / 16384.f;

// Largest norms and magnitudes of one (batch, kv head) as bits of non-negative floats, whose
// order is the values' (a maximum does not depend on the order of its atomics).
struct Peak {
  uint32_t dout, d, v;
};
__device__ __forceinline__ void raise(uint32_t* peak, uint32_t bits) {
  if (bits > *static_cast<volatile uint32_t*>(peak)) atomicMax(peak, bits);
}

// The power of two f that brings bound f to [1/2, 1); 1 where the bound is 0 or not finite.
__device__ __forceinline__ float power_below(float bound) {
  const uint32_t e = __float_as_uint(bound) >> 23;  // bound >= 0 or NaN
  return e >= 27u && e < 250u ? __uint_as_float((253u - e) << 23) : 1.f;
}
// What a sum of dS 2^kPUp f is scaled by.
__device__ __forceinline__ float scale_down(float scale, float f) {
  return scale * (kPDown * __uint_as_float((254u << 23) - __float_as_uint(f)));  // 1 / f
}

// ------------------------------------------------------------------ row statistics
// stat[row] = (-lse log2 e, -D); D / 8 threads a row, each with kStatRows rows' 16-byte
// loads in flight: 22 us for 2 x 4096 x 32 rows of 128, 5.9 TB/s (one row a thread: 31 us,
// 4.3 TB/s). Flat: dout is contiguous like out. With fp16 also norm[row] = |dout| and the
// peaks of the rows that see something.
constexpr int kStatRows = 4;

template <typename T, int D, bool Flat>
__global__ void __launch_bounds__(256) window_stat_kernel(const uint16_t* out, const uint16_t* dout,
                                                          Strides ds, const float* lse, float2* stat,
                                                          float* norm, Peak* peaks, int64_t rows,
                                                          int m, int h, int g) {
  constexpr int kLanes = D / 8;
  constexpr int kStep = 256 / kLanes;  // rows of a block at once
  // fp16: maxima of the block's (token, kv head) groups of rows, which then raise the peaks:
  // an atomic a row took 75 us more
  __shared__ uint32_t top[T::kNarrow ? 2 : 1][T::kNarrow ? kStep * kStatRows + 1 : 1];
  const int64_t group0 = static_cast<int64_t>(blockIdx.x) * (kStep * kStatRows) / g;
  if constexpr (T::kNarrow) {
    for (int i = threadIdx.x; i <= kStep * kStatRows; i += 256) top[0][i] = top[1][i] = 0u;
    __syncthreads();
  }
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * (kStep * kStatRows) + threadIdx.x / kLanes;
  const int x = threadIdx.x % kLanes;
  uint4 a[kStatRows], up[kStatRows];
#pragma unroll
  for (int r = 0; r < kStatRows; ++r) {
    const int64_t row = row0 + r * kStep;
    a[r] = up[r] = make_uint4(0u, 0u, 0u, 0u);
    if (row < rows) {
      int64_t at = row * D;
      a[r] = __ldcs(reinterpret_cast<const uint4*>(out + at + x * 8));
      if (!Flat) {
        const int64_t bt = row / h;
        const int64_t b = bt / m;
        at = b * ds.b + (bt - b * m) * ds.t + (row - bt * h) * ds.h;
      }
      up[r] = *reinterpret_cast<const uint4*>(dout + at + x * 8);
    }
  }
#pragma unroll
  for (int r = 0; r < kStatRows; ++r) {
    const int64_t row = row0 + r * kStep;
    const uint32_t aw[4] = {a[r].x, a[r].y, a[r].z, a[r].w};
    const uint32_t gw[4] = {up[r].x, up[r].y, up[r].z, up[r].w};
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      sum = fmaf(T::lo(aw[i]), T::lo(gw[i]), sum);
      sum = fmaf(T::hi(aw[i]), T::hi(gw[i]), sum);
    }
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    float sq = 0.f;
    if constexpr (T::kNarrow) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sq = fmaf(T::lo(gw[i]), T::lo(gw[i]), sq);
        sq = fmaf(T::hi(gw[i]), T::hi(gw[i]), sq);
      }
#pragma unroll
      for (int o = kLanes / 2; o > 0; o >>= 1) sq += __shfl_xor_sync(0xFFFFFFFFu, sq, o);
    }
    if (row < rows && x == 0) {
      const float l = lse[row];
      if constexpr (T::kNarrow) {
        const float size = sqrtf(sq);
        norm[row] = size;
        if (l != -INFINITY) {
          const int i = static_cast<int>(row - group0 * g) / g;
          atomicMax(&top[0][i], __float_as_uint(size));
          atomicMax(&top[1][i], __float_as_uint(fabsf(sum)));
        }
      }
      // a row that sees nothing has no weights: 2^(s - inf) = 0
      stat[row] = make_float2(l == -INFINITY ? -INFINITY : -l * kLog2e, -sum);
    }
  }
  if constexpr (T::kNarrow) {
    __syncthreads();
    const int hk = h / g;
    for (int i = threadIdx.x; i <= kStep * kStatRows; i += 256) {
      if ((top[0][i] | top[1][i]) != 0u) {
        const int64_t bt = (group0 + i) / hk;
        Peak* peak = peaks + (bt / m) * hk + (group0 + i - bt * hk);
        raise(&peak->dout, top[0][i]);
        raise(&peak->d, top[1][i]);
      }
    }
  }
}

// ------------------------------------------------------------------ dk, dv
template <int D>
struct DkvCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kRows * D * 2;
  static constexpr int kStageBytes = 2 * kStream * D * 2;  // q rows, dout rows
  static constexpr int kStages = 4;
  static constexpr int kOffK = 0;
  static constexpr int kOffV = kTileBytes;
  static constexpr int kOffS = 2 * kTileBytes;
  static constexpr int kOffStat = kOffS + kStages * kStageBytes;  // [stage][2][64] f32
  static constexpr int kOffStage = kOffStat + kStages * 2 * kStream * 4;  // [8 warps] 2 KB
  static constexpr int kOffBar = kOffStage + 8 * 2048;
  static constexpr int kNumBars = 2 + 2 * kStages + 2 + 2 + 2 + 2 + 2 + 1 + 1 + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 16 + 1024;
};

struct DkvParams {
  Shape s;
  int gb, hb, tt;        // heads and tokens of a streamed tile, head parts of a group
  int key_tiles;         // per (batch, kv head)
  int first_tiles;       // of them, those with first tokens (every later row sees them)
  int split_first, split;  // units of a key tile
  int units_per_head;
  int64_t units;
  float scale, scale_log2;
  const float2* stat;    // [batch, m, h]
  uint16_t* dk;          // [batch, n, hk, D]
  uint16_t* dv;          // null: dk receives dk + dv
  float* parts;          // [unit][dv ? 2 : 1][128][D] of the key tiles with several units
  unsigned int* err;
};

// Tokens [ta, tb) that see a key of tile kt (an upper bound when kv_lens is short).
__host__ __device__ __forceinline__ void dkv_tokens(const Shape& s, int kt, int* ta, int* tb) {
  const int off = s.n - s.m;
  const int k0 = kt * kRows;
  const int64_t top = k0 < s.n_first ? s.n : static_cast<int64_t>(k0) + kRows - 1 + s.window;
  const int pe = top < s.n ? static_cast<int>(top) : s.n;  // positions [k0, pe)
  *ta = k0 - off > 0 ? k0 - off : 0;
  *tb = pe - off > *ta ? pe - off : *ta;
}

struct Unit {
  int b, kvh, kv_len;
  int kt, part, parts;
  int ta, tb;      // tokens of the key tile
  int r0, r1;      // streamed tiles of the unit
};

__device__ __forceinline__ Unit make_unit(const DkvParams& p, int64_t unit) {
  Unit u;
  const int64_t bh = unit / p.units_per_head;
  int x = static_cast<int>(unit - bh * p.units_per_head);
  u.b = static_cast<int>(bh / p.s.hk);
  u.kvh = static_cast<int>(bh - static_cast<int64_t>(u.b) * p.s.hk);
  u.kv_len = kv_len_of(p.s, u.b);
  const int heavy = p.first_tiles * p.split_first;
  if (x < heavy) {
    u.parts = p.split_first;
    u.kt = x / p.split_first;
    u.part = x - u.kt * p.split_first;
  } else {
    x -= heavy;
    u.parts = p.split;
    u.kt = x / p.split;
    u.part = x - u.kt * p.split;
    u.kt += p.first_tiles;
  }
  dkv_tokens(p.s, u.kt, &u.ta, &u.tb);
  if (u.kt * kRows >= u.kv_len) u.tb = u.ta;
  const int64_t tiles = static_cast<int64_t>((u.tb - u.ta + p.tt - 1) / p.tt) * p.hb;
  u.r0 = static_cast<int>(tiles * u.part / u.parts);
  u.r1 = static_cast<int>(tiles * (u.part + 1) / u.parts);
  return u;
}

// peaks (fp16 only): of the rows when the kernel starts; the keys' norms are added. A
// parameter of its own: inside DkvParams it cost the bf16 kernel 12 bytes of spills and 1 %.
template <typename T, int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    window_dkv_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                      const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                      const DkvParams p, Peak* peaks) {
  using C = DkvCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* kv_full = bars;
  uint64_t* kv_empty = bars + 1;               // products done (and with fp16, the norms taken)
  uint64_t* st_full = bars + 2;                // [kStages] rows and statistics (1 + 32 arrivals)
  uint64_t* st_empty = st_full + C::kStages;   // [kStages] products done and statistics read
  uint64_t* s_full = st_empty + C::kStages;    // [2] S^T of a tile in TMEM
  uint64_t* dp_full = s_full + 2;              // [2] dP^T of a tile in TMEM
  uint64_t* p_full = dp_full + 2;              // [2] P^T written (128 arrivals)
  uint64_t* ds_full = p_full + 2;              // [2] dS^T written (128 arrivals)
  uint64_t* o_done = ds_full + 2;              // [2] products of a tile completed
  uint64_t* acc_full = o_done + 2;             // all products of the unit completed
  uint64_t* acc_empty = acc_full + 1;          // accumulators read (256 arrivals)
  uint64_t* drain_bar = acc_empty + 1;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);
  float* stat_s = reinterpret_cast<float*>(smem + C::kOffStat);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(kv_empty, T::kNarrow ? 1 + 256 : 1);
    for (int s = 0; s < C::kStages; ++s) {
      mbar_init(&st_full[s], 33);
      mbar_init(&st_empty[s], 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(&s_full[w], 1);
      mbar_init(&dp_full[w], 1);
      mbar_init(&p_full[w], 128);
      mbar_init(&ds_full[w], 128);
      mbar_init(&o_done[w], 1);
    }
    mbar_init(acc_full, 1);
    mbar_init(acc_empty, 256);
    mbar_init(drain_bar, 2);
    *abort_flag = 0;
    fence_barrier_init();
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_do);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  // rows that no copy writes (a group size that does not fill the tile) take part
  // in the products over rows with weight 0: they must be finite
  for (int i = threadIdx.x; i < C::kStages * C::kStageBytes / 16; i += kBwdThreads)
    st_shared_v4(smem_u32(smem + C::kOffS + i * 16), 0u, 0u, 0u, 0u);
  fence_proxy_async_smem();
  if (warp == 1) {
    tmem_alloc(tmem_holder, kBwdTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;
  const int off = p.s.n - p.s.m;

  // first token and first head (in the group) of streamed tile r; the second head
  // part of a group of more than 64 ends at the group's last head, its first `dup`
  // rows repeat heads of the first part and carry weight 0
  auto tile_token = [&](const Unit& u, int r) { return u.ta + (r / p.hb) * p.tt; };
  auto tile_head = [&](int r) { return (r % p.hb) == 0 ? 0 : p.s.g - p.gb; };

  if (warp < 4) {
    set_max_regs_dec<kBwdRegsAux>();
    if (warp == 0) {
      // ---------------------------------------------------------- producer
      int gs = 0, uses = 0;
      bool ok = true;
      for (int64_t x = blockIdx.x; ok && x < p.units; x += gridDim.x) {
        const Unit u = make_unit(p, x);
        if (u.r1 <= u.r0) continue;
        ok = mbar_wait_warp(kv_empty, (uses & 1) ^ 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(kv_full, 2 * C::kTileBytes);
#pragma unroll
          for (int half = 0; half < C::kHalves; ++half) {
            tma_load_4d(smem + C::kOffK + half * kBoxBytes, &tm_k, half * 64, u.kt * kRows, u.kvh,
                        u.b, kv_full);
            tma_load_4d(smem + C::kOffV + half * kBoxBytes, &tm_v, half * 64, u.kt * kRows, u.kvh,
                        u.b, kv_full);
          }
        }
        ++uses;
        for (int r = u.r0; r < u.r1; ++r, ++gs) {
          const int s = gs % C::kStages;
          const int t0 = tile_token(u, r), h0 = u.kvh * p.s.g + tile_head(r);
          // the rows' statistics, fetched while the stage is still in use
          float2 st[2];
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int row = lane + 32 * i;
            const int tok = row / p.gb;
            st[i] = make_float2(-INFINITY, 0.f);
            if (tok < p.tt && t0 + tok < p.s.m)
              st[i] = __ldg(p.stat + (static_cast<int64_t>(u.b) * p.s.m + t0 + tok) * p.s.h + h0 +
                            (row - tok * p.gb));
          }
          ok = mbar_wait_warp(&st_empty[s], ((gs / C::kStages) & 1) ^ 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
          if (!ok) break;
          if (lane == 0) {
            uint8_t* dst = smem + C::kOffS + s * C::kStageBytes;
            mbar_arrive_expect_tx(&st_full[s], static_cast<uint32_t>(2 * p.gb * p.tt * D * 2));
#pragma unroll
            for (int half = 0; half < C::kHalves; ++half) {
              tma_load_4d(dst + half * kHalfBox, &tm_q, half * 64, h0, t0, u.b, &st_full[s]);
              tma_load_4d(dst + C::kStageBytes / 2 + half * kHalfBox, &tm_do, half * 64, h0, t0, u.b,
                          &st_full[s]);
            }
          }
          float* ss = stat_s + s * 2 * kStream;
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            ss[lane + 32 * i] = T::kNarrow ? st[i].x + kPUp : st[i].x;
            ss[kStream + lane + 32 * i] = st[i].y;
          }
          mbar_arrive(&st_full[s]);
        }
      }
      // copies in flight land before the CTA's shared memory goes away
      if (uses > 0) mbar_drain(kv_full, (uses - 1) & 1);
      for (int i = (gs > C::kStages ? gs - C::kStages : 0); i < gs; ++i)
        mbar_drain(&st_full[i % C::kStages], (i / C::kStages) & 1);
    } else if (warp == 1 || warp == 2) {
      // ---------------------------------------------------------- MMA issuers
      // warp 1: S^T and dP^T, warp 2: the products over the rows. Each walks and waits as
      // a whole, one elected lane issues. A tile's four products start one by one as their
      // operands are there: P^T is formed while dP^T is computed, dV summed while dS^T is
      // formed
      constexpr uint32_t idesc_s = make_idesc<T>(128, kStream, 0);
      constexpr uint32_t idesc_o = make_idesc<T>(128, D, 1);
      const uint64_t dk0 = make_smem_desc(smem_u32(smem + C::kOffK), 16u, 1024u, kLayoutSW128);
      const uint32_t hi = static_cast<uint32_t>(dk0 >> 32);
      const uint32_t k_lo = static_cast<uint32_t>(dk0);
      const uint32_t v_lo = k_lo + static_cast<uint32_t>((C::kOffV - C::kOffK) >> 4);
      const uint32_t s_lo = k_lo + static_cast<uint32_t>((C::kOffS - C::kOffK) >> 4);
      const uint32_t mn_lo = static_cast<uint32_t>(make_smem_desc(
          smem_u32(smem + C::kOffS), static_cast<uint32_t>(kHalfBox), 1024u, kLayoutSW128));
      int gs = 0, uses = 0;
      bool ok = true;
      auto wait_warp = [&](uint64_t* b, uint32_t parity) -> bool {
        return mbar_wait_warp(b, parity, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
      };
      auto commit = [&](uint64_t* b) {
        if (elect_one()) umma_commit(b);
        __syncwarp();
      };
      // i: number of the streamed tile in the CTA; it uses buffer i & 1
      auto issue_s = [&](int i) -> bool {
        const int w = i & 1, s = i % C::kStages;
        if (!wait_warp(&st_full[s], (i / C::kStages) & 1)) return false;
        if (i >= 2 && !wait_warp(&o_done[w], ((i - 2) >> 1) & 1)) return false;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(w * 128);
        const uint32_t qb = s_lo + static_cast<uint32_t>(s * (C::kStageBytes >> 4));
        const uint32_t ob = qb + static_cast<uint32_t>(C::kStageBytes >> 5);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t ao = static_cast<uint32_t>(((k >> 2) * kBoxBytes + (k & 3) * 32) >> 4);
            const uint32_t bo = static_cast<uint32_t>(((k >> 2) * kHalfBox + (k & 3) * 32) >> 4);
            umma_bf16(d, desc_from_words(k_lo + ao, hi), desc_from_words(qb + bo, hi), idesc_s,
                      k > 0 ? 1u : 0u);
          }
          umma_commit(&s_full[w]);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t ao = static_cast<uint32_t>(((k >> 2) * kBoxBytes + (k & 3) * 32) >> 4);
            const uint32_t bo = static_cast<uint32_t>(((k >> 2) * kHalfBox + (k & 3) * 32) >> 4);
            umma_bf16(d + 64u, desc_from_words(v_lo + ao, hi), desc_from_words(ob + bo, hi), idesc_s,
                      k > 0 ? 1u : 0u);
          }
          umma_commit(&dp_full[w]);
        }
        __syncwarp();
        return true;
      };
      auto issue_o = [&](int i, bool fresh) -> bool {
        const int w = i & 1, s = i % C::kStages;
        const uint32_t d = tmem + static_cast<uint32_t>(w * 128);
        const uint32_t qb = mn_lo + static_cast<uint32_t>(s * (C::kStageBytes >> 4));
        const uint32_t ob = qb + static_cast<uint32_t>(C::kStageBytes >> 5);
        const uint32_t more = fresh ? 0u : 1u;
        if (!wait_warp(&p_full[w], (i >> 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int st = 0; st < kStream / 16; ++st)
            umma_bf16_tmem_a(tmem + 384u, d + static_cast<uint32_t>(st * 8),
                             desc_from_words(ob + static_cast<uint32_t>(st * 128), hi), idesc_o,
                             st > 0 ? 1u : more);
        }
        __syncwarp();
        if (!wait_warp(&ds_full[w], (i >> 1) & 1)) return false;
        tc_fence_after();
        if (elect_one()) {
#pragma unroll
          for (int st = 0; st < kStream / 16; ++st)
            umma_bf16_tmem_a(tmem + 256u, d + 64u + static_cast<uint32_t>(st * 8),
                             desc_from_words(qb + static_cast<uint32_t>(st * 128), hi), idesc_o,
                             st > 0 ? 1u : more);
          umma_commit(&o_done[w]);
          umma_commit(&st_empty[s]);
        }
        __syncwarp();
        return true;
      };
      for (int64_t x = blockIdx.x; ok && x < p.units; x += gridDim.x) {
        const Unit u = make_unit(p, x);
        const int nt = u.r1 - u.r0;
        if (nt <= 0) continue;
        if (warp == 1) {
          ok = wait_warp(kv_full, uses & 1);
          for (int i = 0; i < nt && ok; ++i) ok = issue_s(gs + i);
          if (ok) commit(kv_empty);  // the key tile is no longer read
        } else {
          ok = uses == 0 || wait_warp(acc_empty, (uses - 1) & 1);
          for (int i = 0; i < nt && ok; ++i) ok = issue_o(gs + i, i == 0);
          if (ok) commit(acc_full);
        }
        gs += nt;
        ++uses;
      }
      commit(drain_bar);
      mbar_drain(drain_bar, 0);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ P^T and dS^T
    set_max_regs_inc<kBwdRegsSoftmax>();
    const int w = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;  // key of the tile
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t sp = tmem + lane_off + static_cast<uint32_t>(w * 128);
    const uint32_t stage = smem_u32(smem + C::kOffStage) + static_cast<uint32_t>((warp - 4) * 2048);
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    int gs = 0, gw = 0, uses = 0;
    bool ok = true;
    for (int64_t x = blockIdx.x; x < p.units; x += gridDim.x) {
      const Unit u = make_unit(p, x);
      const int nt = max(u.r1 - u.r0, 0);
      const int key = u.kt * kRows + row;
      // positions [key, end) see this key
      const int64_t far = static_cast<int64_t>(key) + p.s.window;
      int end = p.s.n;
      if (key >= p.s.n_first && far < end) end = static_cast<int>(far);
      if (key >= u.kv_len) end = key;
      float up = 1.f;  // the key's scale of dS (fp16)
      if constexpr (T::kNarrow) {
        if (nt > 0) {
          ok = mbar_wait_warp(kv_full, uses & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
          if (!ok) break;
          float sq = 0.f;
#pragma unroll
          for (int half = 0; half < C::kHalves; ++half) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              // 16-byte pieces in an order that keeps the lanes on different banks
              const float4 x = ld_shared_f4(smem_u32(smem + C::kOffV + half * kBoxBytes + row * 128) +
                                            ((static_cast<uint32_t>(j) ^ static_cast<uint32_t>(row & 7)) << 4));
              const uint32_t vw[4] = {__float_as_uint(x.x), __float_as_uint(x.y),
                                      __float_as_uint(x.z), __float_as_uint(x.w)};
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                sq = fmaf(T::lo(vw[i]), T::lo(vw[i]), sq);
                sq = fmaf(T::hi(vw[i]), T::hi(vw[i]), sq);
              }
            }
          }
          mbar_arrive(kv_empty);
          const float size = sqrtf(sq);
          Peak* peak = peaks + (static_cast<int64_t>(u.b) * p.s.hk + u.kvh);
          const uint32_t most =
              __reduce_max_sync(0xFFFFFFFFu, key < u.kv_len ? __float_as_uint(size) : 0u);
          if (w == 0 && lane == 0) raise(&peak->v, most);
          up = power_below(__uint_as_float(peak->dout) * size + __uint_as_float(peak->d));
        }
      }
      auto scaled = [&](uint64_t g2) -> uint64_t {
        if constexpr (T::kNarrow) return f2_mul(g2, f2_pack(up, up));
        return g2;
      };
      for (int i = 0; i < nt; ++i) {
        if (((gs + i) & 1) != w) continue;
        const int s = (gs + i) % C::kStages;
        ok = mbar_wait_warp(&s_full[w], gw & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        // the statistics were written with ordinary stores: their barrier is waited
        // for here too (it completed before this tile's products were issued)
        ok = mbar_wait_warp(&st_full[s], ((gs + i) / C::kStages) & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        tc_fence_after();
        // the columns (rows of the streamed tile) that see this key: one range,
        // since rows are token-major
        const int r = u.r0 + i;
        const int p0 = tile_token(u, r) + off;
        const int tok_a = min(max(key - p0, 0), p.tt);
        const int tok_b = min(max(end - p0, 0), p.tt);
        const int dup = (r % p.hb) == 0 ? 0 : p.hb * p.gb - p.s.g;
        const int ca = max(tok_a * p.gb, dup), cb = tok_b * p.gb;
        const uint32_t seen[2] = {bits_between(ca, cb), bits_between(ca - 32, cb - 32)};
        const bool all = __all_sync(0xFFFFFFFFu, (seen[0] & seen[1]) == 0xFFFFFFFFu);
        // two 16-bit weights of a word that their rows do not see become 0
        auto keep = [&](uint32_t word, uint32_t bits, int k) -> uint32_t {
          const uint32_t two = (bits >> (2 * k)) & 3u;
          return word & ((two & 1u ? 0x0000FFFFu : 0u) | (two & 2u ? 0xFFFF0000u : 0u));
        };
        const uint32_t stat4 = smem_u32(smem + C::kOffStat) + static_cast<uint32_t>(s * 2 * kStream * 4);
        uint32_t sv[2][32];  // S^T, then P^T in fp32
        tmem_ld_32x32b_x32_nowait(sp, sv[0]);
        tmem_ld_32x32b_x32_nowait(sp + 32u, sv[1]);
        tmem_wait_ld_dep(sv[0]);
        tmem_wait_ld_dep(sv[1]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 nl = ld_shared_f4(stat4 + static_cast<uint32_t>((q * 8 + k) * 16));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int c = 4 * k + 2 * e;
              float z0, z1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(sv[q][c]), __uint_as_float(sv[q][c + 1])),
                               scale2, e ? f2_pack(nl.z, nl.w) : f2_pack(nl.x, nl.y)),
                        z0, z1);
              z0 = ex2_approx(z0);
              z1 = ex2_approx(z1);
              sv[q][c] = __float_as_uint(z0);
              sv[q][c + 1] = __float_as_uint(z1);
              pk[c >> 1] = T::pack(z0, z1);
            }
          }
          if (!all) {
#pragma unroll
            for (int k = 0; k < 16; ++k) pk[k] = keep(pk[k], seen[q], k);
          }
          tmem_st_x16_nowait(sp + static_cast<uint32_t>(q * 16), pk);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[w]);
        ok = mbar_wait_warp(&dp_full[w], gw & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        tc_fence_after();
        uint32_t dv[2][32];
        tmem_ld_32x32b_x32_nowait(sp + 64u, dv[0]);
        tmem_ld_32x32b_x32_nowait(sp + 96u, dv[1]);
        tmem_wait_ld_dep(dv[0]);
        tmem_wait_ld_dep(dv[1]);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          uint32_t dk[16];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const float4 nd = ld_shared_f4(stat4 + static_cast<uint32_t>((16 + q * 8 + k) * 16));
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int c = 4 * k + 2 * e;
              float g0, g1;
              f2_unpack(f2_mul(f2_pack(__uint_as_float(sv[q][c]), __uint_as_float(sv[q][c + 1])),
                               scaled(f2_add(f2_pack(__uint_as_float(dv[q][c]),
                                                     __uint_as_float(dv[q][c + 1])),
                                             e ? f2_pack(nd.z, nd.w) : f2_pack(nd.x, nd.y)))),
                        g0, g1);
              dk[c >> 1] = T::pack(g0, g1);
            }
          }
          if (!all) {
#pragma unroll
            for (int k = 0; k < 16; ++k) dk[k] = keep(dk[k], seen[q], k);
          }
          tmem_st_x16_nowait(sp + 64u + static_cast<uint32_t>(q * 16), dk);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ds_full[w]);
        ++gw;
      }
      if (!ok) break;
      gs += nt;
      // ---- epilogue: warpgroup 0 the first half of the columns, 1 the second
      if (nt > 0) {
        ok = mbar_wait_warp(acc_full, uses & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        tc_fence_after();
        ++uses;
      }
      const bool live = nt > 0 && key < u.kv_len;
      const int c0 = w * (D / 2);
#pragma unroll 1
      for (int q = 0; q < D / 64; ++q) {
        uint32_t a[32], b[32];
        if (nt > 0) {
          tmem_ld_32x32b_x32(tmem + lane_off + 256u + static_cast<uint32_t>(c0 + q * 32), a);
          tmem_ld_32x32b_x32(tmem + lane_off + 384u + static_cast<uint32_t>(c0 + q * 32), b);
        }
        const float down = T::kNarrow ? scale_down(p.scale, up) : p.scale;
        float fk[32], fv[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          fk[k] = live ? __uint_as_float(a[k]) * down : 0.f;
          fv[k] = live ? __uint_as_float(b[k]) * (T::kNarrow ? kPDown : 1.f) : 0.f;
          if (p.dv == nullptr) fk[k] += fv[k];
        }
        if (u.parts > 1) {
          const int kinds = p.dv == nullptr ? 1 : 2;
          float* dst = p.parts + ((x * kinds) * kRows + row) * D + c0 + q * 32;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            reinterpret_cast<float4*>(dst)[k] =
                make_float4(fk[4 * k], fk[4 * k + 1], fk[4 * k + 2], fk[4 * k + 3]);
            if (kinds == 2)
              reinterpret_cast<float4*>(dst + kRows * D)[k] =
                  make_float4(fv[4 * k], fv[4 * k + 1], fv[4 * k + 2], fv[4 * k + 3]);
          }
        } else {
          const int64_t at =
              ((static_cast<int64_t>(u.b) * p.s.n + key) * p.s.hk + u.kvh) * D + c0 + q * 32;
          uint32_t y[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) y[k] = T::pack(fk[2 * k], fk[2 * k + 1]);
          store_rows(stage, y, key < p.s.n ? p.dk + at : nullptr, lane);
          if (p.dv != nullptr) {
#pragma unroll
            for (int k = 0; k < 16; ++k) y[k] = T::pack(fv[2 * k], fv[2 * k + 1]);
            store_rows(stage, y, key < p.s.n ? p.dv + at : nullptr, lane);
          }
        }
      }
      if (nt > 0) {
        tc_fence_before();
        mbar_arrive(acc_empty);
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kBwdTmemCols);
  }
}

// Sums the parts of the key tiles with several units, in a fixed order: eight lanes take
// every eighth part of four columns of a key, then their sums are added in lane order.
// (One thread for all parts took 25 us where the first tokens' tile had 75 of them.)
template <typename T, int D>
__global__ void __launch_bounds__(256) window_join_kernel(const DkvParams p, int64_t batch) {
  const bool two = p.split > 1;  // all key tiles have parts, else only the first ones
  const int tiles = two ? p.key_tiles : p.first_tiles;
  const int kinds = p.dv == nullptr ? 1 : 2;
  // a warp: 8 parts x 16 columns of one key
  const int lane = threadIdx.x & 31;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int col = static_cast<int>(i % (D / 16)) * 16 + (lane & 3) * 4;
  int64_t x = i / (D / 16);
  const int row = static_cast<int>(x % kRows);
  x /= kRows;
  const int kind = static_cast<int>(x % kinds);
  x /= kinds;
  const int kt = static_cast<int>(x % tiles);
  const int64_t bh = x / tiles;
  const int key = kt * kRows + row;
  if (bh >= batch * p.s.hk || key >= p.s.n) return;
  const bool first = kt < p.first_tiles;
  const int parts = first ? p.split_first : p.split;
  if (parts <= 1) return;
  const int64_t unit = bh * p.units_per_head +
                       (first ? static_cast<int64_t>(kt) * p.split_first
                              : static_cast<int64_t>(p.first_tiles) * p.split_first +
                                    static_cast<int64_t>(kt - p.first_tiles) * p.split);
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = lane >> 2; s < parts; s += 8) {
    const float4 v = *reinterpret_cast<const float4*>(
        p.parts + (((unit + s) * kinds + kind) * kRows + row) * D + col);
    sum.x += v.x;
    sum.y += v.y;
    sum.z += v.z;
    sum.w += v.w;
  }
#pragma unroll
  for (int o = 16; o >= 4; o >>= 1) {
    sum.x += __shfl_down_sync(0xFFFFFFFFu, sum.x, o);
    sum.y += __shfl_down_sync(0xFFFFFFFFu, sum.y, o);
    sum.z += __shfl_down_sync(0xFFFFFFFFu, sum.z, o);
    sum.w += __shfl_down_sync(0xFFFFFFFFu, sum.w, o);
  }
  if (lane >= 4) return;
  const int64_t b = bh / p.s.hk;
  uint16_t* out = kind ? p.dv : p.dk;
  *reinterpret_cast<uint2*>(out + ((b * p.s.n + key) * p.s.hk + (bh - b * p.s.hk)) * D + col) =
      make_uint2(T::pack(sum.x, sum.y), T::pack(sum.z, sum.w));
}

// ------------------------------------------------------------------ dq
template <int D>
struct DqCfg {
  static constexpr int kHalves = D / 64;
  static constexpr int kTileBytes = kRows * D * 2;
  static constexpr int kSlotBytes = kCB * kBlk * D * 2;
  static constexpr int kSlots = D == 128 ? 5 : 8;
  static constexpr int kOffQ = 0;                      // [2 tiles] q, dout
  static constexpr int kOffKV = 4 * kTileBytes;
  static constexpr int kOffStage = kOffKV + kSlots * kSlotBytes;  // [8 warps] 2 KB, dq rows
  static constexpr int kOffBar = kOffStage + 8 * 2048;
  static constexpr int kNumBars = 2 + 2 + 2 * kSlots + 2 + 2 + 2 + 2 + 2 + 1;
  static constexpr int kOffMisc = kOffBar + kNumBars * 8;
  static constexpr int kSmemBytes = kOffMisc + 16 + 1024;
};

struct DqParams {
  Shape s;
  TileGrid grid;
  float scale, scale_log2;
  const float2* stat;   // [batch, m, h]
  const float* sink;    // [h] or null
  const Peak* peaks;    // [batch, hk], fp16 only
  uint16_t* dq;         // [batch, m, h, D]
  // [batch, m, h]: with fp16 a row's |dout| when the kernel starts; then, with sink,
  // e^(sink - lse) sum_j P_j dP_j
  float* sink_rows;
  int shared;
  unsigned int* err;
};

template <typename T, int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    window_dq_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_do,
                     const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                     const DqParams p) {
  using C = DqCfg<D>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kOffBar);
  uint64_t* q_full = bars;                  // [2] TMA -> MMA
  uint64_t* q_empty = q_full + 2;           // [2] last products of the tile's rows done -> TMA
  uint64_t* kv_full = q_empty + 2;          // [kSlots]
  uint64_t* kv_empty = kv_full + C::kSlots; // [kSlots]
  uint64_t* s_full = kv_empty + C::kSlots;  // [2] S of a chunk in TMEM
  uint64_t* dp_full = s_full + 2;           // [2] dP of a chunk in TMEM
  uint64_t* p_full = dp_full + 2;           // [2] dS written (128 arrivals)
  uint64_t* o_done = p_full + 2;            // [2] dq product of a chunk completed
  uint64_t* o_empty = o_done + 2;           // [2] dq read by the epilogue (128 arrivals)
  uint64_t* drain_bar = o_empty + 2;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + C::kOffMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + C::kOffMisc + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int w = 0; w < 2; ++w) {
      mbar_init(&q_full[w], 1);
      mbar_init(&q_empty[w], 1);
      mbar_init(&s_full[w], 1);
      mbar_init(&dp_full[w], 1);
      mbar_init(&p_full[w], 128);
      mbar_init(&o_done[w], 1);
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
    tma_prefetch_desc(&tm_do);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, kBwdTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_holder;

  if (warp < 4) {
    set_max_regs_dec<kBwdRegsAux>();
    if (warp == 0 && lane == 0) {
      // ---------------------------------------------------------- producer
      Ring<C::kSlots> at;
      int loads = 0;
      int uses0 = 0, uses1 = 0;
      bool ok = true;
      auto load_slot = [&](const Item<kCB>& it, const CUtensorMap* tm, int c) -> bool {
        if (!mbar_wait(&kv_empty[at.slot], at.parity ^ 1u, abort_flag, p.err, DSA_DEVERR_WIN_WAIT))
          return false;
        const int nb = it.blocks(c);
        uint8_t* dst = smem + C::kOffKV + at.slot * C::kSlotBytes;
        mbar_arrive_expect_tx(&kv_full[at.slot], static_cast<uint32_t>(nb * kBlk * D * 2));
        for (int i = 0; i < nb; ++i) {
          const int key = it.r.key(c * kCB + i);
#pragma unroll
          for (int half = 0; half < C::kHalves; ++half)
            tma_load_4d(dst + half * kHalfBox + i * kBlk * 128, tm, half * 64, key, it.kvh, it.b,
                        &kv_full[at.slot]);
        }
        at.next();
        ++loads;
        return true;
      };
      auto load_rows = [&](const Item<kCB>& it, int w, int& uses) -> bool {
        if (it.last(w) < 0) return true;
        if (!mbar_wait(&q_empty[w], (uses & 1) ^ 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT))
          return false;
        uint8_t* qs = smem + C::kOffQ + 2 * w * C::kTileBytes;
        mbar_arrive_expect_tx(&q_full[w], static_cast<uint32_t>(2 * p.grid.tt * p.s.g * D * 2));
#pragma unroll
        for (int half = 0; half < C::kHalves; ++half) {
          tma_load_4d(qs + half * kBoxBytes, &tm_q, half * 64, it.kvh * p.s.g, it.t0(w), it.b,
                      &q_full[w]);
          tma_load_4d(qs + C::kTileBytes + half * kBoxBytes, &tm_do, half * 64, it.kvh * p.s.g,
                      it.t0(w), it.b, &q_full[w]);
        }
        ++uses;
        return true;
      };
      for (ItemWalk wk(p.s, p.grid); ok && wk.item < p.grid.items; wk.next(p.s, p.grid)) {
        const Item<kCB> it = make_item<kCB>(p.s, p.grid, wk);
        ok = load_rows(it, 0, uses0) && load_rows(it, 1, uses1);
        for (int c = 0; c < it.chunks && ok; ++c) {
          ok = load_slot(it, &tm_k, c);
          if (ok && !p.shared) ok = load_slot(it, &tm_v, c);
        }
      }
      for (int i = max(loads - C::kSlots, 0); i < loads; ++i)
        mbar_drain(&kv_full[i % C::kSlots], (i / C::kSlots) & 1);
      if (uses0 > 0) mbar_drain(&q_full[0], (uses0 - 1) & 1);
      if (uses1 > 0) mbar_drain(&q_full[1], (uses1 - 1) & 1);
    } else if (warp == 1 || warp == 2) {
      // ---------------------------------------------------------- MMA issuers, one per tile
      // the whole warp walks and waits; one elected lane issues
      const int w = warp - 1;
      constexpr uint32_t idesc_o = make_idesc<T>(128, D, 1);
      const uint64_t dq0 = make_smem_desc(smem_u32(smem + C::kOffQ), 16u, 1024u, kLayoutSW128);
      const uint32_t hi = static_cast<uint32_t>(dq0 >> 32);
      const uint32_t q_lo = static_cast<uint32_t>(dq0);
      const uint32_t k_lo = q_lo + static_cast<uint32_t>((C::kOffKV - C::kOffQ) >> 4);
      const uint32_t mn_lo = static_cast<uint32_t>(make_smem_desc(
          smem_u32(smem + C::kOffKV), static_cast<uint32_t>(kHalfBox), 1024u, kLayoutSW128));
      Ring<C::kSlots> at;  // the next slot in the order of the loads
      int gp = 0, uses = 0;
      bool ok = true;
      auto wait_warp = [&](uint64_t* b, uint32_t parity) -> bool {
        return mbar_wait_warp(b, parity, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
      };
      auto commit = [&](uint64_t* b) {
        if (elect_one()) umma_commit(b);
        __syncwarp();
      };
      // waits for the next slot and returns its number
      auto take = [&]() -> int {
        const int s = at.slot;
        ok = ok && wait_warp(&kv_full[s], at.parity);
        at.next();
        return s;
      };
      auto issue_s = [&](const Item<kCB>& it, int c, int ks, int vs) {
        if (!ok || !it.active(w, c)) return;
        if (gp >= 1) ok = wait_warp(&o_done[w], (gp - 1) & 1);
        if (!ok) return;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(w * 256);
        const uint32_t qa = q_lo + static_cast<uint32_t>(2 * w * (C::kTileBytes >> 4));
        const uint32_t oa = qa + static_cast<uint32_t>(C::kTileBytes >> 4);
        const uint32_t kb = k_lo + static_cast<uint32_t>(ks * (C::kSlotBytes >> 4));
        const uint32_t vb = k_lo + static_cast<uint32_t>(vs * (C::kSlotBytes >> 4));
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
          umma_commit(&s_full[w]);
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const uint32_t ao = static_cast<uint32_t>(((k >> 2) * kBoxBytes + (k & 3) * 32) >> 4);
            const uint32_t bo = static_cast<uint32_t>(((k >> 2) * kHalfBox + (k & 3) * 32) >> 4);
            umma_bf16(d + 64u, desc_from_words(oa + ao, hi), desc_from_words(vb + bo, hi), idesc_s,
                      k > 0 ? 1u : 0u);
          }
          umma_commit(&dp_full[w]);
          if (end) umma_commit(&q_empty[w]);
        }
        __syncwarp();
      };
      auto issue_o = [&](const Item<kCB>& it, int c, int slot) {
        if (!ok || !it.active(w, c)) return;
        const bool fresh = c == it.first(w);
        ok = wait_warp(&p_full[w], gp & 1);
        if (ok && fresh && uses > 1) ok = wait_warp(&o_empty[w], (uses - 2) & 1);
        if (!ok) return;
        tc_fence_after();
        const uint32_t d = tmem + static_cast<uint32_t>(w * 256);
        const uint32_t kb = mn_lo + static_cast<uint32_t>(slot * (C::kSlotBytes >> 4));
        const int nb = it.blocks(c);
        const uint32_t more = fresh ? 0u : 1u;
        if (elect_one()) {
#pragma unroll
          for (int st = 0; st < kCB * 2; ++st)
            if (st < nb * 2)
              umma_bf16_tmem_a(d + 128u, d + static_cast<uint32_t>(st * 8),
                               desc_from_words(kb + static_cast<uint32_t>(st * 128), hi), idesc_o,
                               st > 0 ? 1u : more);
          umma_commit(&o_done[w]);
        }
        __syncwarp();
        ++gp;
      };
      // K rows at or past kv_len may hold anything, and 0 x NaN is NaN: cleared before
      // the product that sums over them (by both issuers, to the same zeros)
      auto clear_tail = [&](const Item<kCB>& it, int c, int slot, int nb) {
        uint8_t* base = smem + C::kOffKV + slot * C::kSlotBytes;
        bool wrote = false;
        for (int i = 0; i < nb; ++i) {
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
        if (it.last(w) >= 0) ok = wait_warp(&q_full[w], uses++ & 1);
        int ks = take();
        int vs = p.shared ? ks : take();
        issue_s(it, 0, ks, vs);
        if (!p.shared) commit(&kv_empty[vs]);
        for (int c = 0; c < n && ok; ++c) {
          const int now = ks;
          if (p.s.kv_lens != nullptr) clear_tail(it, c, now, it.blocks(c));
          if (c + 1 < n) {
            ks = take();
            vs = p.shared ? ks : take();
          }
          issue_o(it, c, now);
          if (c + 1 < n) {
            issue_s(it, c + 1, ks, vs);
            if (!p.shared) commit(&kv_empty[vs]);
          }
          commit(&kv_empty[now]);
        }
      }
      commit(drain_bar);
      mbar_drain(drain_bar, 0);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ dS
    set_max_regs_inc<kBwdRegsSoftmax>();
    const int w = (warp - 4) >> 2;
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int tok = row / p.s.g;
    const int head = row - tok * p.s.g;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t sp = tmem + lane_off + static_cast<uint32_t>(w * 256);
    const uint32_t od = sp + 128u;
    const uint32_t stage = smem_u32(smem + C::kOffStage) + static_cast<uint32_t>((warp - 4) * 2048);
    const uint64_t scale2 = f2_pack(p.scale_log2, p.scale_log2);
    int gc = 0;
    bool ok = true;
    for (ItemWalk wk(p.s, p.grid); wk.item < p.grid.items; wk.next(p.s, p.grid)) {
      const Item<kCB> it = make_item<kCB>(p.s, p.grid, wk);
      const int first = it.first(w), last = it.last(w);
      const int t = it.t0(w) + tok;
      const bool valid = tok < p.grid.tt && t < it.t1(w);
      const int pos = min(t, it.t1(w) - 1) + p.s.n - p.s.m;
      const int64_t orow = (static_cast<int64_t>(it.b) * p.s.m + t) * p.s.h + it.kvh * p.s.g + head;
      const float2 st = valid ? __ldg(p.stat + orow) : make_float2(-INFINITY, 0.f);
      const float nl = T::kNarrow ? st.x + kPUp : st.x;
      const uint64_t l2 = f2_pack(nl, nl), d2 = f2_pack(st.y, st.y);
      float up = 1.f;  // the row's scale of dS (fp16)
      if constexpr (T::kNarrow) {
        const Peak* peak = p.peaks + (static_cast<int64_t>(it.b) * p.s.hk + it.kvh);
        if (valid) up = power_below(p.sink_rows[orow] * __uint_as_float(__ldg(&peak->v)) + fabsf(st.y));
      }
      uint64_t psum[2] = {0ull, 0ull};  // sum_j P_j dP_j
      for (int c = first; c <= last; ++c) {
        if (!it.active(w, c)) continue;
        const int nb = it.blocks(c);
        ok = mbar_wait_warp(&s_full[w], gc & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        tc_fence_after();
        const bool full = chunk_full<kCB>(p.s, it, it.t0(w), it.t1(w), c);
        uint32_t seen[kCB];
        uint32_t sv[kCB][32];  // S, then P in fp32, formed while dP is computed
#pragma unroll
        for (int i = 0; i < kCB; ++i)
          if (i < nb) tmem_ld_32x32b_x32_nowait(sp + static_cast<uint32_t>(i * kBlk), sv[i]);
#pragma unroll
        for (int i = 0; i < kCB; ++i) {
          if (i < nb) {
            tmem_wait_ld_dep(sv[i]);
            if (!full) {
              seen[i] = seen_bits(p.s, it.r, c * kCB + i, pos, it.kv_len);
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!((seen[i] >> k) & 1u)) sv[i][k] = 0xFF800000u;  // P = 0
            }
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float z0, z1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(sv[i][2 * k]), __uint_as_float(sv[i][2 * k + 1])),
                               scale2, l2),
                        z0, z1);
              sv[i][2 * k] = __float_as_uint(ex2_approx(z0));
              sv[i][2 * k + 1] = __float_as_uint(ex2_approx(z1));
            }
          }
        }
        ok = mbar_wait_warp(&dp_full[w], gc & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int i = 0; i < kCB; ++i) {
          if (i < nb) {
            uint32_t dv[32];
            tmem_ld_32x32b_x32(sp + 64u + static_cast<uint32_t>(i * kBlk), dv);
            if (!full) {
#pragma unroll
              for (int k = 0; k < 32; ++k)
                if (!((seen[i] >> k) & 1u)) dv[k] = 0u;  // of a key that may hold anything
            }
            uint32_t pk[16];
#pragma unroll
            for (int k = 0; k < 16; ++k) {
              float g0, g1;
              const uint64_t e2 = f2_pack(__uint_as_float(sv[i][2 * k]), __uint_as_float(sv[i][2 * k + 1]));
              const uint64_t g2 = f2_pack(__uint_as_float(dv[2 * k]), __uint_as_float(dv[2 * k + 1]));
              psum[k & 1] = f2_fma(e2, g2, psum[k & 1]);
              uint64_t ds2 = f2_add(g2, d2);
              if constexpr (T::kNarrow) ds2 = f2_mul(ds2, f2_pack(up, up));
              f2_unpack(f2_mul(e2, ds2), g0, g1);
              pk[k] = T::pack(g0, g1);
            }
            tmem_st_x16_nowait(sp + static_cast<uint32_t>(i * 16), pk);
          }
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[w]);
        ++gc;
      }
      if (!ok) break;
      if (last >= 0) {
        ok = mbar_wait_warp(&o_done[w], (gc - 1) & 1, abort_flag, p.err, DSA_DEVERR_WIN_WAIT);
        if (!ok) break;
        tc_fence_after();
      }
      const float down = T::kNarrow ? scale_down(p.scale, up) : p.scale;
#pragma unroll 1
      for (int q = 0; q < D / 32; ++q) {
        uint32_t ov[32], x[16];
        if (last >= 0) tmem_ld_32x32b_x32(od + static_cast<uint32_t>(q * 32), ov);
#pragma unroll
        for (int k = 0; k < 16; ++k)
          x[k] = last < 0 ? 0u
                          : T::pack(__uint_as_float(ov[2 * k]) * down,
                                    __uint_as_float(ov[2 * k + 1]) * down);
        if (last >= 0 && q == D / 32 - 1) {
          tc_fence_before();
          mbar_arrive(&o_empty[w]);
        }
        store_rows(stage, x, valid ? p.dq + orow * D + q * 32 : nullptr, lane);
      }
      if (valid && p.sink != nullptr) {
        float a0, a1, b0, b1;
        f2_unpack(psum[0], a0, a1);
        f2_unpack(psum[1], b0, b1);
        // the sink's own weight e^(sink - lse): 0 where the sink is -inf
        const float weight = ex2_approx(fmaf(__ldg(p.sink + it.kvh * p.s.g + head), kLog2e, st.x));
        const float sum = ((a0 + a1) + (b0 + b1)) * (T::kNarrow ? kPDown : 1.f);
        p.sink_rows[orow] = st.x == -INFINITY ? 0.f : weight * sum;
      }
    }
  }

  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, kBwdTmemCols);
  }
}

// ------------------------------------------------------------------ dsink
// Column sums of sink_rows [rows, h] in two fixed-order steps: blocks of
// kSinkRows rows, then the blocks. A block holds 32 heads x 8 row lanes.
constexpr int kSinkRows = 256;

__global__ void __launch_bounds__(256) window_dsink_kernel(const float* in, float* out, int64_t rows,
                                                           int h, float sign) {
  __shared__ float part[8][33];
  const int head = blockIdx.y * 32 + (threadIdx.x & 31);
  const int y = threadIdx.x >> 5;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * kSinkRows;
  const int64_t r1 = r0 + kSinkRows < rows ? r0 + kSinkRows : rows;
  float sum = 0.f;
  if (head < h) {
#pragma unroll 8
    for (int64_t r = r0 + y; r < r1; r += 8) sum += in[r * h + head];
  }
  part[y][threadIdx.x & 31] = sum;
  __syncthreads();
  if (y == 0 && head < h) {
#pragma unroll
    for (int i = 1; i < 8; ++i) sum += part[i][threadIdx.x];
    out[static_cast<int64_t>(blockIdx.x) * h + head] = sum * sign;
  }
}

// ------------------------------------------------------------------ host
struct BwdPlan {
  int gb, hb, tt;
  int key_tiles, first_tiles, split_first, split, units_per_head;
  int64_t units;
  size_t off_stat, off_rows, off_sum, off_peaks, off_parts, bytes;
};

inline int64_t div_up(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Key tiles are split over their rows so that no unit is much longer than an equal
// share of a third of an SM (kUnits = 3 x 148; the number is fixed, so that a sum's parts are
// the same on every device), and none is shorter than 16
// streamed tiles, below which the fp32 parts cost more than the balance gives.
inline BwdPlan plan_bwd(const Shape& s, int64_t batch, int d, bool shared) {
  constexpr int64_t kUnits = 3 * 148;
  BwdPlan b;
  b.hb = s.g <= kStream ? 1 : 2;
  b.gb = b.hb == 1 ? s.g : (s.g + 1) / 2;
  b.tt = b.hb == 1 ? kStream / s.g : 1;
  b.key_tiles = static_cast<int>(div_up(s.n, kRows));
  b.first_tiles = static_cast<int>(div_up(s.n_first, kRows));
  int64_t total = 0, most_first = 0, most = 0;
  for (int kt = 0; kt < b.key_tiles; ++kt) {
    int ta, tb;
    dkv_tokens(s, kt, &ta, &tb);
    const int64_t tiles = div_up(tb - ta, b.tt) * b.hb;
    total += tiles;
    int64_t& top = kt < b.first_tiles ? most_first : most;
    if (tiles > top) top = tiles;
  }
  int64_t share = div_up(total * batch * s.hk, kUnits);
  if (share < 16) share = 16;
  b.split_first = static_cast<int>(most_first > 0 ? div_up(most_first, share) : 1);
  b.split = static_cast<int>(most > 0 ? div_up(most, share) : 1);
  b.units_per_head = b.first_tiles * b.split_first + (b.key_tiles - b.first_tiles) * b.split;
  b.units = batch * s.hk * b.units_per_head;
  const auto pad = [](size_t x) { return (x + 255) & ~static_cast<size_t>(255); };
  const size_t rows = static_cast<size_t>(batch) * s.m * s.h;
  b.off_stat = 0;
  b.off_rows = pad(rows * sizeof(float2));
  b.off_sum = b.off_rows + pad(rows * sizeof(float));
  b.off_peaks = b.off_sum + pad(static_cast<size_t>(div_up(batch * s.m, kSinkRows)) * s.h * sizeof(float));
  b.off_parts = b.off_peaks + pad(static_cast<size_t>(batch) * s.hk * sizeof(Peak));
  const bool parts = b.split > 1 || (b.first_tiles > 0 && b.split_first > 1);
  b.bytes = b.off_parts +
            (parts ? static_cast<size_t>(b.units) * (shared ? 1 : 2) * kRows * d * sizeof(float) : 0);
  return b;
}

template <typename T, int D>
int launch_bwd(const Tensors& x, const Shape& s, int64_t batch, float scale, const float* sink,
               const void* out, const void* dout, const Strides& dos, const float* lse, void* dq,
               void* dk, void* dv, float* dsink, uint8_t* ws, const BwdPlan& b, cudaStream_t stream) {
  DeviceInfo di;
  int st = current_device_info(&di);
  if (st != DSA_OK) return st;
  if (di.max_smem_optin < DkvCfg<D>::kSmemBytes || di.max_smem_optin < DqCfg<D>::kSmemBytes)
    return DSA_ERR_UNSUPPORTED;
  unsigned int* err = nullptr;
  st = device_error_word(&err);
  if (st != DSA_OK) return st;
  const int64_t rows = batch * s.m * s.h;
  float2* stat = reinterpret_cast<float2*>(ws + b.off_stat);
  float* sink_rows = reinterpret_cast<float*>(ws + b.off_rows);
  float* sink_sum = reinterpret_cast<float*>(ws + b.off_sum);
  Peak* peaks = reinterpret_cast<Peak*>(ws + b.off_peaks);
  if (rows > 0) {
    if (T::kNarrow) {
      st = cuda_status(cudaMemsetAsync(peaks, 0, static_cast<size_t>(batch) * s.hk * sizeof(Peak), stream));
      if (st != DSA_OK) return st;
    }
    const bool flat = dos.h == D && dos.t == static_cast<int64_t>(s.h) * D &&
                      (batch == 1 || dos.b == dos.t * s.m);
    auto kernel = flat ? window_stat_kernel<T, D, true> : window_stat_kernel<T, D, false>;
    kernel<<<static_cast<unsigned>(div_up(rows, 256 / (D / 8) * kStatRows)), 256, 0, stream>>>(
        static_cast<const uint16_t*>(out), static_cast<const uint16_t*>(dout), dos, lse, stat,
        sink_rows, peaks, rows, s.m, s.h, s.g);
    st = cuda_status(cudaGetLastError());
    if (st != DSA_OK) return st;
  }
  CUtensorMap tm_q, tm_do, tm_k, tm_v;
  if (s.n > 0) {
    st = map_rows_by_head(&tm_q, T::kFmt, x.q, x.qs, batch, s.m, s.h, D, b.gb, b.tt);
    if (st == DSA_OK)
      st = map_rows_by_head(&tm_do, T::kFmt, dout, dos, batch, s.m, s.h, D, b.gb, b.tt);
    if (st == DSA_OK) st = map_head_by_rows(&tm_k, T::kFmt, x.k, x.ks, batch, s.n, s.hk, D, kRows);
    if (st == DSA_OK) st = map_head_by_rows(&tm_v, T::kFmt, x.v, x.vs, batch, s.n, s.hk, D, kRows);
    if (st != DSA_OK) return st;
    DkvParams p;
    p.s = s;
    p.gb = b.gb;
    p.hb = b.hb;
    p.tt = b.tt;
    p.key_tiles = b.key_tiles;
    p.first_tiles = b.first_tiles;
    p.split_first = b.split_first;
    p.split = b.split;
    p.units_per_head = b.units_per_head;
    p.units = b.units;
    p.scale = scale;
    p.scale_log2 = scale * kLog2e;
    p.stat = stat;
    p.dk = static_cast<uint16_t*>(dk);
    p.dv = static_cast<uint16_t*>(dv);
    p.parts = reinterpret_cast<float*>(ws + b.off_parts);
    p.err = err;
    auto kernel = window_dkv_kernel<T, D>;
    st = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), DkvCfg<D>::kSmemBytes);
    if (st != DSA_OK) return st;
    const int64_t grid = p.units < di.num_sms ? p.units : di.num_sms;
    kernel<<<static_cast<unsigned>(grid), kBwdThreads, DkvCfg<D>::kSmemBytes, stream>>>(
        tm_q, tm_do, tm_k, tm_v, p, peaks);
    st = cuda_status(cudaGetLastError());
    if (st != DSA_OK) return st;
    const int tiles = b.split > 1 ? b.key_tiles : (b.split_first > 1 ? b.first_tiles : 0);
    if (tiles > 0) {
      const int64_t warps = batch * s.hk * tiles * (dv ? 2 : 1) * kRows * (D / 16);
      window_join_kernel<T, D><<<static_cast<unsigned>(div_up(warps, 8)), 256, 0, stream>>>(p, batch);
      st = cuda_status(cudaGetLastError());
      if (st != DSA_OK) return st;
    }
  }
  if (rows == 0) {
    if (dsink != nullptr) return cuda_status(cudaMemsetAsync(dsink, 0, s.h * sizeof(float), stream));
    return DSA_OK;
  }
  DqParams p;
  p.s = s;
  if (!tile_grid(s, batch, &p.grid)) return DSA_ERR_UNSUPPORTED;
  p.scale = scale;
  p.scale_log2 = scale * kLog2e;
  p.stat = stat;
  p.peaks = peaks;
  p.sink = dsink != nullptr ? sink : nullptr;
  p.dq = static_cast<uint16_t*>(dq);
  p.sink_rows = sink_rows;
  p.shared = x.v == x.k && same_strides(x.vs, x.ks);
  p.err = err;
  st = map_rows_by_head(&tm_q, T::kFmt, x.q, x.qs, batch, s.m, s.h, D, s.g, p.grid.tt);
  if (st == DSA_OK)
    st = map_rows_by_head(&tm_do, T::kFmt, dout, dos, batch, s.m, s.h, D, s.g, p.grid.tt);
  if (st == DSA_OK) st = map_head_by_rows(&tm_k, T::kFmt, x.k, x.ks, batch, s.n, s.hk, D, kBlk);
  if (st == DSA_OK) st = map_head_by_rows(&tm_v, T::kFmt, x.v, x.vs, batch, s.n, s.hk, D, kBlk);
  if (st != DSA_OK) return st;
  auto kernel = window_dq_kernel<T, D>;
  st = set_max_dynamic_smem(reinterpret_cast<const void*>(kernel), DqCfg<D>::kSmemBytes);
  if (st != DSA_OK) return st;
  const int grid = p.grid.items < di.num_sms ? p.grid.items : di.num_sms;
  kernel<<<static_cast<unsigned>(grid), kBwdThreads, DqCfg<D>::kSmemBytes, stream>>>(tm_q, tm_do, tm_k,
                                                                                    tm_v, p);
  st = cuda_status(cudaGetLastError());
  if (st != DSA_OK || dsink == nullptr) return st;
  // rows of all heads -> blocks of rows -> one row; more steps while one block is not enough
  const float* in = sink_rows;
  int64_t left = batch * s.m;
  float* sums = sink_sum;
  const unsigned hx = static_cast<unsigned>(div_up(s.h, 32));
  while (true) {
    const int64_t blocks = div_up(left, kSinkRows);
    const bool end = blocks == 1;
    window_dsink_kernel<<<dim3(static_cast<unsigned>(blocks), hx), 256, 0, stream>>>(
        in, end ? dsink : sums, left, s.h, end ? -1.f : 1.f);
    st = cuda_status(cudaGetLastError());
    if (st != DSA_OK || end) return st;
    // the next step reads this one's sums and writes over the rows, which are done with
    in = sums;
    left = blocks;
    sums = sums == sink_sum ? sink_rows : sink_sum;
  }
}

}  // namespace win
}  // namespace dsa

extern "C" size_t dsa_window_attn_bwd_workspace_bytes(int64_t batch, int64_t m, int64_t n,
                                                      int n_heads, int n_kv_heads, int head_dim,
                                                      int64_t window, int64_t n_first, int shared_kv) {
  using namespace dsa::win;
  static const char dummy = 0;
  const void* at = reinterpret_cast<const void*>(reinterpret_cast<uintptr_t>(&dummy) & ~uintptr_t{15});
  Tensors x;
  Shape s;
  if (check_window_args(at, nullptr, at, nullptr, at, nullptr, nullptr, DSA_DTYPE_BF16, batch, m, n,
                        n_heads, n_kv_heads, head_dim, window, n_first, 1.f, &x, &s) != DSA_OK)
    return 0;
  return plan_bwd(s, batch, head_dim, shared_kv != 0).bytes;
}

extern "C" int dsa_window_attn_bwd(const void* q, const int64_t* q_strides, const void* k,
                                   const int64_t* k_strides, const void* v,
                                   const int64_t* v_strides, const float* sink, const int* kv_lens,
                                   const void* out, const float* lse, const void* dout,
                                   const int64_t* dout_strides, void* dq, void* dk, void* dv,
                                   float* dsink, int dtype, int64_t batch, int64_t m, int64_t n,
                                   int n_heads, int n_kv_heads, int head_dim, int64_t window,
                                   int64_t n_first, float softmax_scale, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace dsa;
  using namespace dsa::win;
  Tensors x;
  Shape s;
  int st = check_window_args(q, q_strides, k, k_strides, v, v_strides, kv_lens, dtype, batch, m, n,
                             n_heads, n_kv_heads, head_dim, window, n_first, softmax_scale, &x, &s);
  if (st != DSA_OK) return st;
  Strides dos;
  st = read_strides(dout_strides, batch, m, n_heads, head_dim, &dos);
  if (st != DSA_OK) return st;
  const bool shared = dv == nullptr;
  if (shared && !(x.v == x.k && same_strides(x.vs, x.ks))) return DSA_ERR_INVALID_ARGUMENT;
  if (dsink != nullptr && sink == nullptr) return DSA_ERR_INVALID_ARGUMENT;
  cudaStream_t cs = static_cast<cudaStream_t>(stream);
  if (batch == 0)
    return dsink ? cuda_status(cudaMemsetAsync(dsink, 0, n_heads * sizeof(float), cs)) : DSA_OK;
  if (m > 0 && (out == nullptr || lse == nullptr || dout == nullptr || dq == nullptr))
    return DSA_ERR_INVALID_ARGUMENT;
  if (n > 0 && dk == nullptr) return DSA_ERR_INVALID_ARGUMENT;
  if (!aligned16(out) || !aligned16(dout) || !aligned16(dq) || !aligned16(dk) || !aligned16(dv))
    return DSA_ERR_MISALIGNED;
  if (m == 0) {  // no row sees any key
    const size_t bytes = static_cast<size_t>(batch) * n * n_kv_heads * head_dim * 2;
    if (n > 0) st = cuda_status(cudaMemsetAsync(dk, 0, bytes, cs));
    if (st == DSA_OK && n > 0 && dv) st = cuda_status(cudaMemsetAsync(dv, 0, bytes, cs));
    if (st == DSA_OK && dsink)
      st = cuda_status(cudaMemsetAsync(dsink, 0, n_heads * sizeof(float), cs));
    return st;
  }
  const BwdPlan b = plan_bwd(s, batch, head_dim, shared);
  if (workspace == nullptr || workspace_bytes < b.bytes) return DSA_ERR_WORKSPACE;
  if ((reinterpret_cast<uintptr_t>(workspace) & 255u) != 0) return DSA_ERR_MISALIGNED;
  if (b.units > (int64_t{1} << 40) || batch * m * n_heads > (int64_t{1} << 34))
    return DSA_ERR_UNSUPPORTED;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  if (head_dim == 128)
    return dtype == DSA_DTYPE_BF16
               ? launch_bwd<Bf16, 128>(x, s, batch, softmax_scale, sink, out, dout, dos, lse, dq, dk,
                                       dv, dsink, ws, b, cs)
               : launch_bwd<Fp16, 128>(x, s, batch, softmax_scale, sink, out, dout, dos, lse, dq, dk,
                                       dv, dsink, ws, b, cs);
  return dtype == DSA_DTYPE_BF16
             ? launch_bwd<Bf16, 64>(x, s, batch, softmax_scale, sink, out, dout, dos, lse, dq, dk, dv,
                                    dsink, ws, b, cs)
             : launch_bwd<Fp16, 64>(x, s, batch, softmax_scale, sink, out, dout, dos, lse, dq, dk, dv,
                                    dsink, ws, b, cs);
}
