// Attention over packed sequences, backward.
//
//   P_ij = exp(scale q_i.k_j - lse_i)          delta_i = dO_i . O_i
//   dS_ij = P_ij (dO_i . v_j - delta_i)
//   dV_j = sum_i P_ij dO_i      dK_j = scale sum_i dS_ij q_i      dQ_i = scale sum_j dS_ij k_j
//
// Two launches: delta (and lse in powers of two) per row; then one grid whose first CTAs are the keys' side (dK, dV) and whose
// others are the queries' side (dQ): they read the same inputs, write nothing in common, and the queries' side fills the SMs
// that the keys' side leaves free.  Scores and
// probabilities are formed again in both: two sums that each stay in one CTA's TMEM, so every gradient is
// written once, in its own type, and there are no atomics -- the same bits every time.  The rows of a tile are packed from
// the group's heads as in the forward pass, which makes the sum over a group's heads part of the product.
//
// One scheme for both sides.  The lane side (128 rows) stays in shared memory, the streamed side passes through two rings:
//   kDkv : lanes = keys;    streamed: Q (ring A), dO (ring B)     S^T = K Q^T, dP^T = V dO^T, dV += P^T dO, dK += dS^T Q
//   kDq  : lanes = queries; streamed: K (ring A), V (ring B)      S = Q K^T,   dP = dO V^T,   dQ += dS K
// warp 0: TMA producer; warp 1: issues S and dP; warp 2: lse and delta of the streamed rows (kDkv); warp 3: issues the
// gradient products, and zeroes the streamed rows behind the sequence's end (they are summed over, and 0 x NaN would reach
// the sums); warps 4..19: sixteen warps turn a tile's S and dP into P and dS, (row quarter, 32 of the columns) each.  P (kDkv)
// and dS go back into TMEM as bf16 pairs over the columns of dP that the warp has read, as the A operand of the gradient products
// (16-bit operands: each entry is off by at most 2^-8); S's columns are free as soon as it is in registers, so the next tile's
// products are formed meanwhile.
//
// Bound: the tensor pipe, 48 (D = 64) and 66 % (D = 128) busy, and the threads that issue to it (one is blocked 75 to 95 cycles an
// instruction, which is why there are two).  Both sides: 8188 tokens in 3 sequences, 12 heads of 64: 471 us; 8192 causal tokens,
// 16 heads of 128 sharing two key heads: 780 us.
#include <algorithm>
#include <cmath>
#include <cstring>

#include "packed.cuh"

namespace swv {

bool packed_aligned(const void* p, const int64_t* s, int es);
int packed_tmap(CUtensorMap* out, const void* base, const int64_t* s, int64_t tokens, int heads_kv, int group, int d,
                int box_tok);
int packed_plan_header(const int32_t* plan_host, PackedHeader* h);

namespace {

enum { kDkv = 0, kDq = 1 };
constexpr int kBwdWarps = 16;                  // warps that turn a tile's products into P and dS, 32 columns each
constexpr int kBwdThreads = 128 + 32 * kBwdWarps;
constexpr int kBwdRegsControl = 64, kBwdRegsTerms = 104;        // of 640 x 96 = 61440 at launch: all
constexpr int kBwdRegs = 128 * kBwdRegsControl + 32 * kBwdWarps * kBwdRegsTerms;

struct PackedBwdParams {
  const PackedUnit* units;
  int n_units, group, group_inv, tok, Tq, d, Hkv, heads_at_once;
  const float2* stats;          // [Hkv][Tq][group] {-lse in powers of two, -delta}; -inf where a row sees no key
  void *g1, *g2;                // kDkv: dK, dV; kDq: dQ
  int64_t g1_t, g1_h, g2_t, g2_h;
  float scale, scale_log2;
  float* part;                  // [slot][Hkv][128][D (kDq) or 2 D (kDkv: dV, dK)] sums of divided units, before the scale
  int* status;
};

template <int D, int MODE>
struct BwdCfg {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kA = D == 64 ? 4 : (MODE == kDkv ? 2 : 3);       // stages of ring A and ring B
  static constexpr int kB = D == 64 ? 4 : (MODE == kDkv ? 2 : 1);
  static constexpr int kOffA = 2 * kTileBytes;
  static constexpr int kOffB = kOffA + kA * kTileBytes;
  // kDkv: two tiles of 128 rows of 128 bytes (see the warp that fills them)
  static constexpr int kOffOnes = kOffB + kB * kTileBytes;
  static constexpr int kOffStats = kOffOnes + (MODE == kDkv ? kTile * 128 : 0);
  static constexpr int kOffCtl = kOffStats + (MODE == kDkv ? kTile * 128 : 0);
  // TMEM.  Where two accumulators of 128 columns leave room for two tiles only (kTurns), a tile's S and dP take turns in one of
  // them: dP is formed there once S has been read, while P is computed, and P and dS go over it.  Otherwise S has a tile of its
  // own and dP two.  (One tile for S, one for dP: dP(j+1) waits for the gradients of tile j, which cost 500 us where this
  // takes 473 at 8192 causal tokens, 16 heads of 128 sharing two key heads.)
  static constexpr bool kTurns = MODE == kDkv && D == 128;
  static constexpr uint32_t kColG = kTurns ? 256 : 384;
  __device__ static uint32_t s_tile(int j) { return kTurns ? (j & 1) * 128 : 0; }
  __device__ static uint32_t dp_tile(int j) { return kTurns ? (j & 1) * 128 : 128 + (j & 1) * 128; }
};
struct BwdCtl {
  uint64_t lane_full, a_full[4], a_empty[4], b_full[4], b_empty[4], tail_a, tail_b;
  uint64_t s_full, s_read, dp_full[2], ds_ready[2], ds_done[2], all_done, stat_full[2], stat_empty[2], staged;
  uint32_t tmem_base, abort_flag;
};
template <int D, int MODE>
constexpr size_t bwd_smem() { return 1024 + BwdCfg<D, MODE>::kOffCtl + sizeof(BwdCtl) + 64; }

// bits [lo, hi) of the 32 columns from `base` on
__device__ __forceinline__ uint32_t column_bits(int lo, int hi, int base) {
  auto low = [](int n) { return n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << n) - 1u); };
  return low(hi - base) & ~low(lo - base);
}

// zeroes rows [first, 128) of a tile of D / 64 swizzled halves (whole 128-byte rows, so the swizzle does not matter)
template <int D>
__device__ __forceinline__ void zero_rows(uint32_t tile, int first, int thread, int threads) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
    for (int i = first * 8 + thread; i < kTile * 8; i += threads) sts128(tile + c * (kTile * 128) + i * 16, 0u, 0u, 0u, 0u);
}

// What CTA `block` of a side does; everything that earlier kernels wrote is there.
template <int D, int MODE>
__device__ __forceinline__ void bwd_side(const CUtensorMap& tm_l1, const CUtensorMap& tm_l2, const CUtensorMap& tm_a,
                                         const CUtensorMap& tm_b, const PackedBwdParams& p, int block) {
  using Cfg = BwdCfg<D, MODE>;
  constexpr int NA = Cfg::kA, NB = Cfg::kB, TB = Cfg::kTileBytes;
  constexpr uint32_t kIdescS = make_idesc(/*bf16*/ 1, kTile, kTile, 0, 0);
  constexpr uint32_t kIdescG = make_idesc(/*bf16*/ 1, kTile, D, 0, /*B is MN-major*/ 1);
  constexpr uint32_t kColG = Cfg::kColG;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  BwdCtl* ctl = reinterpret_cast<BwdCtl*>(smem + Cfg::kOffCtl);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  int kvh;
  const PackedUnit u = packed_unit(p.units, p.n_units, p.Hkv, p.heads_at_once, block, kvh);
  if (threadIdx.x == 0) {
    mbar_init(&ctl->lane_full, 1);
    for (int s = 0; s < 4; ++s) {
      mbar_init(&ctl->a_full[s], 1);
      mbar_init(&ctl->a_empty[s], 1);
      mbar_init(&ctl->b_full[s], 1);
      mbar_init(&ctl->b_empty[s], 1);
    }
    mbar_init(&ctl->tail_a, 1);
    mbar_init(&ctl->tail_b, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&ctl->stat_full[s], 1);
      mbar_init(&ctl->stat_empty[s], 1);
      mbar_init(&ctl->dp_full[s], 1);
      mbar_init(&ctl->ds_ready[s], kBwdWarps);
      mbar_init(&ctl->ds_done[s], 1);
    }
    mbar_init(&ctl->s_full, 1);
    mbar_init(&ctl->s_read, kBwdWarps);
    mbar_init(&ctl->all_done, 1);
    mbar_init(&ctl->staged, kBwdWarps);
    ctl->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  const int n = u.b1 - u.b0;
  const int per = MODE == kDkv ? p.tok * p.group : kTile;      // streamed rows a tile
  const int step = MODE == kDkv ? p.tok : kTile;               // streamed tokens a tile
  const int last_rows = min(step, u.len - (u.b1 - 1) * step) * (MODE == kDkv ? p.group : 1);
  const bool tail = n > 0 && last_rows < per;                  // the last tile holds rows behind the sequence

  if (MODE == kDkv) {
    // rows that no load fills: they are summed over as zeros
    if (per < kTile)
      for (int s = 0; s < NA + NB; ++s) zero_rows<D>(smem_u32(smem + Cfg::kOffA + s * TB), per, threadIdx.x, kBwdThreads);
    // row r of the tile of ones: {1, 1, 1, 0, ...} in its first 16 channels
    for (int i = threadIdx.x; i < kTile * 8; i += kBwdThreads) {
      const int r = i >> 3, chunk = (i & 7) ^ (r & 7);
      sts128(smem_u32(smem + Cfg::kOffOnes) + i * 16, chunk == 0 ? 0x3f803f80u : 0u, chunk == 0 ? 0x3f80u : 0u, 0u, 0u);
      sts128(smem_u32(smem + Cfg::kOffStats) + i * 16, 0u, 0u, 0u, 0u);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl->tmem_base;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  grid_release();                                              // (after the wait of every thread of the CTA)
  auto wait = [&](uint64_t* bar, uint32_t parity, int code) {
    if (mbar_wait_bounded(bar, parity, abort_flag)) return true;
    record_status(p.status, code);
    return false;
  };

  if (warp < 4) {
  reg_dec<kBwdRegsControl>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && n > 0) {
      mbar_expect_tx(&ctl->lane_full, 2 * (MODE == kDkv ? TB : p.tok * p.group * D * 2));
#pragma unroll
      for (int c = 0; c < D / 64; ++c) {
        if (MODE == kDkv) {
          tma_load_3d(smem + c * (kTile * 128), &tm_l1, &ctl->lane_full, c * 64, u.t0, kvh);
          tma_load_3d(smem + TB + c * (kTile * 128), &tm_l2, &ctl->lane_full, c * 64, u.t0, kvh);
        } else {
          tma_load_4d(smem + c * (kTile * 128), &tm_l1, &ctl->lane_full, c * 64, 0, u.t0, kvh);
          tma_load_4d(smem + TB + c * (kTile * 128), &tm_l2, &ctl->lane_full, c * 64, 0, u.t0, kvh);
        }
      }
      int loads[2] = {0, 0};                                    // of ring A and ring B
      for (int j = 0; j < n; ++j) {
        const int at = u.s0 + (u.b0 + j) * step;
        // (the stages of the tail are declared full by the warp that cleans them)
        const bool cut = tail && j == n - 1;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int N = r == 0 ? NA : NB, s = j % N;
          uint64_t* full = r == 0 ? &ctl->a_full[s] : &ctl->b_full[s];
          if (*abort_flag != 0u || !wait(r == 0 ? &ctl->a_empty[s] : &ctl->b_empty[s], ((j / N) & 1) ^ 1, kDevWaitStageEmpty))
            break;
          uint8_t* dst = smem + (r == 0 ? Cfg::kOffA : Cfg::kOffB) + s * TB;
          uint64_t* bar = !cut ? full : r == 0 ? &ctl->tail_a : (MODE == kDkv ? &ctl->tail_b : full);
          mbar_expect_tx(bar, per * D * 2);
          ++loads[r];
          const CUtensorMap* tm = r == 0 ? &tm_a : &tm_b;
#pragma unroll
          for (int c = 0; c < D / 64; ++c) {
            if (MODE == kDkv) tma_load_4d(dst + c * (kTile * 128), tm, bar, c * 64, 0, at, kvh);
            else tma_load_3d(dst + c * (kTile * 128), tm, bar, c * 64, at, kvh);
          }
        }
        if (*abort_flag != 0u) break;
      }
      drain_copy(&ctl->lane_full, 0);
      for (int r = 0; r < 2; ++r) {
        const int N = r == 0 ? NA : NB;
        for (int j = max(0, loads[r] - N); j < loads[r]; ++j) {
          const bool cut = tail && j == n - 1 && (r == 0 || MODE == kDkv);
          uint64_t* bar = cut ? (r == 0 ? &ctl->tail_a : &ctl->tail_b) : r == 0 ? &ctl->a_full[j % N] : &ctl->b_full[j % N];
          drain_copy(bar, cut ? 0 : (j / N) & 1);
        }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------- issues S and dP of every tile
    if (lane == 0 && n > 0) {
      const uint32_t l1 = smem_u32(smem), l2 = l1 + TB, ra = l1 + Cfg::kOffA, rb = l1 + Cfg::kOffB;
      auto product = [&](uint32_t col, uint32_t a, uint32_t b) {          // both operands along the channels
        const uint64_t da = smem_desc_sw128(a), db = smem_desc_sw128(b);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t off = (ks >> 2) * (kTile * 128 / 16) + (ks & 3) * 2;
          umma_f16_ss(col, da + off, db + off, kIdescS, ks > 0);
        }
      };
      // col += 1 x (row statistic of the streamed side): 16 more channels, see the warp that fills them
      auto plus_stat = [&](uint32_t col, int channels16) {
        umma_f16_ss(col, smem_desc_sw128(l1 + Cfg::kOffOnes), smem_desc_sw128(l1 + Cfg::kOffStats) + channels16 * 2, kIdescS, 1);
      };
      bool ok = wait(&ctl->lane_full, 0, kDevWaitQ);
      for (int j = 0; ok && j < n; ++j) {
        ok = wait(&ctl->a_full[j % NA], (j / NA) & 1, kDevWaitTmaFull) &&
             (MODE == kDq || wait(&ctl->stat_full[j & 1], (j >> 1) & 1, kDevWaitTmaFull)) &&
             (Cfg::kTurns ? j < 2 || wait(&ctl->ds_done[j & 1], ((j >> 1) & 1) ^ 1, kDevWaitPvDone)      // dS(j-2) lay there
                          : j == 0 || wait(&ctl->s_read, (j - 1) & 1, kDevWaitAccEmpty));                // S(j-1)
        if (!ok) break;
        tc_fence_after();
        product(tmem_base + Cfg::s_tile(j), l1, ra + (j % NA) * TB);
        if (MODE == kDkv) plus_stat(tmem_base + Cfg::s_tile(j), (j & 1) * 2);
        umma_commit(&ctl->s_full);
        ok = wait(&ctl->b_full[j % NB], (j / NB) & 1, kDevWaitTmaFull) &&
             (Cfg::kTurns ? wait(&ctl->s_read, j & 1, kDevWaitAccEmpty)                                  // S(j) lay there
                          : j < 2 || wait(&ctl->ds_done[j & 1], ((j >> 1) & 1) ^ 1, kDevWaitPvDone));    // dS(j-2)
        if (!ok) break;
        tc_fence_after();
        const uint32_t col = tmem_base + Cfg::dp_tile(j);
        product(col, l2, rb + (j % NB) * TB);
        if (MODE == kDkv) {
          plus_stat(col, (j & 1) * 2 + 1);
          umma_commit(&ctl->stat_empty[j & 1]);
        } else {
          umma_commit(&ctl->b_empty[j % NB]);
        }
        umma_commit(&ctl->dp_full[j & 1]);
      }
    }
  } else if (warp == 2) {
    // Row statistics of the streamed queries (kDkv).  S - lse / scale and dP - delta are formed by the products themselves: a
    // tile of ones times the statistic, as three bf16 terms whose sum has all 24 bits (the columns' values read from
    // shared memory by every thread cost 65 of 419 us at 3 bags of 12 heads of 64).  Channels of the 128-byte rows: two tiles' lse
    // and delta in 16 each, of which three are used.
    if (MODE == kDkv) {
      const uint32_t tile = smem_u32(smem + Cfg::kOffStats);
      const float per_score = 1.f / p.scale_log2;
      for (int j = 0; j < n; ++j) {
        const int tok0 = (u.b0 + j) * step;
        const int rows = min(step, u.len - tok0) * p.group;
        const float2* src = p.stats + (static_cast<int64_t>(kvh) * p.Tq + u.s0 + tok0) * p.group;
        float2 f[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 32 + lane;
          f[i] = r < rows ? load_written(src + r) : make_float2(0.f, 0.f);
        }
        bool ok = j < 2 || wait(&ctl->stat_empty[j & 1], ((j >> 1) & 1) ^ 1, kDevWaitAccEmpty);
        if (!__all_sync(0xffffffffu, ok)) break;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int r = i * 32 + lane;
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const float x = k == 0 ? f[i].x * per_score : f[i].y;
            const uint32_t hi = __float_as_uint(x) & 0xffff0000u;
            const bool finite = fabsf(x) < __int_as_float(0x7f800000);
            const float y = finite ? x - __uint_as_float(hi) : 0.f;      // (an infinity is one term; NaN stays in the first)
            const uint32_t mid = __float_as_uint(y) & 0xffff0000u;
            const uint32_t lo = __float_as_uint(y - __uint_as_float(mid));
            const int chunk = ((j & 1) * 2 + k) * 2;
            sts128(tile + r * 128 + ((chunk ^ (r & 7)) << 4), ((x == x ? hi : 0x7fc00000u) >> 16) | mid, lo >> 16, 0u, 0u);
          }
        }
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->stat_full[j & 1]);
      }
    }
  } else {
    // -------------- zeroes the rows behind the sequence's end in the last tile, and issues the gradient products
    bool ok = n > 0;
    auto clean = [&]() {
      bool r = wait(&ctl->tail_a, 0, kDevWaitTmaFull) && (MODE == kDq || wait(&ctl->tail_b, 0, kDevWaitTmaFull));
      r = __all_sync(0xffffffffu, r);
      if (r) {
        const int sa = (n - 1) % NA, sb = (n - 1) % NB;
        zero_rows<D>(smem_u32(smem + Cfg::kOffA + sa * TB), last_rows, lane, 32);
        if (MODE == kDkv) zero_rows<D>(smem_u32(smem + Cfg::kOffB + sb * TB), last_rows, lane, 32);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ctl->a_full[sa]);
          if (MODE == kDkv) mbar_arrive(&ctl->b_full[sb]);
        }
      }
      return r;
    };
    const uint32_t ra = smem_u32(smem) + Cfg::kOffA, rb = smem_u32(smem) + Cfg::kOffB;
    auto gradient = [&](uint32_t col, uint32_t a_col, uint32_t b, bool first) {     // the 128 streamed rows are summed over
      const uint64_t db = smem_desc_sw128(b, kTile * 128);
#pragma unroll
      for (int ks = 0; ks < kTile / 16; ++ks)
        umma_f16_ts(col, a_col + (ks >> 1) * 32 + (ks & 1) * 8, db + ks * 128, kIdescG, !first || ks > 0);
    };
    // The last tile lands while tile n - 2 is worked on at the latest: its loads wait for the stages of tiles n - 1 - NA
    // and n - 1 - NB, which the products of tile n - 2 no longer need.
    for (int j = 0; ok && j < n; ++j) {
      if (tail && j == max(n - 2, 0)) ok = clean();
      if (!ok) break;
      ok = wait(&ctl->ds_ready[j & 1], (j >> 1) & 1, kDevWaitPReady);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      if (lane == 0) {
        tc_fence_after();
        const uint32_t col = tmem_base + Cfg::dp_tile(j);
        gradient(tmem_base + kColG + (MODE == kDkv ? D : 0), col + 16, ra + (j % NA) * TB, j == 0);   // (dK first: Q's stage
        umma_commit(&ctl->a_empty[j % NA]);                                                           // is wanted sooner)
        if (MODE == kDkv) {
          gradient(tmem_base + kColG, col, rb + (j % NB) * TB, j == 0);
          umma_commit(&ctl->b_empty[j % NB]);
        }
        umma_commit(j + 1 < n ? &ctl->ds_done[j & 1] : &ctl->all_done);
      }
      __syncwarp();
    }
  }
  } else {
    // ------------------------------- sixteen warps: (row quarter, 32 of the columns)
    reg_inc<kBwdRegsTerms>();
    const int quarter = warp & 3, grp = (warp - 4) >> 2;
    const int row = quarter * 32 + lane, c0 = grp * 32;
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const float c2 = p.scale_log2;
    bool ok = true;
    float neg_lse = 0.f, neg_delta = 0.f;
    int limit = 0;                                             // kDq: keys the row sees from block b0 on
    const int rows = MODE == kDkv ? u.n : u.n * p.group;
    const bool row_ok = row < rows;
    const int tk = MODE == kDkv ? row : row_token(row, p.group_inv);         // token of the lane side
    if (MODE == kDq && row_ok) {
      const float2 f = load_written(p.stats + (static_cast<int64_t>(kvh) * p.Tq + u.t0) * p.group + row);
      neg_lse = f.x;
      neg_delta = f.y;
      limit = min(u.len, u.off + tk + 1) - u.b0 * kTile;
    }
    for (int j = 0; j < n; ++j) {
      const uint32_t s_col = tmem_base + lane_off + Cfg::s_tile(j) + c0;
      const uint32_t dp_col = tmem_base + lane_off + Cfg::dp_tile(j) + c0;
      // the columns that the row sees: keys before its limit, or queries from `lo` on
      int lo = 0, hi;
      if (MODE == kDq) {
        hi = limit - j * kTile;
      } else {
        const int tok0 = (u.b0 + j) * step;
        lo = min(max(u.off + row - tok0, 0), step) * p.group;
        hi = min(step, u.len - tok0) * p.group;
      }
      const uint32_t vis = column_bits(lo, hi, c0);
      const bool all = __all_sync(0xffffffffu, vis == 0xffffffffu);
      ok = wait(&ctl->s_full, j & 1, kDevWaitAccFull);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      float pr[32];
      {
        uint32_t s[32];
        tmem_ld32(s_col, s);
        tc_wait_ld();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->s_read);              // S(j+1) or dP(j) may go there
#pragma unroll
        for (int i = 0; i < 32; i += 2) {                      // (kDkv: the scores hold -lse already)
          fma2(pr[i], pr[i + 1], __uint_as_float(s[i]), __uint_as_float(s[i + 1]), c2, neg_lse, neg_lse);
          pr[i] = ex2_approx(pr[i]);
          pr[i + 1] = ex2_approx(pr[i + 1]);
        }
        if (!all) {
          KEEP_BRANCH();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((vis >> i) & 1u)) pr[i] = 0.f;
        }
      }
      ok = wait(&ctl->dp_full[j & 1], (j >> 1) & 1, kDevWaitAccFull);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t w[16];
      {
        uint32_t x[32];
        tmem_ld32(dp_col, x);
        tc_wait_ld();
        if (!all) {                                            // (what lies behind the sequence may be infinite)
          KEEP_BRANCH();
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!((vis >> i) & 1u)) x[i] = 0u;
        }
        if (MODE == kDkv) {                                    // P over the first half of the warp's own columns of dP
#pragma unroll
          for (int i = 0; i < 16; ++i) w[i] = pack_bf16x2(pr[2 * i], pr[2 * i + 1]);
          tmem_st16(dp_col, w);
        }
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          float y0 = __uint_as_float(x[i]), y1 = __uint_as_float(x[i + 1]);
          if (MODE == kDq) add2(y0, y1, neg_delta, neg_delta);  // (kDkv: -delta is in dP already)
          mul2(y0, y1, pr[i], pr[i + 1]);
          w[i / 2] = pack_bf16x2(y0, y1);
        }
      }
      tmem_st16(dp_col + 16, w);                               // dS over the second half of them
      tc_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->ds_ready[j & 1]);
    }
    if (ok && n > 0) ok = wait(&ctl->all_done, 0, kDevWaitPvDone);
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    // The gradients: kDkv groups 0 and 1 take the halves of dV, 2 and 3 those of dK; kDq each a quarter of dQ.
    constexpr int kCols = MODE == kDkv ? D / 2 : D / 4;
    constexpr int kWidth = MODE == kDkv ? 2 * D : D;
    const uint32_t col = tmem_base + lane_off + kColG + grp * kCols;
    const bool is_dv = MODE == kDkv && grp < 2;
    const bool divided = u.slot >= 0;
    // (the lane side's tiles are no longer needed: dV or dQ over the first, dK over the second)
    const uint32_t stage = smem_u32(smem) + (MODE == kDkv && !is_dv ? TB : 0);
    const int ch0 = MODE == kDkv ? (grp & 1) * kCols : grp * kCols;
    if (ok) {
      const float f = is_dv ? 1.f : p.scale;
      float* part = p.part + ((static_cast<int64_t>(divided ? u.slot : 0) * p.Hkv + kvh) * kTile + row) * kWidth + grp * kCols;
      constexpr int kStep = kCols < 32 ? kCols : 32;           // (kDq at D = 64: 16 columns a warp)
#pragma unroll 1
      for (int c = 0; c < kCols / kStep; ++c) {
        uint32_t o[32];
        if (n > 0) {
          if constexpr (kStep == 32) tmem_ld32(col + c * 32, o);
          else tmem_ld16(col, *reinterpret_cast<uint32_t(*)[16]>(o));
          tc_wait_ld();
        } else {
#pragma unroll
          for (int i = 0; i < kStep; ++i) o[i] = 0u;
        }
        if (!divided) {
          stage_columns<D, kStep>(stage, row, ch0 / kStep + c, o, f);
        } else if (row_ok) {
#pragma unroll
          for (int i = 0; i < kStep; i += 4)
            *reinterpret_cast<uint4*>(part + c * 32 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      }
    }
    if (ok && !divided) {
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->staged);
      ok = wait(&ctl->staged, 0, kDevWaitAccEmpty);
      ok = __all_sync(0xffffffffu, ok);
      // sixteen warps write eight rows each of every gradient
      const int r0 = (warp - 4) * 8, r1 = min(rows, r0 + 8);
      if (ok && MODE == kDkv) {
        uint16_t* dv = static_cast<uint16_t*>(p.g2) + static_cast<int64_t>(u.t0) * p.g2_t + static_cast<int64_t>(kvh) * p.g2_h;
        uint16_t* dk = static_cast<uint16_t*>(p.g1) + static_cast<int64_t>(u.t0) * p.g1_t + static_cast<int64_t>(kvh) * p.g1_h;
        write_staged<D>(smem_u32(smem), r0, r1, p.d, [&](int r) { return dv + r * p.g2_t; });
        write_staged<D>(smem_u32(smem) + TB, r0, r1, p.d, [&](int r) { return dk + r * p.g1_t; });
      } else if (ok) {
        uint16_t* dq = static_cast<uint16_t*>(p.g1) + static_cast<int64_t>(u.t0) * p.g1_t +
                       static_cast<int64_t>(kvh) * p.group * p.g1_h;
        write_staged<D>(smem_u32(smem), r0, r1, p.d,
                        [&](int r) {
                          const int w = row_token(r, p.group_inv);
                          return dq + w * p.g1_t + (r - w * p.group) * p.g1_h;
                        });
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    __syncwarp();
    tmem_dealloc(tmem_base, 512);
  }
}

template <int D>
__global__ void __launch_bounds__(kBwdThreads, 1)
    packed_attn_bwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_g,
                           const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                           const PackedBwdParams keys, const PackedBwdParams queries) {
  if (threadIdx.x == 0) {                            // (fetched during the wait)
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_g);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  grid_wait();                                       // of every CTA: both sides read delta, q, k, v and dO
  const int first = keys.n_units * keys.Hkv;
  if (static_cast<int>(blockIdx.x) < first) bwd_side<D, kDkv>(tm_k, tm_v, tm_q, tm_g, keys, blockIdx.x);
  else bwd_side<D, kDq>(tm_q, tm_g, tm_k, tm_v, queries, blockIdx.x - first);
}

// -delta = -dO . O per row, and -lse in powers of two.  L lanes a row (8 channels each), four rows a thread in flight.  Bound: HBM.
constexpr int kDeltaRows = 4;
template <int L>
__global__ void __launch_bounds__(256) packed_attn_delta_kernel(const __nv_bfloat16* o, int64_t os_t, int64_t os_h,
                                                                const __nv_bfloat16* g, int64_t gs_t, int64_t gs_h,
                                                                const float* lse, float2* stats, int Tq, int tokens,
                                                                int group, int d) {
  grid_wait();
  grid_release();
  constexpr int kAtOnce = 256 / L;                             // rows a CTA has in flight in each step
  const int sub = threadIdx.x % L, kvh = blockIdx.y, c = sub * 8;
  // rows in the order of the tiles: [kv head][token][head of the group]
  const int64_t first = static_cast<int64_t>(blockIdx.x) * (kAtOnce * kDeltaRows);
  const int64_t t0 = first / group;
  const int rest = static_cast<int>(first - t0 * group) + threadIdx.x / L;
  uint4 x[kDeltaRows], y[kDeltaRows];
  float l[kDeltaRows];
  int64_t t[kDeltaRows];
  int hg[kDeltaRows];
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    const int j = rest + i * kAtOnce;
    t[i] = t0 + j / group;
    hg[i] = j % group;
    const int head = kvh * group + hg[i];
    x[i] = y[i] = make_uint4(0u, 0u, 0u, 0u);
    l[i] = 0.f;
    if (t[i] >= tokens) continue;
    if (c < d) {
      x[i] = *reinterpret_cast<const uint4*>(o + t[i] * os_t + head * os_h + c);
      y[i] = *reinterpret_cast<const uint4*>(g + t[i] * gs_t + head * gs_h + c);
    }
    if (sub == 0) l[i] = lse[static_cast<int64_t>(head) * Tq + t[i]];
  }
#pragma unroll
  for (int i = 0; i < kDeltaRows; ++i) {
    const uint32_t xs[4] = {x[i].x, x[i].y, x[i].z, x[i].w}, ys[4] = {y[i].x, y[i].y, y[i].z, y[i].w};
    float a = 0.f;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      a = fmaf(__uint_as_float(xs[k] << 16), __uint_as_float(ys[k] << 16), a);
      a = fmaf(__uint_as_float(xs[k] & 0xffff0000u), __uint_as_float(ys[k] & 0xffff0000u), a);
    }
#pragma unroll
    for (int off = L / 2; off > 0; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
    const float inf = __int_as_float(0x7f800000);
    if (sub == 0 && t[i] < tokens)
      stats[(static_cast<int64_t>(kvh) * Tq + t[i]) * group + hg[i]] =
          make_float2(l[i] == -inf ? -inf : l[i] * -1.4426950408889634f, -a);
  }
}

// Adds up the sums of divided units in the parts' order, one warp per row.
template <int D, int MODE>
__global__ void __launch_bounds__(256) packed_attn_bwd_join_kernel(const PackedJoin* joins, const PackedBwdParams p) {
  constexpr int kWidth = MODE == kDkv ? 2 * D : D;
  grid_wait();
  grid_release();
  const PackedJoin jn = joins[blockIdx.x];
  const int kvh = blockIdx.y, lane = threadIdx.x & 31;
  const int rows = MODE == kDkv ? jn.n : jn.n * p.group;
  const int64_t step = static_cast<int64_t>(p.Hkv) * kTile * kWidth;
  for (int r = blockIdx.z * 8 + (threadIdx.x >> 5); r < rows; r += gridDim.z * 8) {
    const float* part = p.part + ((static_cast<int64_t>(jn.slot) * p.Hkv + kvh) * kTile + r) * kWidth;
    const int64_t token = jn.t0 + (MODE == kDkv ? r : r / p.group);
    const int head = MODE == kDkv ? kvh : kvh * p.group + r % p.group;
    constexpr int V = D / 32;                                  // channels a lane of each gradient
#pragma unroll
    for (int g = 0; g < kWidth / D; ++g) {
      float a[V];
#pragma unroll
      for (int c = 0; c < V; ++c) a[c] = 0.f;
#pragma unroll 8
      for (int k = 0; k < jn.parts; ++k) {
        const float* src = part + k * step + g * D + lane * V;
        float v[V];
        if constexpr (V == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
#pragma unroll
        for (int c = 0; c < V; ++c) a[c] += v[c];
      }
      if (lane * V >= p.d) continue;                           // (d is a multiple of 8)
      const bool is_dv = MODE == kDkv && g == 0;
      const float f = is_dv ? 1.f : p.scale;
      uint16_t* out = (is_dv ? static_cast<uint16_t*>(p.g2) + token * p.g2_t + head * p.g2_h
                             : static_cast<uint16_t*>(p.g1) + token * p.g1_t + head * p.g1_h) + lane * V;
      uint32_t w[V / 2];
#pragma unroll
      for (int c = 0; c < V / 2; ++c) w[c] = pack_bf16x2(a[2 * c] * f, a[2 * c + 1] * f);
      if constexpr (V == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(out) = w[0];
    }
  }
}

template <int D, int MODE>
int launch_join(const PackedBwdParams& p, const int32_t* joins, int n_join, cudaStream_t st) {
  if (n_join > 0)
    SWV_CUDA_OK(launch_after(packed_attn_bwd_join_kernel<D, MODE>, dim3(n_join, p.Hkv, 16), 256, 0, st,
                             reinterpret_cast<const PackedJoin*>(joins), p));
  return SWV_OK;
}
template <int D>
int launch_sides(const CUtensorMap& tq, const CUtensorMap& tg, const CUtensorMap& tk, const CUtensorMap& tv,
                 const PackedBwdParams& keys, const PackedBwdParams& queries, const PackedHeader& h, const int32_t* plan,
                 cudaStream_t st) {
  static std::atomic<uint64_t> prepared{0};
  constexpr size_t kSmem = std::max(bwd_smem<D, kDkv>(), bwd_smem<D, kDq>());
  int rc = prepare_kernel(packed_attn_bwd_kernel<D>, prepared, kBwdThreads, kBwdRegs, kSmem);
  if (rc != SWV_OK) return rc;
  SWV_CUDA_OK(launch_after(packed_attn_bwd_kernel<D>, static_cast<unsigned>(h.n_dkv + h.n_dq) * h.Hkv, kBwdThreads, kSmem, st, tq,
                           tg, tk, tv, keys, queries));
  rc = launch_join<D, kDkv>(keys, plan + h.dkv_join_off, h.n_dkv_join, st);
  if (rc == SWV_OK) rc = launch_join<D, kDq>(queries, plan + h.dq_join_off, h.n_dq_join, st);
  return rc;
}

struct BwdSizes {
  size_t stats, dq, dkv;
};
BwdSizes bwd_sizes(const PackedHeader& h, int64_t Tq, int D) {
  const size_t Dk = D <= 64 ? 64 : 128;
  BwdSizes s;
  s.stats = (static_cast<size_t>(h.H) * Tq * sizeof(float2) + 255) / 256 * 256;
  s.dq = static_cast<size_t>(h.dq_slots) * h.Hkv * kTile * Dk * sizeof(float);
  s.dkv = static_cast<size_t>(h.dkv_slots) * h.Hkv * kTile * 2 * Dk * sizeof(float);
  return s;
}

}  // namespace

int packed_attn_bwd_bytes_impl(const int32_t* plan_host, int64_t Tq, int D, size_t* bytes) {
  if (!plan_host || !bytes) return SWV_ERR_NULL;
  PackedHeader h;
  const int rc = packed_plan_header(plan_host, &h);
  if (rc != SWV_OK) return rc;
  if (Tq < h.Tq) return SWV_ERR_SHAPE;
  if (D < 8 || D % 8 != 0 || D > 128) return SWV_ERR_UNSUPPORTED;
  const BwdSizes s = bwd_sizes(h, Tq, D);
  *bytes = s.stats + s.dq + s.dkv;
  return SWV_OK;
}

int packed_attn_bwd_impl(const void* d_out, const int64_t* gs, const void* q, const int64_t* qs, const void* k,
                         const int64_t* ks, const void* v, const int64_t* vs, const void* o, const int64_t* os,
                         const float* lse, void* dq, const int64_t* dqs, void* dk, const int64_t* dks, void* dv,
                         const int64_t* dvs, const int32_t* plan_host, const int32_t* plan, int64_t Tq, int64_t Tk, int D,
                         float scale, void* workspace, size_t workspace_bytes, int* status, cudaStream_t st) {
  if (!plan_host || !gs || !qs || !ks || !vs || !os || !dqs || !dks || !dvs) return SWV_ERR_NULL;
  PackedHeader h;
  int rc = packed_plan_header(plan_host, &h);
  if (rc != SWV_OK) return rc;
  if (Tq < h.Tq || Tk < h.Tk || Tq > 0x7fffffff || Tk > 0x7fffffff) return SWV_ERR_SHAPE;
  if (!(scale >= kMinScale && scale <= 1.f / kMinScale)) return SWV_ERR_SHAPE;
  if (D < 8 || D % 8 != 0 || D > 128) return SWV_ERR_UNSUPPORTED;
  if (h.Tq == 0 && h.Tk == 0) return SWV_OK;
  if (!plan || !status) return SWV_ERR_NULL;
  if (h.Tq > 0 && (!d_out || !q || !o || !lse || !dq)) return SWV_ERR_NULL;
  if (h.Tk > 0 && (!k || !v || !dk || !dv)) return SWV_ERR_NULL;
  // one side empty: the maps need some memory, nothing reads it
  if (h.Tq == 0) { q = d_out = o = k; qs = gs = os = ks; Tq = 1; }
  if (h.Tk == 0) { k = v = q; ks = vs = qs; Tk = 1; }
  if (!packed_aligned(q, qs, 2) || !packed_aligned(k, ks, 2) || !packed_aligned(v, vs, 2) || !packed_aligned(o, os, 2) ||
      !packed_aligned(d_out, gs, 2))
    return SWV_ERR_ALIGN;
  if ((h.Tq > 0 && !packed_aligned(dq, dqs, 2)) ||
      (h.Tk > 0 && (!packed_aligned(dk, dks, 2) || !packed_aligned(dv, dvs, 2))))
    return SWV_ERR_ALIGN;
  if ((static_cast<int64_t>(h.n_dq) + h.n_dkv) * h.Hkv > 0x7fffffff || h.Hkv > 65535) return SWV_ERR_UNSUPPORTED;
  const BwdSizes sz = bwd_sizes(h, h.Tq == 0 ? 0 : Tq, D);
  if (!workspace && sz.stats + sz.dq + sz.dkv > 0) return SWV_ERR_NULL;
  if (workspace_bytes < sz.stats + sz.dq + sz.dkv) return SWV_ERR_WORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return SWV_ERR_ALIGN;

  PackedBwdParams p{};
  p.group = h.H / h.Hkv;
  p.group_inv = group_inverse(p.group);
  p.tok = kTile / p.group;
  p.Tq = static_cast<int>(Tq); p.d = D; p.Hkv = h.Hkv;
  p.scale = scale; p.scale_log2 = scale * 1.4426950408889634f;
  p.status = status;
  float2* stats = static_cast<float2*>(workspace);
  p.stats = stats;
  if (h.Tq > 0) {
    const int lanes = D <= 64 ? 8 : 16, per_cta = 256 / lanes * kDeltaRows;
    const int64_t ctas = (static_cast<int64_t>(h.Tq) * p.group + per_cta - 1) / per_cta;
    if (ctas > 0x7fffffff) return SWV_ERR_UNSUPPORTED;
    SWV_CUDA_OK(launch_after(lanes == 8 ? packed_attn_delta_kernel<8> : packed_attn_delta_kernel<16>,
                             dim3(static_cast<unsigned>(ctas), h.Hkv), 256, 0, st, static_cast<const __nv_bfloat16*>(o), os[0],
                             os[1], static_cast<const __nv_bfloat16*>(d_out), gs[0], gs[1], lse, stats, static_cast<int>(Tq),
                             h.Tq, p.group, D));
  }
  CUtensorMap tq, tg, tk, tv;
  if ((rc = packed_tmap(&tq, q, qs, Tq, h.Hkv, p.group, D, p.tok)) != SWV_OK) return rc;
  if ((rc = packed_tmap(&tg, d_out, gs, Tq, h.Hkv, p.group, D, p.tok)) != SWV_OK) return rc;
  if ((rc = packed_tmap(&tk, k, ks, Tk, h.Hkv, 0, D, kTile)) != SWV_OK) return rc;
  if ((rc = packed_tmap(&tv, v, vs, Tk, h.Hkv, 0, D, kTile)) != SWV_OK) return rc;
  uint8_t* w = static_cast<uint8_t*>(workspace) + sz.stats;

  PackedBwdParams a = p;                                       // keys' side
  a.units = reinterpret_cast<const PackedUnit*>(plan + h.dkv_off);
  a.n_units = h.n_dkv;
  a.heads_at_once = packed_heads_at_once(h.Hkv, static_cast<int64_t>(h.longest_q) * p.group, D);
  a.g1 = dk; a.g1_t = dks[0]; a.g1_h = dks[1];
  a.g2 = dv; a.g2_t = dvs[0]; a.g2_h = dvs[1];
  a.part = reinterpret_cast<float*>(w + sz.dq);
  PackedBwdParams b = p;                                       // queries' side
  b.units = reinterpret_cast<const PackedUnit*>(plan + h.dq_off);
  b.n_units = h.n_dq;
  b.heads_at_once = packed_heads_at_once(h.Hkv, h.longest_k, D);
  b.g1 = dq; b.g1_t = dqs[0]; b.g1_h = dqs[1];
  b.part = reinterpret_cast<float*>(w);
  return D <= 64 ? launch_sides<64>(tq, tg, tk, tv, a, b, h, plan, st) : launch_sides<128>(tq, tg, tk, tv, a, b, h, plan, st);
}

}  // namespace swv
