// Attention over packed sequences, forward: sequences of different lengths lie one behind the other, every query token
// sees the keys of its own sequence, all of them or (causal) those up to its own place counted from the end.
//
//   S = scale q k^T     m = max S     P = exp(S - m)     l = sum P     o = P v / l     lse = m + log l
//
// One pass over the keys with running m and l.  The query heads that share a key head are packed into the rows of a
// tile: row r of a tile is head r % group of token r / group, so a key tile is read once for the whole group and a
// single token of many heads still fills its rows.  A CTA owns two such tiles (A and B) of one key head:
//   warp 0      : TMA producer; Q of both tiles once, then K(j) and V(j) in turn through one ring
//   warps 1, 2  : one thread each issues the products of its tile, S = Q K(j)^T and then O += P V(j) with P read from
//                 TMEM; while one tile's softmax runs, the tensor cores work for the other
//   warp 3      : zeroes the value rows behind the sequence's end in its last tile (they belong to the next sequence
//                 or to nobody, and 0 x NaN would reach O)
//   warps 4..7 and 8..11 : softmax of tile A and of tile B, one thread per row: the row's 128 scores are read into registers,
//                 P is written as bf16 pairs, in two halves, so that P V starts under the second half's exponentials.
//                 P is rounded to bf16 because the product takes 16-bit operands (each entry is off by at most 2^-8);
//                 l sums the unrounded values.
//                 The stabiliser is raised (and O in TMEM rescaled) only when a row's maximum exceeds it by 2^8.
// The scores' slot is free as soon as they are in registers, so S = Q K(j+1)^T is formed while the exponentials of block j run
// (D = 128 has one slot for both tiles in turn); P has columns of its own.
// TMEM: D = 128: S [0,128), P_A, P_B [128,256), O_A [256,384), O_B [384,512)
//       D = 64:  S_A, S_B [0,256), P_A, P_B [256,384), O_A [384,448), O_B [448,512)
//
// Bound: the exponential unit (16 per clock and SM) at D = 64, it and the tensor pipe alike at D = 128; both are 63 % busy, by the
// chain scores -> maximum -> exponentials -> P V of two tiles.  16387 tokens in 5 sequences, 12 heads of 64: 437 us, 0.72 PFLOP/s;
// 15292 causal tokens in 4 sequences, 16 heads of 128 sharing two key heads: 316 us, 1.2 PFLOP/s (in runs of many calls the card's
// power limit makes it 360, 1.05 PFLOP/s).
#include <algorithm>
#include <cmath>
#include <cstring>

#include "packed.cuh"

namespace swv {
namespace {

struct PackedFwdParams {
  const PackedUnit* units;
  int n_units, group, group_inv, tok;      // tok = 128 / group query tokens a tile
  int Tq, d;                    // d <= D channels
  void* o;                      // bf16
  int64_t os_t, os_h;
  float* lse;                   // (H, Tq), natural logarithm
  float scale_log2;
  float* part_o;                // [slot][Hkv][256][D] unnormalised rows of divided units
  float2* part_ml;              // [slot][Hkv][256] (stabiliser, sum)
  int Hkv, heads_at_once;
  int* status;
};

constexpr int kFwdThreads = 384;
constexpr int kFwdRegsControl = 80, kFwdRegsSoftmax = 208;      // of 384 x 168 = 64512 at launch: 63488
constexpr int kFwdRegs = 128 * kFwdRegsControl + 256 * kFwdRegsSoftmax;

template <int D>
struct FwdCfg {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kStages = D == 128 ? 4 : 8;
  static constexpr int kOffRing = 2 * kTileBytes;
  // TMEM columns
  static constexpr int kSlots = D == 128 ? 1 : 2;             // score slots: one for both tiles in turn, or one each
  static constexpr uint32_t kColP = kSlots * 128;             // P of tile A, of tile B: 64 columns of bf16 pairs each
  static constexpr uint32_t kColO = kColP + 128;
  static constexpr int kOffCtl = kOffRing + kStages * kTileBytes;
};
struct FwdCtl {
  uint64_t q_full[2];
  uint64_t full[8], empty[8];
  uint64_t s_full[2], s_read[2], p_full[2][2], pv_done[2];
  uint64_t tail_full;                       // the last value block of the sequence, before it is cleaned
  uint32_t tmem_base, abort_flag;
};
template <int D>
constexpr size_t fwd_smem() { return 1024 + FwdCfg<D>::kOffCtl + sizeof(FwdCtl) + 64; }

__device__ __forceinline__ uint32_t first_bits(int n) { return n >= 32 ? 0xFFFFFFFFu : (n <= 0 ? 0u : (1u << n) - 1u); }

__device__ __forceinline__ float max_of3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

template <int D>
__global__ void __launch_bounds__(kFwdThreads, 1)
    packed_attn_fwd_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                           const __grid_constant__ CUtensorMap tm_v, const PackedFwdParams p) {
  using Cfg = FwdCfg<D>;
  constexpr int NST = Cfg::kStages;
  constexpr uint32_t kIdescQK = make_idesc(/*bf16*/ 1, kTile, kTile, 0, 0);
  constexpr uint32_t kIdescPV = make_idesc(/*bf16*/ 1, kTile, D, 0, /*V is MN-major*/ 1);
  constexpr float kStep = 8.0f;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  FwdCtl* ctl = reinterpret_cast<FwdCtl*>(smem + Cfg::kOffCtl);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {                            // (fetched while the barriers are made)
    tma_prefetch_desc(&tm_q);
    tma_prefetch_desc(&tm_k);
    tma_prefetch_desc(&tm_v);
  }
  if (threadIdx.x == 0) {
    for (int t = 0; t < 2; ++t) {
      mbar_init(&ctl->q_full[t], 1);
      mbar_init(&ctl->s_full[t], 1);
      mbar_init(&ctl->s_read[t], 4);
      mbar_init(&ctl->p_full[t][0], 4);
      mbar_init(&ctl->p_full[t][1], 4);
      mbar_init(&ctl->pv_done[t], 1);
    }
    for (int s = 0; s < NST; ++s) {
      mbar_init(&ctl->full[s], 1);
      mbar_init(&ctl->empty[s], 2);
    }
    mbar_init(&ctl->tail_full, 1);
    ctl->abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&ctl->tmem_base, 512);
    tmem_relinquish();
  }
  grid_wait();
  int kvh;
  const PackedUnit u = packed_unit(p.units, p.n_units, p.Hkv, p.heads_at_once, blockIdx.x, kvh);
  const int n = u.b1 - u.b0;
  // tokens and key blocks of tile t (its last token sees the most keys)
  auto tokens = [&](int t) { return min(p.tok, u.n - t * p.tok); };
  auto blocks = [&](int t) {
    const int tk = tokens(t);
    if (tk <= 0) return 0;
    const int sees = max(0, min(u.len, u.off + t * p.tok + tk));
    return min(n, max(0, (sees + kTile - 1) / kTile - u.b0));
  };
  const bool tail = n > 0 && u.b1 * kTile > u.len;   // the last block holds rows behind the sequence

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = ctl->tmem_base;
  volatile uint32_t* abort_flag = &ctl->abort_flag;
  grid_release();

  if (warp < 4) {
  reg_dec<kFwdRegsControl>();
  if (warp == 0) {
    // ------------------------------------------------------------ TMA producer
    if (lane == 0 && n > 0) {
      for (int t = 0; t < 2; ++t) {
        if (blocks(t) == 0) continue;                        // (its rows, zeros, may be staged there at once)
        mbar_expect_tx(&ctl->q_full[t], p.tok * p.group * D * 2);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_4d(smem + t * Cfg::kTileBytes + c * (kTile * 128), &tm_q, &ctl->q_full[t], c * 64, 0, u.t0 + t * p.tok, kvh);
      }
      int it = 0;
      for (; it < 2 * n; ++it) {
        const int s = it % NST;
        if (!mbar_wait_bounded(&ctl->empty[s], ((it / NST) & 1) ^ 1, abort_flag)) {
          record_status(p.status, kDevWaitStageEmpty);
          break;
        }
        // (the stage of the tail is declared full by the warp that cleans it)
        uint64_t* bar = tail && it == 2 * n - 1 ? &ctl->tail_full : &ctl->full[s];
        mbar_expect_tx(bar, Cfg::kTileBytes);
        const int key0 = u.s0 + (u.b0 + (it >> 1)) * kTile;
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          tma_load_3d(smem + Cfg::kOffRing + s * Cfg::kTileBytes + c * (kTile * 128), (it & 1) ? &tm_v : &tm_k, bar,
                      c * 64, key0, kvh);
      }
      for (int t = 0; t < 2; ++t)
        if (blocks(t) > 0) drain_copy(&ctl->q_full[t], 0);
      for (int i = max(0, it - NST); i < it; ++i) {
        const bool cut = tail && i == 2 * n - 1;
        drain_copy(cut ? &ctl->tail_full : &ctl->full[i % NST], cut ? 0 : (i / NST) & 1);
      }
    }
  } else if (warp <= 2) {
    // ---------------------------------------------- one MMA issuer for each tile
    const int t = warp - 1;
    const int nt = blocks(t), nother = blocks(1 - t);
    if (lane == 0 && n > 0) {
      const uint32_t q_addr = smem_u32(smem + t * Cfg::kTileBytes);
      const uint32_t ring = smem_u32(smem + Cfg::kOffRing);
      const uint32_t s_col = tmem_base + (t % Cfg::kSlots) * kTile, p_col = tmem_base + Cfg::kColP + t * 64;
      const uint32_t o_col = tmem_base + Cfg::kColO + t * D;
      bool ok = nt == 0 || mbar_wait_bounded(&ctl->q_full[t], 0, abort_flag);
      if (!ok) record_status(p.status, kDevWaitQ);
      auto landed = [&](int it) {
        if (mbar_wait_bounded(&ctl->full[it % NST], (it / NST) & 1, abort_flag)) return true;
        record_status(p.status, kDevWaitTmaFull);
        return false;
      };
      auto scores = [&](int j) {
        const int it = 2 * j, s = it % NST;
        if (!landed(it)) return false;
        // The slot's last scores have been read.  One slot: its users are A(0), B(0), A(1), ... until one tile has
        // no more blocks; two slots: the tile's own last block.
        const int before = Cfg::kSlots == 1 && j - 1 + t < nother ? j - 1 + t : j - 1;
        const int whose = Cfg::kSlots == 1 && j - 1 + t < nother ? 1 - t : t;
        if (before >= 0 && !mbar_wait_bounded(&ctl->s_read[whose], before & 1, abort_flag)) {
          record_status(p.status, kDevWaitAccEmpty);
          return false;
        }
        tc_fence_after();
        const uint64_t da = smem_desc_sw128(q_addr), db = smem_desc_sw128(ring + s * Cfg::kTileBytes);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint64_t off = (ks >> 2) * (kTile * 128 / 16) + (ks & 3) * 2;     // 64-channel halves are tiles of their own
          umma_f16_ss(s_col, da + off, db + off, kIdescQK, ks > 0);
        }
        umma_commit(&ctl->empty[s]);
        umma_commit(&ctl->s_full[t]);
        return true;
      };
      if (ok && nt > 0) ok = scores(0);
      for (int j = 0; ok && j < nt; ++j) {
        if (j + 1 < nt) ok = scores(j + 1);                  // a block ahead of P V
        if (!ok) break;
        const int it = 2 * j + 1, s = it % NST;
        if (!landed(it)) break;
        const uint64_t dv = smem_desc_sw128(ring + s * Cfg::kTileBytes, kTile * 128);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          if (ok && !mbar_wait_bounded(&ctl->p_full[t][half], j & 1, abort_flag)) {
            record_status(p.status, kDevWaitPReady);
            ok = false;
          }
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int ks = half * 4; ks < half * 4 + 4; ++ks)
            umma_f16_ts(o_col, p_col + ks * 8, dv + ks * 128, kIdescPV, (j > 0 || ks > 0));
        }
        if (!ok) break;
        umma_commit(&ctl->empty[s]);
        umma_commit(&ctl->pv_done[t]);
      }
      // blocks that only the other tile needs (a stage is given back in the phase in which it was filled)
      for (int it = 2 * nt; ok && it < 2 * n; ++it) {
        ok = landed(it);
        if (ok) mbar_arrive(&ctl->empty[it % NST]);
      }
    }
  } else {
    if (tail) {
      const int s = (2 * n - 1) % NST;
      bool ok = mbar_wait_bounded(&ctl->tail_full, 0, abort_flag);
      if (!ok) record_status(p.status, kDevWaitTmaFull);
      if (__all_sync(0xffffffffu, ok)) {
        const int first = u.len - (u.b1 - 1) * kTile;
        const uint32_t base = smem_u32(smem + Cfg::kOffRing + s * Cfg::kTileBytes);
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          for (int i = first * 8 + lane; i < kTile * 8; i += 32) sts128(base + c * (kTile * 128) + i * 16, 0u, 0u, 0u, 0u);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ctl->full[s]);
      }
    }
  }
  } else {
    // ----------------------------------------------------------------- softmax
    reg_inc<kFwdRegsSoftmax>();
    const int t = (warp - 4) >> 2;
    const int nt = blocks(t);
    const int quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const int rows = tokens(t) * p.group;
    const bool live = quarter * 32 < rows;
    const bool row_ok = row < rows;
    const int tk = row_token(row, p.group_inv);                            // token of the tile
    const int limit = row_ok ? min(u.len, u.off + t * p.tok + tk + 1) - u.b0 * kTile : 0;   // keys it sees from block b0 on
    const uint32_t lane_off = static_cast<uint32_t>(quarter * 32) << 16;
    const uint32_t s_col = tmem_base + lane_off + (t % Cfg::kSlots) * kTile;
    const uint32_t p_col = tmem_base + lane_off + Cfg::kColP + t * 64;
    const uint32_t o_col = tmem_base + lane_off + Cfg::kColO + t * D;
    const float sc = p.scale_log2;
    const float ninf = -__int_as_float(0x7f800000), nan = __int_as_float(0x7fc00000);
    float m_used = ninf;
    float l = 0.f;
    bool ok = true;
    for (int j = 0; j < nt; ++j) {
      if (!mbar_wait_bounded(&ctl->s_full[t], j & 1, abort_flag)) {
        record_status(p.status, kDevWaitAccFull);
        ok = false;
      }
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      uint32_t s[kTile];
      if (live) {
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(s_col + c * 32, *reinterpret_cast<uint32_t(*)[32]>(s + c * 32));
        tc_wait_ld();
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&ctl->s_read[t]);
      // P V(j-1) has retired: P's columns are free, O may be rescaled
      auto retired = [&]() {
        bool r = j == 0 || mbar_wait_bounded(&ctl->pv_done[t], (j - 1) & 1, abort_flag);
        if (!r) record_status(p.status, kDevWaitPvDone);
        r = __all_sync(0xffffffffu, r);
        tc_fence_after();
        return r;
      };
      if (live) {
        const int vis = limit - j * kTile;                   // the first `vis` columns are seen
        if (__any_sync(0xffffffffu, vis < kTile)) {
          KEEP_BRANCH();
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const uint32_t w = first_bits(vis - c * 32);
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (!((w >> i) & 1u)) s[c * 32 + i] = __float_as_uint(ninf);
          }
        }
        float m0 = ninf, m1 = ninf, m2 = ninf, m3 = ninf;
#pragma unroll
        for (int i = 0; i < kTile; i += 8) {
          m0 = max_of3(m0, __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
          m1 = max_of3(m1, __uint_as_float(s[i + 2]), __uint_as_float(s[i + 3]));
          m2 = max_of3(m2, __uint_as_float(s[i + 4]), __uint_as_float(s[i + 5]));
          m3 = max_of3(m3, __uint_as_float(s[i + 6]), __uint_as_float(s[i + 7]));
        }
        const float m_new = fmaxf(m_used, fmaxf(max_of3(m0, m1, m2), m3) * sc);
        ok = retired();
        if (!ok) break;
        if (__any_sync(0xffffffffu, m_new > m_used + kStep)) {
          const float factor = (m_new == m_used) ? 1.f : ex2_approx(m_used - m_new);
          l *= factor;
          m_used = m_new;
          if (j > 0) {
#pragma unroll 1
            for (int c = 0; c < D / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(o_col + c * 16, o);
              tc_wait_ld();
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * factor);
              tmem_st16(o_col + c * 16, o);
            }
          }
        }
        // Scores of -inf have probability zero, also where the row has met nothing else yet (-inf + inf would be NaN).
        const float neg_m = m_used == ninf ? 0.f : -m_used;
        float l0 = 0.f, l1 = 0.f;
#pragma unroll
        for (int v = 0; v < 8; ++v) {
          uint32_t packed[8];
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            float x0, x1;
            fma2(x0, x1, __uint_as_float(s[v * 16 + i]), __uint_as_float(s[v * 16 + i + 1]), sc, neg_m, neg_m);
            x0 = ex2_approx(x0);
            x1 = ex2_approx(x1);
            add2(l0, l1, x0, x1);
            packed[i >> 1] = pack_bf16x2(x0, x1);
          }
          tmem_st8(p_col + v * 8, packed);
          if (v == 4 || v == 7) {          // the first half is handed over under the next 16 columns' exponentials
            tc_wait_st();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ctl->p_full[t][v == 7]);
          }
        }
        l += l0 + l1;
      } else {
        ok = retired();                                      // (not ahead of the others' P of block j - 1)
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive(&ctl->p_full[t][0]);
          mbar_arrive(&ctl->p_full[t][1]);
        }
      }
    }
    if (nt > 0 && ok && !mbar_wait_bounded(&ctl->pv_done[t], (nt - 1) & 1, abort_flag)) {
      record_status(p.status, kDevWaitPvDone);
      ok = false;
    }
    ok = __all_sync(0xffffffffu, ok);
    tc_fence_after();
    if (ok && live) {
      const int head = kvh * p.group + row - tk * p.group;
      const int64_t token = u.t0 + t * p.tok + tk;
      if (u.slot >= 0) {
        const int64_t r = (static_cast<int64_t>(u.slot) * p.Hkv + kvh) * (2 * kTile) + t * kTile + row;
        if (row_ok) p.part_ml[r] = make_float2(m_used, l);
#pragma unroll 1
        for (int c = 0; c < D / 16; ++c) {
          uint32_t o[16];
          if (nt > 0) {
            tmem_ld16(o_col + c * 16, o);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) o[i] = 0u;
          }
          if (!row_ok) continue;
#pragma unroll
          for (int i = 0; i < 16; i += 4)
            *reinterpret_cast<uint4*>(p.part_o + r * D + c * 16 + i) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
        }
      } else {
        // A row that sees no key is zero (lse -inf), one whose scores are all -inf is NaN, as 0 / 0 (an undivided unit
        // starts at its sequence's first key, so `limit` counts all that the row sees).
        const bool none = limit <= 0;
        const float inv = none ? 0.f : l == 0.f ? nan : 1.f / l;
        if (row_ok && p.lse != nullptr)
          p.lse[static_cast<int64_t>(head) * p.Tq + token] =
              none ? ninf : l == 0.f ? nan : (m_used + log2f(l)) * 0.6931471805599453f;
        // (the tile's Q is no longer needed: its last scores are done)
        const uint32_t stage = smem_u32(smem + t * Cfg::kTileBytes);
#pragma unroll 1
        for (int c = 0; c < D / 32; ++c) {
          uint32_t o[32];
          if (nt > 0) {
            tmem_ld32(o_col + c * 32, o);
            tc_wait_ld();
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0u;
          }
          if (__any_sync(0xffffffffu, none)) {                 // (also where 0 x v is NaN)
            KEEP_BRANCH();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = none ? 0u : o[i];
          }
          stage_columns<D, 32>(stage, row, c, o, inv);
        }
        __syncwarp();
        uint16_t* out = static_cast<uint16_t*>(p.o) + static_cast<int64_t>(u.t0 + t * p.tok) * p.os_t +
                        static_cast<int64_t>(kvh) * p.group * p.os_h;
        write_staged<D>(stage, quarter * 32, min(rows, quarter * 32 + 32), p.d,
                        [&](int r) {
                          const int w = row_token(r, p.group_inv);
                          return out + w * p.os_t + (r - w * p.group) * p.os_h;
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

// Joins the sums of divided units, one warp per row: o = sum_i 2^(m_i - m) O_i / sum_i 2^(m_i - m) l_i.  The parts'
// (m, l) lie in the lanes, 32 parts at a time, their rows are added up in the parts' order with eight loads in flight.
// Every row of a divided unit sees a key (the unit has more than two blocks, its 256 tokens at most follow each other), so one without
// any weight has scores of -inf alone: NaN.
template <int D>
__global__ void __launch_bounds__(256) packed_attn_join_kernel(const PackedJoin* joins, const PackedFwdParams p) {
  constexpr int V = D / 32;                                    // channels a lane
  grid_wait();
  const PackedJoin jn = joins[blockIdx.x];
  const int kvh = blockIdx.y, lane = threadIdx.x & 31;
  const float ninf = -__int_as_float(0x7f800000);
  const int rows = jn.n * p.group;                             // rows of both tiles, tile B's from row tok * group on
  const int64_t step = static_cast<int64_t>(p.Hkv) * (2 * kTile);
  for (int i = blockIdx.z * 8 + (threadIdx.x >> 5); i < rows; i += gridDim.z * 8) {
    const int per = p.tok * p.group;
    const int64_t r0 = (static_cast<int64_t>(jn.slot) * p.Hkv + kvh) * (2 * kTile) + (i / per) * kTile + i % per;
    float m = ninf;
    for (int k = lane; k < jn.parts; k += 32) m = fmaxf(m, p.part_ml[r0 + k * step].x);
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
    float l = 0.f, acc[V];
#pragma unroll
    for (int c = 0; c < V; ++c) acc[c] = 0.f;
    for (int k0 = 0; k0 < jn.parts; k0 += 32) {
      float f = 0.f;
      if (k0 + lane < jn.parts) {
        const float2 ml = p.part_ml[r0 + (k0 + lane) * step];
        f = ml.x == m ? 1.f : ex2_approx(ml.x - m);
        l = fmaf(ml.y, f, l);
      }
      const int here = min(32, jn.parts - k0);
#pragma unroll 8
      for (int k = 0; k < here; ++k) {
        const float fk = __shfl_sync(0xffffffffu, f, k);
        const float* src = p.part_o + (r0 + (k0 + k) * step) * D + lane * V;
        float v[V];
        if constexpr (V == 4) *reinterpret_cast<float4*>(v) = *reinterpret_cast<const float4*>(src);
        else *reinterpret_cast<float2*>(v) = *reinterpret_cast<const float2*>(src);
#pragma unroll
        for (int c = 0; c < V; ++c) acc[c] = fmaf(v[c], fk, acc[c]);
      }
    }
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) l += __shfl_xor_sync(0xffffffffu, l, off);
    const int head = kvh * p.group + i % p.group;
    const int64_t token = jn.t0 + i / p.group;
    const float inv = l == 0.f ? __int_as_float(0x7fc00000) : 1.f / l;
    if (lane == 0 && p.lse != nullptr)
      p.lse[static_cast<int64_t>(head) * p.Tq + token] = l == 0.f ? inv : (m + log2f(l)) * 0.6931471805599453f;
    if (lane * V >= p.d) continue;                             // (d is a multiple of 8)
    uint32_t w[V / 2];
#pragma unroll
    for (int c = 0; c < V / 2; ++c) w[c] = pack_bf16x2(acc[2 * c] * inv, acc[2 * c + 1] * inv);
    uint16_t* out = static_cast<uint16_t*>(p.o) + token * p.os_t + head * p.os_h + lane * V;
    if constexpr (V == 4) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(out) = w[0];
  }
}

template <int D>
int launch_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const PackedFwdParams& p,
               const PackedHeader& h, const int32_t* plan, cudaStream_t st) {
  static std::atomic<uint64_t> prepared{0};
  const int rc = prepare_kernel(packed_attn_fwd_kernel<D>, prepared, kFwdThreads, kFwdRegs, fwd_smem<D>());
  if (rc != SWV_OK) return rc;
  SWV_CUDA_OK(launch_after(packed_attn_fwd_kernel<D>, static_cast<unsigned>(p.n_units) * p.Hkv, kFwdThreads, fwd_smem<D>(), st,
                           tq, tk, tv, p));
  if (h.n_fwd_join > 0) {
    // a row a warp where there are few rows; at most 16 CTAs a unit
    const int rows = std::min(2 * p.tok, p.Tq) * p.group;
    const dim3 grid(h.n_fwd_join, p.Hkv, std::min(16, (rows + 7) / 8));
    SWV_CUDA_OK(launch_after(packed_attn_join_kernel<D>, grid, 256, 0, st,
                             reinterpret_cast<const PackedJoin*>(plan + h.fwd_join_off), p));
  }
  return SWV_OK;
}

}  // namespace

bool packed_aligned(const void* p, const int64_t* s, int es) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && s[2] == 1 && (s[0] * es) % 16 == 0 && (s[1] * es) % 16 == 0;
}

// Tensor maps of token-major tensors (tokens, heads, d).  Rows packed from `group` heads of `tok` tokens: the box's
// heads run fastest, then its tokens.
int packed_tmap(CUtensorMap* out, const void* base, const int64_t* s, int64_t tokens, int heads_kv, int group, int d,
                int box_tok) {
  EncodeTiledFn enc = get_encode_tiled();
  if (enc == nullptr) return SWV_ERR_CUDA;
  const cuuint64_t b = 2;
  CUresult r;
  if (group > 0) {
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(group), static_cast<cuuint64_t>(tokens),
                          static_cast<cuuint64_t>(heads_kv)};
    cuuint64_t strides[3] = {s[1] * b, s[0] * b, s[1] * b * group};
    cuuint32_t box[4] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(box_tok), 1}, es[4] = {1, 1, 1, 1};
    r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  } else {
    cuuint64_t dims[3] = {static_cast<cuuint64_t>(d), static_cast<cuuint64_t>(tokens), static_cast<cuuint64_t>(heads_kv)};
    cuuint64_t strides[2] = {s[0] * b, s[1] * b};
    cuuint32_t box[3] = {64, static_cast<cuuint32_t>(box_tok), 1}, es[3] = {1, 1, 1};
    r = enc(out, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, es,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  }
  return r == CUDA_SUCCESS ? SWV_OK : SWV_ERR_TENSORMAP;
}

int packed_plan_header(const int32_t* plan_host, PackedHeader* h) {
  memcpy(h, plan_host, sizeof(*h));
  return h->magic == kPlanMagic ? SWV_OK : SWV_ERR_SHAPE;
}

int packed_attn_bytes_impl(const int32_t* plan_host, int D, size_t* bytes) {
  if (!plan_host || !bytes) return SWV_ERR_NULL;
  PackedHeader h;
  const int rc = packed_plan_header(plan_host, &h);
  if (rc != SWV_OK) return rc;
  if (D < 8 || D % 8 != 0 || D > 128) return SWV_ERR_UNSUPPORTED;
  const size_t rows = static_cast<size_t>(h.fwd_slots) * h.Hkv * 2 * kTile;
  *bytes = rows * (D <= 64 ? 64 : 128) * sizeof(float) + rows * sizeof(float2);
  return SWV_OK;
}

int packed_attn_fwd_impl(const void* q, const int64_t* qs, const void* k, const int64_t* ks, const void* v,
                         const int64_t* vs, void* o, const int64_t* os, float* lse, const int32_t* plan_host,
                         const int32_t* plan, int64_t Tq, int64_t Tk, int D, float scale, void* workspace,
                         size_t workspace_bytes, int* status, cudaStream_t st) {
  if (!plan_host || !qs || !ks || !vs || !os) return SWV_ERR_NULL;
  PackedHeader h;
  int rc = packed_plan_header(plan_host, &h);
  if (rc != SWV_OK) return rc;
  if (Tq < h.Tq || Tk < h.Tk || Tq > 0x7fffffff || Tk > 0x7fffffff) return SWV_ERR_SHAPE;
  if (!(scale >= kMinScale && scale <= 1.f / kMinScale)) return SWV_ERR_SHAPE;
  if (D < 8 || D % 8 != 0 || D > 128) return SWV_ERR_UNSUPPORTED;
  if (h.n_fwd == 0) return SWV_OK;                           // no query
  if (!q || !o || !plan || !status) return SWV_ERR_NULL;
  if (h.Tk > 0 && (!k || !v)) return SWV_ERR_NULL;
  if (h.Tk == 0) {                                           // no key at all: the maps need some memory, nothing reads it
    k = v = q;
    ks = vs = qs;
    Tk = 1;
  }
  if (!packed_aligned(q, qs, 2) || !packed_aligned(k, ks, 2) || !packed_aligned(v, vs, 2) || !packed_aligned(o, os, 2))
    return SWV_ERR_ALIGN;
  if (static_cast<int64_t>(h.n_fwd) * h.Hkv > 0x7fffffff || h.Hkv > 65535) return SWV_ERR_UNSUPPORTED;
  size_t need = 0;
  packed_attn_bytes_impl(plan_host, D, &need);
  if (need > 0) {
    if (!workspace) return SWV_ERR_NULL;
    if (workspace_bytes < need) return SWV_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return SWV_ERR_ALIGN;
  }
  PackedFwdParams p{};
  p.group = h.H / h.Hkv;
  p.group_inv = group_inverse(p.group);
  p.tok = kTile / p.group;
  p.units = reinterpret_cast<const PackedUnit*>(plan + h.fwd_off);
  p.n_units = h.n_fwd;
  p.Tq = static_cast<int>(Tq); p.d = D; p.o = o; p.os_t = os[0]; p.os_h = os[1]; p.lse = lse;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.Hkv = h.Hkv; p.status = status;
  p.heads_at_once = packed_heads_at_once(h.Hkv, h.longest_k, D);
  const int Dk = D <= 64 ? 64 : 128;
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = reinterpret_cast<float2*>(p.part_o + static_cast<size_t>(h.fwd_slots) * h.Hkv * 2 * kTile * Dk);
  CUtensorMap tq, tk, tv;
  if ((rc = packed_tmap(&tq, q, qs, Tq, h.Hkv, p.group, D, p.tok)) != SWV_OK) return rc;
  if ((rc = packed_tmap(&tk, k, ks, Tk, h.Hkv, 0, D, kTile)) != SWV_OK) return rc;
  if ((rc = packed_tmap(&tv, v, vs, Tk, h.Hkv, 0, D, kTile)) != SWV_OK) return rc;
  return Dk == 64 ? launch_fwd<64>(tq, tk, tv, p, h, plan, st) : launch_fwd<128>(tq, tk, tv, p, h, plan, st);
}

}  // namespace swv
