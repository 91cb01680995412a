// Work tables of the packed attention kernels: built on the host from the sequences' lengths, read by the kernels on
// the device.  One int32 array holds all of them; its first 32 words say where each one lies.
#pragma once
#include "common.cuh"

namespace swv {

constexpr int kPlanMagic = 0x53575031;
constexpr int kPlanHeader = 32;           // words

struct PackedHeader {                     // words 0..31 of a plan
  int magic, words;                       // size of the whole plan in 32-bit words
  int n_seq, H, Hkv, causal;
  int Tq, Tk;                             // tokens of all sequences
  int fwd_off, n_fwd;                     // units of the forward pass (PackedUnit)
  int dq_off, n_dq;                       // units of the backward pass, queries' side
  int dkv_off, n_dkv;                     // ..., keys' side
  int fwd_join_off, n_fwd_join, fwd_slots;    // units that were divided over the keys (PackedJoin) and their slots
  int dq_join_off, n_dq_join, dq_slots;
  int dkv_join_off, n_dkv_join, dkv_slots;
  int longest_q, longest_k;               // tokens of the longest sequence
  int reserved[7];
};
static_assert(sizeof(PackedHeader) == kPlanHeader * 4, "the header is 32 words");

// Forward and dq: `n` query tokens from packed token `t0` on, against blocks [b0, b1) of 128 keys of their sequence,
// whose keys start at packed key `s0` and are `len` in number.  Token i of the unit sees the keys j with
// j < min(len, off + i + 1).
// dkv: `n` keys from packed key `t0` on, against tiles [b0, b1) of 128 / group query tokens of their sequence, whose
// queries start at packed token `s0` and are `len` in number.  Key i of the unit is seen by the queries j with
// off + i <= j.
struct PackedUnit {
  int t0, n, s0, len, off, b0, b1;
  int slot;                               // where a divided unit leaves its sums; -1: it writes its rows itself
};
// Registers of the calling warpgroup (all four warps execute it); the block's shares add up to no more than its
// registers at launch.
template <int N>
__device__ __forceinline__ void reg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void reg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

struct PackedJoin {                       // the slots [slot, slot + parts) are sums of the rows t0 .. t0 + n - 1
  int t0, n, slot, parts;
};

// Which unit and key head a CTA serves.  The units of `at_once` heads go together, the longest units of all of them
// first: the launch ends with short ones, and what the CTAs in flight read stays in L2.
__device__ __forceinline__ PackedUnit packed_unit(const PackedUnit* units, int n_units, int heads, int at_once, int& head) {
  const int g = blockIdx.x / (n_units * at_once);
  const int r = blockIdx.x - g * n_units * at_once;
  const int here = min(at_once, heads - g * at_once);
  head = g * at_once + r % here;
  return units[r / here];
}
// Heads whose two streamed tensors (`rows` rows of the longest sequence) fill half of the L2.
inline int packed_heads_at_once(int heads, int64_t rows, int D) {
  const int64_t bytes = 4ll * D * (rows > 0 ? rows : 1);
  const int64_t n = (64ll << 20) / bytes;
  return static_cast<int>(n < 1 ? 1 : n > heads ? heads : n);
}

}  // namespace swv
