// Work tables of the packed attention kernels: built on the host from the sequences' lengths, read by the kernels on
// the device.  One int32 array holds all of them; its first 32 words say where each one lies.
#pragma once
#include <atomic>

#include "common.cuh"

namespace swv {

constexpr int kPlanMagic = 0x53575031;
constexpr float kMinScale = 8.673617379884035e-19f;       // 2^-60; lse / scale and scale x score stay in fp32's range
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

// Loads of what an earlier kernel of the stream may have written, behind grid_wait: from L2, and not moved ahead of the wait.
__device__ __forceinline__ float2 load_written(const float2* p) {
  float2 v;
  asm volatile("ld.global.cg.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ int4 load_written(const int4* p) {
  int4 v;
  asm volatile("ld.global.cg.v4.s32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}

// Which unit and key head CTA `block` serves.  The units of `at_once` heads go together, the longest units of all of them
// first: the launch ends with short ones, and what the CTAs in flight read stays in L2.
__device__ __forceinline__ PackedUnit packed_unit(const PackedUnit* units, int n_units, int heads, int at_once, int block,
                                                   int& head) {
  const int g = block / (n_units * at_once);
  const int r = block - g * n_units * at_once;
  const int here = min(at_once, heads - g * at_once);
  head = g * at_once + r % here;
  union { int4 v[2]; PackedUnit u; } x;
  const int4* src = reinterpret_cast<const int4*>(units + r / here);
  x.v[0] = load_written(src);
  x.v[1] = load_written(src + 1);
  return x.u;
}
// Heads whose two streamed tensors (`rows` rows of the longest sequence) fill half of the L2.
inline int packed_heads_at_once(int heads, int64_t rows, int D) {
  const int64_t bytes = 4ll * D * (rows > 0 ? rows : 1);
  const int64_t n = (64ll << 20) / bytes;
  return static_cast<int>(n < 1 ? 1 : n > heads ? heads : n);
}

// Rows of D 16-bit values gathered in shared memory before they are written: a thread holds a whole row of a TMEM tile, and
// 32 rows' stores of 16 bytes touch 32 lines each.  Chunks of 16 bytes change places with the row so that the threads'
// stores meet different banks.
template <int D>
__device__ __forceinline__ uint32_t staged_at(uint32_t base, int row, int chunk) {
  return base + row * (D * 2) + ((chunk ^ (row & 7)) << 4);
}
// N (16 or 32) fp32 values of a row, from column N * c on, times f, as bf16
template <int D, int N>
__device__ __forceinline__ void stage_columns(uint32_t base, int row, int c, const uint32_t* o, float f) {
#pragma unroll
  for (int i = 0; i < N / 8; ++i) {
    uint32_t w[4];
#pragma unroll
    for (int q = 0; q < 4; ++q)
      w[q] = pack_bf16x2(__uint_as_float(o[8 * i + 2 * q]) * f, __uint_as_float(o[8 * i + 2 * q + 1]) * f);
    sts128(staged_at<D>(base, row, N / 8 * c + i), w[0], w[1], w[2], w[3]);
  }
}
// Writes rows r0 .. r1 - 1 of the staged tile (one warp; `at(row)` is where a row goes), d <= D channels.
template <int D, typename At>
__device__ __forceinline__ void write_staged(uint32_t base, int r0, int r1, int d, At at) {
  constexpr int kLanes = D / 8;                                // lanes a row
  const int lane = threadIdx.x & 31, chunk = lane % kLanes;
#pragma unroll 4
  for (int r = r0 + lane / kLanes; r < r1; r += 32 / kLanes)
    if (chunk * 8 < d) *reinterpret_cast<uint4*>(at(r) + chunk * 8) = lds128(staged_at<D>(base, r, chunk));
}

// At the head of a rarely taken branch: without it the compiler turns the branch's selections into instructions that every
// pass executes (half of all, in the loops of the attention kernels).
#define KEEP_BRANCH() asm volatile("" ::: "memory")

// Row r < 128 of a tile as (token, head of the group): r / group by a multiplication (inverse = ceil(2^16 / group): the error
// r * (inverse * group - 2^16) < 128 * 128 never reaches the next quotient).
__device__ __forceinline__ int row_token(int r, int inverse) { return (r * inverse) >> 16; }
inline int group_inverse(int group) { return (65536 + group - 1) / group; }

// pairs of fp32 values in one instruction
__device__ __forceinline__ void fma2(float& x, float& y, float a, float b, float m, float c, float d) {
  asm("{\n\t.reg .b64 v, s, e;\n\tmov.b64 v, {%2, %3};\n\tmov.b64 s, {%4, %4};\n\tmov.b64 e, {%5, %6};\n\t"
      "fma.rn.f32x2 v, v, s, e;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "=f"(x), "=f"(y)
      : "f"(a), "f"(b), "f"(m), "f"(c), "f"(d));
}
__device__ __forceinline__ void add2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 v, s;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\tadd.rn.f32x2 v, v, s;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}
__device__ __forceinline__ void mul2(float& x, float& y, float a, float b) {
  asm("{\n\t.reg .b64 v, s;\n\tmov.b64 v, {%0, %1};\n\tmov.b64 s, {%2, %3};\n\tmul.rn.f32x2 v, v, s;\n\tmov.b64 {%0, %1}, v;\n\t}"
      : "+f"(x), "+f"(y)
      : "f"(a), "f"(b));
}

// Prepares a kernel on the current device, once: its shared memory, and whether it is launched with the registers that
// its warpgroups share out (an increase beyond them would wait for ever).
template <typename K>
int prepare_kernel(K kernel, std::atomic<uint64_t>& done, int threads, int shared_out, size_t smem) {
  int dev = 0;
  SWV_CUDA_OK(cudaGetDevice(&dev));
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_acquire) & bit)) return SWV_OK;
  cudaFuncAttributes a;
  SWV_CUDA_OK(cudaFuncGetAttributes(&a, kernel));
  if (a.numRegs * threads < shared_out) return SWV_ERR_CUDA;
  SWV_CUDA_OK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem)));
  if (dev < 64) done.fetch_or(bit, std::memory_order_release);
  return SWV_OK;
}

// The producer ends by waiting for its last copies (with the limit of one wait each): a CTA that gave up does not leave its
// shared memory to copies in flight; otherwise they have landed long since.
__device__ __forceinline__ void drain_copy(uint64_t* bar, uint32_t parity) {
  volatile uint32_t never = 0;
  (void)mbar_wait_bounded(bar, parity, &never);
}

}  // namespace swv
