// Layer norm over the last dimension of N rows of E values, forward and backward.
//
//   mu = mean(x)   rstd = 1 / sqrt(mean((x - mu)^2) + eps)   xh = (x - mu) rstd   y = xh w + b
//   g  = dy w      dx = rstd (g - mean(g) - xh mean(g xh))   dw = sum_rows dy xh  db = sum_rows dy
//
// A group of threads (one warp or more) owns a row: it is read once into registers, the variance is
// taken from the centred values (a second sum over the registers, so a large offset of the row costs no bits), and
// the result is written from the registers.  All sums are fp32.  The groups stay resident and walk over the rows, so
// the weights stay in shared memory and, in the backward pass, the sums of dw and db in registers; the next row is loaded
// before the present one is reduced, and a row is kept as it lies in memory (half the registers for 16-bit types).  Each CTA
// leaves its dw and db sums in the workspace and a second kernel adds them up in a fixed order: no atomics, the same bits every time.
//
// Bound: HBM, 2 N E elements forward, 3 N E backward.  65536 x 768 bf16: 37 and 56 us, 5.4 TB/s each (82 % of the copy rate);
// rows of 384 values reach 68 %: fewer bytes are in flight for a row's sums.
#include <algorithm>
#include <type_traits>

#include "elements.cuh"

namespace swv {
namespace {

constexpr int kLnThreads = 256;                              // forms of wide rows
constexpr int kLnMaxE = 1 << 29;                             // columns and their loops stay within 32 bits
// Threads of a CTA with runs of `run` values a thread and groups of `tpr` threads, and resident CTAs per SM.  Backward: three runs
// of 8 take 168 registers a thread, two take 128.
constexpr int ln_block(int tpr, int run, bool bwd) { return bwd && run == 24 && tpr <= 64 ? 384 : 256 / tpr * tpr; }
constexpr int ln_ctas(int tpr, int run, bool bwd, int es) {
  if (bwd) return run > 16 ? 1 : 2;
  return (run > 24 ? 2 : es == 4 ? 3 : 4) * 256 / ln_block(tpr, run, false);
}

struct LnParams {
  const void* x;
  const void* dy;
  const void* w;
  const void* b;
  void* y;                  // forward: y; backward: dx
  float *mean, *rstd;       // (N), optional in the forward pass
  float* part;              // backward: [grid][2][E] sums of dy xh and of dy, or null
  int64_t N, xs, dys, ys;   // rows and their distances in elements
  int E, w_dtype, b_dtype;
  float eps;
};

// Sums over the threads of a group: a warp, some warps of a CTA (named barrier 1 + the group) or the whole CTA.
template <int TPR, int NT, int K>
__device__ __forceinline__ void group_sum(float (&v)[K], float* smem, int& phase) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) {
#pragma unroll
    for (int k = 0; k < K; ++k) v[k] += __shfl_xor_sync(0xffffffffu, v[k], off);
  }
  if constexpr (TPR > 32) {
    constexpr int W = TPR / 32;
    const int grp = threadIdx.x / TPR, w = (threadIdx.x % TPR) >> 5;
    // two buffers in turn: a warp may be one reduction ahead of the others, never two
    float* buf = smem + ((phase & 1) * (NT / TPR) + grp) * (2 * W);
    ++phase;
    if ((threadIdx.x & 31) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) buf[k * W + w] = v[k];
    }
    if constexpr (TPR == NT) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + grp), "n"(TPR) : "memory");   // (a group's warps do the same rows)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v[k] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) v[k] += buf[k * W + i];
    }
  }
}

// The weights lie in shared memory as fp32, [w | b]; the columns behind E are zero.  A run of 8 is read as two halves, and the
// threads' first halves lie side by side, then their second ones: neighbours 32 bytes apart met in the same banks (forward,
// 65536 x 768: 40.7 us against 37.2).
template <int VEC, int TPR>
__device__ __forceinline__ int weight_at(int c) {
  if constexpr (VEC == 1) return c;
  else return ((c / (8 * TPR) * 2 + (c >> 2 & 1)) * TPR + (c >> 3) % TPR) * 4 + (c & 3);
}
template <int VEC, int ITER, int TPR, int NT>
__device__ __forceinline__ void stage_row(const void* a, int dtype, int E, float otherwise, float* out) {
  constexpr int C = VEC * ITER * TPR;
  if (a != nullptr && dtype == SWV_F32 && (reinterpret_cast<uintptr_t>(a) & 15) == 0) {
    constexpr int kRuns = (C + 4 * NT - 1) / (4 * NT);
    float4 v[kRuns];                                         // all loads in flight together
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = (i * NT + threadIdx.x) * 4;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      const float* f = static_cast<const float*>(a) + c;
      if (c + 3 < E) {
        v[i] = *reinterpret_cast<const float4*>(f);
      } else if (c < E) {
        v[i].x = f[0];
        if (c + 1 < E) v[i].y = f[1];
        if (c + 2 < E) v[i].z = f[2];
      }
    }
#pragma unroll
    for (int i = 0; i < kRuns; ++i) {
      const int c = (i * NT + threadIdx.x) * 4;
      if (c < C) *reinterpret_cast<float4*>(out + weight_at<VEC, TPR>(c)) = v[i];
    }
    return;
  }
  constexpr int kRuns = (C + NT - 1) / NT;
#pragma unroll 8
  for (int i = 0; i < kRuns; ++i) {
    const int c = i * NT + threadIdx.x;
    if (c < C) out[weight_at<VEC, TPR>(c)] = c >= E ? 0.f : a != nullptr ? load_as_f32(a, dtype, c) : otherwise;
  }
}
template <int VEC, int ITER, int TPR, int NT>
__device__ __forceinline__ void stage_weights(const LnParams& p, float* ws, bool bias) {
  constexpr int C = VEC * ITER * TPR;
  stage_row<VEC, ITER, TPR, NT>(p.w, p.w_dtype, p.E, 1.f, ws);
  if (bias) stage_row<VEC, ITER, TPR, NT>(p.b, p.b_dtype, p.E, 0.f, ws + C);
  __syncthreads();
}
// those of a thread's run i
template <int VEC, int TPR>
__device__ __forceinline__ void load_weights(const float* ws, int i, int t, float* v) {
  ws += weight_at<VEC, TPR>((i * TPR + t) * VEC);
  if constexpr (VEC == 8) {
    const float4 a = *reinterpret_cast<const float4*>(ws), b = *reinterpret_cast<const float4*>(ws + 4 * TPR);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    v[0] = *ws;
  }
}

template <typename T, typename U, int VEC, int ITER, int TPR>
__global__ void __launch_bounds__((ln_block(TPR, VEC * ITER, false)), (ln_ctas(TPR, VEC * ITER, false, sizeof(T))))
    layer_norm_fwd_kernel(const LnParams p) {
  constexpr int NT = ln_block(TPR, VEC * ITER, false);
  grid_wait();
  grid_release();
  __shared__ float red[4 * (NT / 32)];
  extern __shared__ float ws[];
  constexpr int C = VEC * ITER * TPR;
  int phase = 0;
  const int t = threadIdx.x % TPR;
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (NT / TPR);
  int64_t row = static_cast<int64_t>(blockIdx.x) * (NT / TPR) + threadIdx.x / TPR;
  const float inv_e = 1.f / p.E;
  Raw<T, VEC> next[ITER];
  auto fetch = [&](int64_t r) {
    const T* xr = static_cast<const T*>(p.x) + r * p.xs;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (r < p.N && c < p.E) next[i].load(xr + c);
      else next[i].zero();
    }
  };
  fetch(row);
  stage_weights<VEC, ITER, TPR, NT>(p, ws, true);
  for (; row < p.N; row += groups) {
    float v[ITER * VEC];
#pragma unroll
    for (int i = 0; i < ITER; ++i) next[i].values(v + i * VEC);
    fetch(row + groups);
    float s[1] = {0.f};
#pragma unroll
    for (int i = 0; i < ITER * VEC; ++i) s[0] += v[i];
    group_sum<TPR, NT>(s, red, phase);
    const float mu = s[0] * inv_e;
    s[0] = 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const bool in = (i * TPR + t) * VEC < p.E;             // (a run lies inside the row or outside it)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float d = in ? v[i * VEC + e] - mu : 0.f;
        v[i * VEC + e] = d;
        s[0] = fmaf(d, d, s[0]);
      }
    }
    group_sum<TPR, NT>(s, red, phase);
    const float rstd = 1.f / sqrtf(fmaf(s[0], inv_e, p.eps));
    U* yr = static_cast<U*>(p.y) + row * p.ys;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * TPR + t) * VEC;
      float w[VEC], b[VEC];
      load_weights<VEC, TPR>(ws, i, t, w);
      load_weights<VEC, TPR>(ws + C, i, t, b);
#pragma unroll
      for (int e = 0; e < VEC; ++e) w[e] = fmaf(v[i * VEC + e] * rstd, w[e], b[e]);
      if (c < p.E) store_run<U, VEC>(yr + c, w);
    }
    if (t == 0 && p.mean != nullptr) {
      p.mean[row] = mu;
      p.rstd[row] = rstd;
    }
  }
}

template <typename T, typename U, int VEC, int ITER, int TPR>
__global__ void __launch_bounds__((ln_block(TPR, VEC * ITER, true)), (ln_ctas(TPR, VEC * ITER, true, 0)))
    layer_norm_bwd_kernel(const LnParams p) {
  constexpr int NT = ln_block(TPR, VEC * ITER, true);
  grid_wait();
  grid_release();
  __shared__ float red[4 * (NT / 32)];
  extern __shared__ float ws[];
  constexpr int R = ITER * VEC, C = R * TPR;
  int phase = 0;
  const int t = threadIdx.x % TPR;
  const int64_t groups = static_cast<int64_t>(gridDim.x) * (NT / TPR);
  int64_t row = static_cast<int64_t>(blockIdx.x) * (NT / TPR) + threadIdx.x / TPR;
  const float inv_e = 1.f / p.E;
  float dw[R], db[R];
  constexpr bool kAhead = sizeof(T) + sizeof(U) <= 4;        // 16-bit rows: the next one is loaded under the present one's sums
  Raw<T, VEC> xn[ITER];
  Raw<U, VEC> gn[ITER];
#pragma unroll
  for (int i = 0; i < R; ++i) dw[i] = db[i] = 0.f;
  float mu_next, rstd_next;
  auto fetch = [&](int64_t r) {
    const T* xr = static_cast<const T*>(p.x) + r * p.xs;
    const U* dyr = static_cast<const U*>(p.dy) + r * p.dys;
    mu_next = r < p.N ? p.mean[r] : 0.f;
    rstd_next = r < p.N ? p.rstd[r] : 0.f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * TPR + t) * VEC;
      if (r < p.N && c < p.E) {
        xn[i].load(xr + c);
        gn[i].load(dyr + c);
      } else {
        xn[i].zero();
        gn[i].zero();
      }
    }
  };
  if (kAhead) fetch(row);
  stage_weights<VEC, ITER, TPR, NT>(p, ws, false);
  for (; row < p.N; row += groups) {
    if (!kAhead) fetch(row);
    const float mu = mu_next, rstd = rstd_next;
    Raw<T, VEC> x[ITER];
    Raw<U, VEC> g[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      x[i] = xn[i];
      g[i] = gn[i];
    }
    if (kAhead) fetch(row + groups);
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      float xv[VEC], gv[VEC], w[VEC];
      x[i].values(xv);
      g[i].values(gv);
      load_weights<VEC, TPR>(ws, i, t, w);       // (zero behind the row, and so is the gradient)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float xh = (xv[e] - mu) * rstd;
        dw[i * VEC + e] = fmaf(gv[e], xh, dw[i * VEC + e]);
        db[i * VEC + e] += gv[e];
        const float gw = gv[e] * w[e];
        s[0] += gw;
        s[1] = fmaf(gw, xh, s[1]);
      }
    }
    group_sum<TPR, NT>(s, red, phase);
    const float m0 = s[0] * inv_e, m1 = s[1] * inv_e;
    T* dxr = static_cast<T*>(p.y) + row * p.ys;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * TPR + t) * VEC;
      float xv[VEC], gv[VEC], w[VEC];
      x[i].values(xv);
      g[i].values(gv);
      load_weights<VEC, TPR>(ws, i, t, w);
#pragma unroll
      for (int e = 0; e < VEC; ++e) xv[e] = rstd * (gv[e] * w[e] - m0 - (xv[e] - mu) * rstd * m1);
      if (c < p.E) store_run<T, VEC>(dxr + c, xv);
    }
  }
  if (p.part == nullptr) return;
  float* out = p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.E;
  if constexpr (TPR == NT) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = (i / VEC * TPR + t) * VEC + i % VEC;
      if (c < p.E) {
        out[c] = dw[i];
        out[p.E + c] = db[i];
      }
    }
  } else {
    // the groups' sums side by side (the weights are no longer read), added up in the groups' order
    __syncthreads();
    float* mine = ws + threadIdx.x / TPR * 2 * C;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      const int c = (i / VEC * TPR + t) * VEC + i % VEC;
      mine[c] = dw[i];
      mine[C + c] = db[i];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * p.E; c += NT) {
      const float* col = ws + (c < p.E ? c : C + c - p.E);
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < NT / TPR; ++k) a += col[k * 2 * C];
      out[c] = a;
    }
  }
}

// Rows that do not fit the registers: one CTA per row, which it reads again for each of its sums (from L2).
template <typename T, typename U>
__global__ void __launch_bounds__(kLnThreads) layer_norm_wide_fwd_kernel(const LnParams p) {
  grid_wait();
  grid_release();
  __shared__ float red[4 * (kLnThreads / 32)];
  int phase = 0;
  const float inv_e = 1.f / p.E;
  for (int64_t row = blockIdx.x; row < p.N; row += gridDim.x) {
    const T* xr = static_cast<const T*>(p.x) + row * p.xs;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < p.E; c += kLnThreads) s[0] += to_f32(xr[c]);
    group_sum<kLnThreads, kLnThreads>(s, red, phase);
    const float mu = s[0] * inv_e;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < p.E; c += kLnThreads) {
      const float d = to_f32(xr[c]) - mu;
      s[0] = fmaf(d, d, s[0]);
    }
    group_sum<kLnThreads, kLnThreads>(s, red, phase);
    const float rstd = 1.f / sqrtf(fmaf(s[0], inv_e, p.eps));
    U* yr = static_cast<U*>(p.y) + row * p.ys;
    for (int c = threadIdx.x; c < p.E; c += kLnThreads) {
      const float w = p.w != nullptr ? load_as_f32(p.w, p.w_dtype, c) : 1.f;
      const float b = p.b != nullptr ? load_as_f32(p.b, p.b_dtype, c) : 0.f;
      yr[c] = from_f32<U>(fmaf((to_f32(xr[c]) - mu) * rstd, w, b));
    }
    if (threadIdx.x == 0 && p.mean != nullptr) {
      p.mean[row] = mu;
      p.rstd[row] = rstd;
    }
  }
}

// The same for the backward pass; a thread's columns are its own, so it adds dw and db into the CTA's row of the
// workspace without conflict.
template <typename T, typename U>
__global__ void __launch_bounds__(kLnThreads) layer_norm_wide_bwd_kernel(const LnParams p) {
  grid_wait();
  grid_release();
  __shared__ float red[4 * (kLnThreads / 32)];
  int phase = 0;
  const float inv_e = 1.f / p.E;
  float* part = p.part == nullptr ? nullptr : p.part + static_cast<int64_t>(blockIdx.x) * 2 * p.E;
  for (int64_t row = blockIdx.x; row < p.N; row += gridDim.x) {
    const bool first = row == blockIdx.x;
    const T* xr = static_cast<const T*>(p.x) + row * p.xs;
    const U* dyr = static_cast<const U*>(p.dy) + row * p.dys;
    const float mu = p.mean[row], rstd = p.rstd[row];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < p.E; c += kLnThreads) {
      const float xh = (to_f32(xr[c]) - mu) * rstd, d = to_f32(dyr[c]);
      const float g = d * (p.w != nullptr ? load_as_f32(p.w, p.w_dtype, c) : 1.f);
      s[0] += g;
      s[1] = fmaf(g, xh, s[1]);
      if (part != nullptr) {
        part[c] = fmaf(d, xh, first ? 0.f : part[c]);
        part[p.E + c] = (first ? 0.f : part[p.E + c]) + d;
      }
    }
    group_sum<kLnThreads, kLnThreads>(s, red, phase);
    const float m0 = s[0] * inv_e, m1 = s[1] * inv_e;
    T* dxr = static_cast<T*>(p.y) + row * p.ys;
    for (int c = threadIdx.x; c < p.E; c += kLnThreads) {
      const float xh = (to_f32(xr[c]) - mu) * rstd;
      const float g = to_f32(dyr[c]) * (p.w != nullptr ? load_as_f32(p.w, p.w_dtype, c) : 1.f);
      dxr[c] = from_f32<T>(rstd * (g - m0 - xh * m1));
    }
  }
}

// dw[c] = sum over the CTAs' rows of the workspace: 32 lanes of rows for 32 columns, added up in order
__global__ void __launch_bounds__(1024) layer_norm_sum_kernel(const float* part, int parts, int E, void* dw, int dw_dtype,
                                                              void* db, int db_dtype) {
  grid_wait();
  __shared__ float s[32][33];
  const int lane = threadIdx.x & 31, r = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;                   // column of [dw | db]
  float a = 0.f;
  if (c < 2 * E)
    for (int k = r; k < parts; k += 32) a += part[static_cast<int64_t>(k) * 2 * E + c];
  s[r][lane] = a;
  __syncthreads();
  // column `r` of the block: its 32 partial sums in the lanes of one warp
  a = s[lane][r];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) a += __shfl_xor_sync(0xffffffffu, a, off);
  const int col = blockIdx.x * 32 + r;
  if (lane == 0 && col < 2 * E) {
    if (col < E) {
      if (dw != nullptr) store_from_f32(dw, dw_dtype, col, a);
    } else if (db != nullptr) {
      store_from_f32(db, db_dtype, col - E, a);
    }
  }
}

// Which kernel serves a row: runs of 8 elements where every row starts on 16 bytes and E is a multiple of 8, single
// elements otherwise.  Runs of 8: few threads with several runs each, as many as the registers hold, so that few warps meet at a
// barrier and few lanes idle behind the row's end.  Forward, 16-bit rows: a warp up to 1280 values (32768 x 1280: 30 us, four
// warps 38, five 40), then two runs a thread (16384 x 2048: 25.5 us, one run 33); fp32 rows, twice the registers: one run a
// thread (4099 x 1280: 11.5 us, two runs 15.7; it loses where there are many rows: 19531 x 1280 52 us, three warps with two runs 35;
// 65104 x 384 46, a warp with two runs 35).  Backward: two runs (x, dy, dw and db of 16 values) in 128 registers, or
// three in 168 where they fit the row better (65536 x 768: 56 us, two warps with two runs 65; 32768 x 1280: 52 us, four warps 65);
// four runs take one CTA an SM instead of two (48828 x 1024: 61 us, two warps with two runs 57).  Beyond 8192 values the form that reads the row again.
// Both sides of the edges, 50 million bf16 values, us (the rule's form first).  Forward: 1280, a warp 35.3, 128 threads 43.6; 1288,
// 128 threads 44.7, two warps with three runs 37.6; 1536, 39.0 and 35.8; 2048, 128 threads with two runs 35.4, 256 with one 54.0; 2056,
// 256 with two 56.7, 128 with three 42.5.  Backward: 768, a warp 56.3, two with two runs 65.0; 776, two warps 66.0, one with four
// runs 66.8; 1536, two warps with three runs 57.6, 128 threads 65.3; 1544, 128 threads 67.2, two warps with four runs 67.1; 2048, 58.4 and
// 61.2; 2056, 256 threads 86.9, 128 with three runs 81.3.  So from 1288 to 1536 and behind 2048 another form would be 1.05 to 1.3
// times as fast.
struct LnForm {
  int vec, tpr, iter;       // iter = 0: the form for wide rows
};
constexpr LnForm ln_form(int E, bool vec8, bool bwd, bool wide) {
  LnForm f{};
  f.vec = vec8 ? 8 : 1;
  if (f.vec == 1) f.tpr = E <= 1024 ? 32 : E <= 4096 ? 128 : 256;
  else if (!bwd && wide) f.tpr = std::min((E + 255) / 256 * 32, 256);
  else f.tpr = E <= (bwd ? 768 : 1280) ? 32 : bwd && E <= 1536 ? 64 : E <= 2048 ? 128 : 256;
  const int n = (E + f.vec * f.tpr - 1) / (f.vec * f.tpr);
  if (f.vec == 8) f.iter = n <= (f.tpr == 32 ? 5 : 4) ? n : 0;
  else f.iter = n <= 8 ? 8 : n <= 32 ? 32 : 0;
  return f;
}

constexpr int kLnBwdCtas = 2;                     // the most of any backward form, also of the wide one
int ln_grid(const LnForm& f, int64_t N, bool bwd, int es) {
  const int run = f.vec * f.iter;
  int64_t rows = 1, per_sm = bwd ? kLnBwdCtas : 4;               // the form for wide rows
  if (f.iter > 0) {
    rows = ln_block(f.tpr, run, bwd) / f.tpr;
    per_sm = ln_ctas(f.tpr, run, bwd, es);
  }
  return static_cast<int>(std::min<int64_t>((N + rows - 1) / rows, sm_count() * per_sm));
}

template <typename T, typename U, int VEC, int ITER, int TPR, bool BWD>
auto ln_kernel() {
  if constexpr (BWD) return layer_norm_bwd_kernel<T, U, VEC, ITER, TPR>;
  else return layer_norm_fwd_kernel<T, U, VEC, ITER, TPR>;
}

// The forms that are compiled: (values a run, runs, threads a row, where: `bwd` or `one`, one run a thread at any width).
#define SWV_LN_FORMS(X, bwd, one)                                                                                         \
  X(8, 1, 32, true) X(8, 2, 32, !one) X(8, 3, 32, !one) X(8, 4, 32, !one && !bwd) X(8, 5, 32, !one && !bwd)                \
  X(8, 1, 64, one) X(8, 1, 96, one) X(8, 1, 128, one) X(8, 1, 160, one) X(8, 1, 192, one) X(8, 1, 224, one)                \
  X(8, 1, 256, one) X(8, 2, 64, bwd) X(8, 3, 64, bwd) X(8, 2, 128, !one) X(8, 2, 256, true) X(8, 3, 256, true)             \
  X(8, 4, 256, true) X(1, 8, 32, true) X(1, 32, 32, true) X(1, 32, 128, true) X(1, 32, 256, true)

// Every row that has a form finds it among them.
constexpr bool ln_compiled(const LnForm& f, bool bwd, bool one) {
#define SWV_LN(V, I, R, USED) \
  if (f.vec == V && f.iter == I && f.tpr == R) return USED;
  SWV_LN_FORMS(SWV_LN, bwd, one)
#undef SWV_LN
  return f.iter == 0;
}
constexpr bool ln_all_compiled(bool vec8, bool bwd, bool one) {
  for (int E = vec8 ? 8 : 1; E <= 9216; E += vec8 ? 8 : 1)
    if (!ln_compiled(ln_form(E, vec8, bwd, one), bwd, one)) return false;
  return true;
}
static_assert(ln_all_compiled(true, false, false) && ln_all_compiled(false, false, false), "a forward form is missing");
static_assert(ln_all_compiled(true, false, true) && ln_all_compiled(false, false, true), "a forward form of fp32 rows is missing");
static_assert(ln_all_compiled(true, true, false) && ln_all_compiled(false, true, false), "a backward form is missing");

template <typename T, typename U, bool BWD>
int ln_launch(const LnParams& p, const LnForm& f, int grid, cudaStream_t st) {
  constexpr bool kOne = !BWD && sizeof(T) == 4;
#define SWV_LN(V, I, R, USED)                                                                                \
  if (f.vec == V && f.iter == I && f.tpr == R) {                                                             \
    if constexpr (USED) {                                                                                    \
      constexpr int kBlock = ln_block(R, V * I, BWD), kSmem = 2 * V * I * (BWD ? kBlock : R) * 4;            \
      auto k = ln_kernel<T, U, V, I, R, BWD>();                                                              \
      if (kSmem > 40 * 1024) SWV_CUDA_OK(cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem)); \
      SWV_CUDA_OK(launch_after(k, grid, kBlock, kSmem, st, p));                                              \
      return SWV_OK;                                                                                         \
    }                                                                                                        \
    return SWV_ERR_UNSUPPORTED;                                                                              \
  }
  SWV_LN_FORMS(SWV_LN, BWD, kOne)
#undef SWV_LN
  if (f.iter != 0) return SWV_ERR_UNSUPPORTED;
  auto k = BWD ? layer_norm_wide_bwd_kernel<T, U> : layer_norm_wide_fwd_kernel<T, U>;
  SWV_CUDA_OK(launch_after(k, grid, kLnThreads, 0, st, p));
  return SWV_OK;
}

template <bool BWD>
int ln_dispatch(const LnParams& p, int x_dtype, int y_dtype, const LnForm& f, int grid, cudaStream_t st) {
  using bf = __nv_bfloat16;
  if (x_dtype == SWV_F32) {
    if (y_dtype == SWV_F32) return ln_launch<float, float, BWD>(p, f, grid, st);
    if (y_dtype == SWV_BF16) return ln_launch<float, bf, BWD>(p, f, grid, st);
    return ln_launch<float, __half, BWD>(p, f, grid, st);
  }
  if (x_dtype == SWV_BF16) {
    if (y_dtype == SWV_BF16) return ln_launch<bf, bf, BWD>(p, f, grid, st);
    return ln_launch<bf, float, BWD>(p, f, grid, st);
  }
  if (y_dtype == SWV_F16) return ln_launch<__half, __half, BWD>(p, f, grid, st);
  return ln_launch<__half, float, BWD>(p, f, grid, st);
}

int ln_check(int64_t N, int E, int x_dtype, int y_dtype, const void* w, int w_dtype, const void* b, int b_dtype) {
  if (N < 0 || E < 1) return SWV_ERR_SHAPE;
  if (E > kLnMaxE) return SWV_ERR_UNSUPPORTED;
  if (!dtype_known(x_dtype) || !dtype_known(y_dtype)) return SWV_ERR_DTYPE;
  if (x_dtype != SWV_F32 && y_dtype != x_dtype && y_dtype != SWV_F32) return SWV_ERR_DTYPE;
  if ((w != nullptr && !dtype_known(w_dtype)) || (b != nullptr && !dtype_known(b_dtype))) return SWV_ERR_DTYPE;
  return SWV_OK;
}

}  // namespace

int layer_norm_fwd_impl(const void* x, int64_t xs, int x_dtype, const void* w, int w_dtype, const void* b, int b_dtype,
                        void* y, int64_t ys, int y_dtype, float* mean, float* rstd, int64_t N, int E, float eps,
                        cudaStream_t st) {
  const int rc = ln_check(N, E, x_dtype, y_dtype, w, w_dtype, b, b_dtype);
  if (rc != SWV_OK) return rc;
  if (N == 0) return SWV_OK;
  if (!x || !y || (mean == nullptr) != (rstd == nullptr)) return SWV_ERR_NULL;
  const bool vec = E % 8 == 0 && rows_vec8(x, xs, dtype_bytes(x_dtype)) && rows_vec8(y, ys, dtype_bytes(y_dtype));
  const LnForm f = ln_form(E, vec, false, x_dtype == SWV_F32);
  LnParams p{};
  p.x = x; p.w = w; p.b = b; p.y = y; p.mean = mean; p.rstd = rstd;
  p.N = N; p.xs = xs; p.ys = ys; p.E = E; p.w_dtype = w_dtype; p.b_dtype = b_dtype; p.eps = eps;
  return ln_dispatch<false>(p, x_dtype, y_dtype, f, ln_grid(f, N, false, dtype_bytes(x_dtype)), st);
}

// The backward pass takes no more CTAs than this, whichever form serves it: room for their sums.
int layer_norm_bwd_bytes_impl(int64_t N, int E, size_t* bytes) {
  if (!bytes) return SWV_ERR_NULL;
  if (N < 0 || E < 1) return SWV_ERR_SHAPE;
  if (E > kLnMaxE) return SWV_ERR_UNSUPPORTED;
  *bytes = static_cast<size_t>(std::min<int64_t>(std::max<int64_t>(N, 1), static_cast<int64_t>(sm_count()) * kLnBwdCtas)) * 2 * E *
           sizeof(float);
  return SWV_OK;
}

int layer_norm_bwd_impl(const void* dy, int64_t dys, int y_dtype, const void* x, int64_t xs, int x_dtype, const void* w,
                        int w_dtype, const float* mean, const float* rstd, void* dx, int64_t dxs, void* dw, int dw_dtype,
                        void* db, int db_dtype, int64_t N, int E, void* workspace, size_t workspace_bytes,
                        cudaStream_t st) {
  const int rc = ln_check(N, E, x_dtype, y_dtype, w, w_dtype, nullptr, 0);
  if (rc != SWV_OK) return rc;
  if ((dw != nullptr && !dtype_known(dw_dtype)) || (db != nullptr && !dtype_known(db_dtype))) return SWV_ERR_DTYPE;
  if (N > 0 && (!dy || !x || !mean || !rstd || !dx)) return SWV_ERR_NULL;
  const bool sums = dw != nullptr || db != nullptr;
  const bool vec = E % 8 == 0 && rows_vec8(x, xs, dtype_bytes(x_dtype)) && rows_vec8(dy, dys, dtype_bytes(y_dtype)) &&
                   rows_vec8(dx, dxs, dtype_bytes(x_dtype));
  const LnForm f = ln_form(E, vec, true, false);
  const int grid = N == 0 ? 0 : ln_grid(f, N, true, 0);
  if (sums && N > 0) {
    size_t need = static_cast<size_t>(grid) * 2 * E * sizeof(float);
    if (!workspace) return SWV_ERR_NULL;
    if (workspace_bytes < need) return SWV_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 3) return SWV_ERR_ALIGN;
  }
  LnParams p{};
  p.x = x; p.dy = dy; p.w = w; p.y = dx;
  p.mean = const_cast<float*>(mean); p.rstd = const_cast<float*>(rstd);
  p.part = sums ? static_cast<float*>(workspace) : nullptr;
  p.N = N; p.xs = xs; p.dys = dys; p.ys = dxs; p.E = E; p.w_dtype = w_dtype;
  if (N > 0) {
    const int r = ln_dispatch<true>(p, x_dtype, y_dtype, f, grid, st);
    if (r != SWV_OK) return r;
  }
  if (sums) {                                             // (no rows: the sums are zero)
    SWV_CUDA_OK(launch_after(layer_norm_sum_kernel, (2 * E + 31) / 32, 1024, 0, st, p.part, grid, E, dw, dw_dtype, db, db_dtype));
  }
  return SWV_OK;
}

}  // namespace swv
