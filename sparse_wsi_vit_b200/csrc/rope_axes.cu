// Rotary positions with several axes (for example level, row and column): every rotated pair of channels (a, b) of a
// token turns by angle = position[axis of the pair] * frequency of the pair,
//   (a, b) -> (a cos - b sin, b cos + a sin),      and by -angle for the gradient (the rotation is orthogonal).
// The pairs are neighbouring channels (2i, 2i + 1) or channels (i, R + i) of the R rotated pairs; the channels behind
// 2 R are copied.
//
// Far positions: the product of a position and a frequency is taken in 64 bits and in turns (the frequencies are
// stored divided by 2 pi), its whole turns are dropped there, and only the rest goes to the 32-bit sine and cosine; in 32
// bits a coordinate of 10^5 would leave an error of 4e-3 in the angle.  One such angle serves a pair of all heads.
//
// A thread owns 8 channels of a token (4 or 8 pairs) and walks over heads; where the tokens are few, the heads are divided
// over the grid.  Bound: HBM, every element read and written once (24576 tokens, 24 heads of 64 bf16: 30 us in a run of launches on
// different buffers, 5.0 TB/s; 27 where one pair of buffers stays in part in L2; 24.6 for a launch by itself, whose last writes
// are still in L2 at its end).
#include <algorithm>
#include <type_traits>

#include "elements.cuh"

namespace swv {
namespace {

constexpr int kMaxPairs = 128, kMaxAxes = 8;

struct RopeAxesParams {
  const void* x;
  void* y;
  const void* pos;          // (T, axes), rows `pos_stride` elements apart
  int64_t T, xs_t, xs_h, ys_t, ys_h, pos_stride;
  int H, hd, pairs, heads_per_cta, pos_dtype;
  float sign;
  double turns[kMaxPairs];  // frequency / (2 pi)
  uint8_t axis[kMaxPairs];
};

__device__ __forceinline__ double rope_position(const RopeAxesParams& p, int64_t t, int axis) {
  const int64_t i = t * p.pos_stride + axis;
  if (p.pos_dtype == SWV_POS_F32) return static_cast<const float*>(p.pos)[i];
  if (p.pos_dtype == SWV_POS_I32) return static_cast<const int32_t*>(p.pos)[i];
  return static_cast<double>(static_cast<const int64_t*>(p.pos)[i]);
}
__device__ __forceinline__ void rope_angle(const RopeAxesParams& p, int64_t t, int pair, float& cs, float& sn) {
  const double a = rope_position(p, t, p.axis[pair]) * p.turns[pair];
  const float r = static_cast<float>(a - rint(a));
  sincospif(2.f * r, &sn, &cs);
  sn *= p.sign;
}

// VEC = 8: 16-byte aligned rows, hd a multiple of 8 and (halves) the number of pairs too; VEC = 1: any layout.
template <typename T, int VEC, bool HALVES>
__global__ void __launch_bounds__(256) rope_axes_kernel(const __grid_constant__ RopeAxesParams p) {
  grid_wait();
  grid_release();
  // units of a token: (halves) VEC pairs a unit, then the channels that are copied; (adjacent) max(VEC / 2, 1) pairs a unit
  constexpr int PAIRS = HALVES ? VEC : (VEC == 8 ? 4 : 1);
  const int turning = (p.pairs + PAIRS - 1) / PAIRS;
  const int copied = p.hd - 2 * p.pairs;
  const int still = HALVES || VEC == 1 ? (copied + VEC - 1) / VEC : (p.hd + 7) / 8 - turning;
  const int units = turning + still;
  const int64_t gid = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
  const int64_t t = gid / units;
  if (t >= p.T) return;
  const int u = static_cast<int>(gid - t * units);
  const int h0 = blockIdx.y * p.heads_per_cta, h1 = min(p.H, h0 + p.heads_per_cta);
  const T* x = static_cast<const T*>(p.x) + t * p.xs_t;
  T* y = static_cast<T*>(p.y) + t * p.ys_t;

  if (u >= turning) {
    const int c = (HALVES || VEC == 1) ? 2 * p.pairs + (u - turning) * VEC : u * 8;
    for (int h = h0; h < h1; ++h) {
      float v[VEC];
      load_run<T, VEC>(x + h * p.xs_h + c, v);
      store_run<T, VEC>(y + h * p.ys_h + c, v);
    }
    return;
  }
  float cs[PAIRS], sn[PAIRS];
#pragma unroll
  for (int i = 0; i < PAIRS; ++i) {
    const int pair = u * PAIRS + i;
    cs[i] = 1.f;
    sn[i] = 0.f;
    if (pair < p.pairs) rope_angle(p, t, pair, cs[i], sn[i]);      // (a unit can reach into the copied channels)
  }
  const int ca = HALVES ? u * PAIRS : 2 * u * PAIRS, cb = ca + p.pairs;
  constexpr int RUN = HALVES ? VEC : 2 * PAIRS;                    // elements of one access (8 or 1; adjacent pairs: 8 or 2)
  constexpr int kRaw = RUN == 8 ? 8 : 1, kRuns = 2 * PAIRS / kRaw;
  for (int h = h0; h < h1; h += 4) {                               // the loads of four heads are in flight together
    Raw<T, kRaw> v[4][kRuns];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (h + k >= h1) continue;
      const T* xh = x + (h + k) * p.xs_h;
#pragma unroll
      for (int r = 0; r < kRuns; ++r) v[k][r].load(xh + (HALVES ? (r < kRuns / 2 ? ca : cb - PAIRS) : ca) + r * kRaw);
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (h + k >= h1) continue;
      T* yh = y + (h + k) * p.ys_h;
      float a[2 * PAIRS], o[2 * PAIRS];
#pragma unroll
      for (int r = 0; r < kRuns; ++r) v[k][r].values(a + r * kRaw);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        const int ia = HALVES ? i : 2 * i, ib = HALVES ? PAIRS + i : 2 * i + 1;
        const float va = a[ia], vb = a[ib];
        o[ia] = fmaf(va, cs[i], -vb * sn[i]);
        o[ib] = fmaf(vb, cs[i], va * sn[i]);
        if (!HALVES && u * PAIRS + i >= p.pairs) {                 // copied as they are (an infinity stays one)
          o[ia] = va;
          o[ib] = vb;
        }
      }
      if constexpr (HALVES) {
        store_run<T, VEC>(yh + ca, o);
        store_run<T, VEC>(yh + cb, o + PAIRS);
      } else {
        store_run<T, 2 * PAIRS>(yh + ca, o);
      }
    }
  }
}

template <typename T>
int rope_axes_launch(RopeAxesParams& p, bool vec, bool halves, cudaStream_t st) {
  const int pairs_per_unit = vec ? (halves ? 8 : 4) : 1;
  const int turning = (p.pairs + pairs_per_unit - 1) / pairs_per_unit;
  const int vecw = vec ? 8 : 1;
  const int still = halves || !vec ? (p.hd - 2 * p.pairs + vecw - 1) / vecw : (p.hd + 7) / 8 - turning;
  const int64_t threads = p.T * (turning + still);
  const int64_t blocks = (threads + 255) / 256;
  if (blocks > 0x7fffffff) return SWV_ERR_SHAPE;
  // few tokens: the heads are divided until some eight CTAs an SM are there, two heads at least
  const int64_t want = 8ll * sm_count();
  const int64_t split = std::min<int64_t>(std::min<int64_t>((want + blocks - 1) / blocks, (p.H + 1) / 2), 65535);
  p.heads_per_cta = static_cast<int>((p.H + split - 1) / split);
  const dim3 grid(static_cast<unsigned>(blocks), (p.H + p.heads_per_cta - 1) / p.heads_per_cta);
  auto k = vec ? (halves ? rope_axes_kernel<T, 8, true> : rope_axes_kernel<T, 8, false>)
               : (halves ? rope_axes_kernel<T, 1, true> : rope_axes_kernel<T, 1, false>);
  SWV_CUDA_OK(launch_after(k, grid, 256, 0, st, p));
  return SWV_OK;
}

}  // namespace

int rope_axes_impl(const void* x, const int64_t* xs, void* y, const int64_t* ys, int dtype, const void* pos,
                   int pos_dtype, int64_t pos_stride, const double* freq_host, const uint8_t* axis_host, int pairs,
                   int axes, int halves, int inverse, int64_t T, int H, int hd, cudaStream_t st) {
  if (!xs || !ys || !freq_host || !axis_host) return SWV_ERR_NULL;
  if (T < 0 || H < 1 || hd < 2 || pairs < 1 || 2 * pairs > hd || axes < 1) return SWV_ERR_SHAPE;
  // (heads, channels and the loops over them stay within 32 bits)
  if (pairs > kMaxPairs || axes > kMaxAxes || H > (1 << 29) || hd > (1 << 29)) return SWV_ERR_UNSUPPORTED;
  if (!dtype_known(dtype) || pos_dtype < SWV_POS_F32 || pos_dtype > SWV_POS_I64) return SWV_ERR_DTYPE;
  if (T == 0) return SWV_OK;
  if (!x || !y || !pos) return SWV_ERR_NULL;
  if (xs[2] != 1 || ys[2] != 1) return SWV_ERR_ALIGN;
  RopeAxesParams p{};
  for (int i = 0; i < pairs; ++i) {
    if (axis_host[i] >= axes) return SWV_ERR_SHAPE;
    p.turns[i] = freq_host[i] * 0.15915494309189533577;            // 1 / (2 pi)
    p.axis[i] = axis_host[i];
  }
  p.x = x; p.y = y; p.pos = pos; p.pos_dtype = pos_dtype; p.pos_stride = pos_stride;
  p.T = T; p.H = H; p.hd = hd; p.pairs = pairs;
  p.xs_t = xs[0]; p.xs_h = xs[1]; p.ys_t = ys[0]; p.ys_h = ys[1];
  p.sign = inverse ? -1.f : 1.f;
  const int es = dtype_bytes(dtype);
  const bool vec = hd % 8 == 0 && (!halves || pairs % 8 == 0) && rows_vec8(x, xs[0], es) && rows_vec8(x, xs[1], es) &&
                   rows_vec8(y, ys[0], es) && rows_vec8(y, ys[1], es);
  if (dtype == SWV_F32) return rope_axes_launch<float>(p, vec, halves != 0, st);
  if (dtype == SWV_BF16) return rope_axes_launch<__nv_bfloat16>(p, vec, halves != 0, st);
  return rope_axes_launch<__half>(p, vec, halves != 0, st);
}

}  // namespace swv
