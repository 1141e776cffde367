// The residual's addition and the root-mean-square norm of the sum, with its gradient and with an
// output in 8 bits.
//
//   t = x + r,  s = 1 / √(mean t² + ε),  y = t·s·w
//   h = t·s, g = dy·w:  dt = dtotal + s (g − h·mean(g·h)),  dw = Σ_rows dy·h
//   8 bits: a = the largest |y| of a group, scale = a / 448 (e4m3) or a / 127 (int8), q = y / scale
//
// Bound by memory: a row is read once into registers, four consecutive values of each 256 to a lane
// (any width of type then fills whole lines), and everything follows from there. 8192 rows of 1536, x
// and y bf16, r and t fp32: 27 us, 5.6 TB/s; the gradient 34, 5.9 of the 201 MB that it moves, and 4 for dw. (A
// copy of that size reaches 5.0; the gradient finds part of t in the last cache, so stores past it lost 5 %.) In
// 8 bits, where a value is one to three bytes, instructions bound it instead: 45 a value, which keep the vector units busy
// for 0.65 of the launch (8192 x 1536 from bf16 to e4m3 in blocks of 128: 17 us, where the bytes take 7.6). The root, the
// scales and the divisions by them are therefore the hardware's approximations improved once (with exact ones 20 us).
// Sums, the norm and y before its rounding are fp32; t is rounded to the residual's type first, since the next layer reads
// that t, and so does the gradient.
//
// dw: every wave adds up its own rows in registers, a block's waves join in LDS, and norm_join adds
// the blocks' sums in their order, so that no atomics are needed.
#include <math.h>

#include "common.h"
#include "gmem.h"
#include "tiles.h"
#include "values.h"

namespace pots {

constexpr uint32_t kMaxDim = 1u << 14;
constexpr float kLeast = 1.17549435e-38f;  // 2^-126, the smallest normal number

// The sum over L = 16, 32 or 64 lanes, in each of them. Within 16 lanes the operands come by the vector
// instructions' own lane permutations (neighbours, pairs, and mirrored halves, whose lanes hold the same
// sum by then).
template <int CONTROL>
__device__ __forceinline__ float permuted(float v) {
  return __int_as_float(
      __builtin_amdgcn_update_dpp(0, __float_as_int(v), CONTROL, 0xf, 0xf, true));
}
template <uint32_t L>
__device__ __forceinline__ float sum_lanes(float v) {
  v += permuted<0xB1>(v);   // quad_perm [1, 0, 3, 2]
  v += permuted<0x4E>(v);   // quad_perm [2, 3, 0, 1]
  v += permuted<0x141>(v);  // row_half_mirror
  v += permuted<0x140>(v);  // row_mirror
  if constexpr (L >= 32) v += __shfl_xor(v, 16);
  if constexpr (L >= 64) v += __shfl_xor(v, 32);
  return v;
}

// 1 / √x of a normal number: the hardware's, off by a step at most, improved once; off by three quarters of a step
// then, in rstd and y of every type. 0 of infinity.
__device__ __forceinline__ float inverse_root(float x) {
  const float y = __builtin_amdgcn_rsqf(x);
  return x < INFINITY ? fmaf(0.5f * y, fmaf(-x * y, y, 1.f), y) : y;
}

// How a row lies in a block: L lanes of a wave, or W whole waves, and G runs of four values to each
// lane, the columns 4·(L·W·i + lane of the row) on; 4·L·W·G columns at the most.
template <uint32_t G, uint32_t W, uint32_t L = 64>
struct Row {
  static constexpr uint32_t kRuns = G, kWaves = W, kLanes = L, kStep = 4 * L * W;
  static constexpr uint32_t kThreads = W == 1 ? 256 : 64 * W;
  static constexpr uint32_t kRows = kThreads / (L * W);  // of a block
  static_assert(L == 64 || W == 1, "a row is a part of one wave or all of some");

  // The sum over a row, in every lane of it; s: W floats of LDS, used in turn by two calls.
  static __device__ __forceinline__ float sum(float v, float (*s)[W], uint32_t& turn) {
    v = sum_lanes<L>(v);
    if constexpr (W > 1) {
      if (threadIdx.x % 64 == 0) s[turn][threadIdx.x / 64] = v;
      __syncthreads();
      v = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < W; w++) v += s[turn][w];
      turn ^= 1;
    }
    return v;
  }
  static __device__ __forceinline__ uint32_t most(uint32_t v, uint32_t (*s)[W], uint32_t& turn) {
#pragma unroll
    for (int m = L / 2; m; m >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, m));
    if constexpr (W > 1) {
      if (threadIdx.x % 64 == 0) s[turn][threadIdx.x / 64] = v;
      __syncthreads();
#pragma unroll
      for (uint32_t w = 0; w < W; w++) v = max(v, s[turn][w]);
      turn ^= 1;
    }
    return v;
  }
};

// y / by, as a division rounds it but for its last bit at times, from the reciprocal that many share: a
// product and its remainder's. (Where a scale is infinite, `by` and `inverse` are 0, and so is this.)
__device__ __forceinline__ float divided(float y, float by, float inverse) {
  const float q = y * inverse;
  return fmaf(fmaf(-q, by, y), inverse, q);
}

// How many columns of the row are left from c on.
__device__ __forceinline__ uint32_t left_of(uint32_t c, uint32_t dim) { return c < dim ? dim - c : 0; }

template <class X, class T, bool RES, bool Q, class R>
__global__ __launch_bounds__(R::kThreads) void norm_rows(pots_rms_norm a) {
  constexpr uint32_t G = R::kRuns, W = R::kWaves, L = R::kLanes, S = R::kStep;
  __shared__ float s_sum[2][W];
  __shared__ uint32_t s_most[2][W];
  uint32_t turn = 0, turn_most = 0;
  const uint32_t lane = threadIdx.x % (L * W), own = threadIdx.x / (L * W), first = 4 * lane;
  const float over = 1.f / (float)a.dim;
  AnyRuns<G> gain;
  gain.load(a.weight, a.weight_type, first, S, a.dim);
  const uint32_t step = gridDim.x * R::kRows;
  for (uint64_t row = blockIdx.x * R::kRows + own; row < a.rows; row += step) {
    float t[G][4];
    Run<X, 4> x[G];
    Run<T, 4> r[G];
    load_runs<X, 4, G>(reinterpret_cast<const typename X::elem*>(a.x) + (int64_t)row * a.x_row, first,
                       S, a.dim, x);
    if (RES)
      load_runs<T, 4, G>(
          reinterpret_cast<const typename T::elem*>(a.residual) + (int64_t)row * a.residual_row, first,
          S, a.dim, r);
    float sum = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      const uint32_t c = first + S * i;
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        t[i][j] = X::get(x[i][j]);
        if (RES) t[i][j] = T::get(T::put(t[i][j] + T::get(r[i][j])));
        sum = fmaf(t[i][j], t[i][j], sum);
      }
      if (RES)
        store_run<T, 4>(reinterpret_cast<typename T::elem*>(a.total) + row * a.dim + c,
                        left_of(c, a.dim), t[i]);
    }
    const float s = inverse_root(R::sum(sum, s_sum, turn) * over + a.eps);
    if (!Q && lane == 0) gstore<float>(a.rstd + row, s);
    uint32_t most = 0;  // sizes as bits, whose order puts NaN above infinity
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      float w[4];
      gain.get(a.weight_type, i, w);
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        t[i][j] = t[i][j] * s * w[j];
        if (Q) most = max(most, __float_as_uint(t[i][j]) & 0x7fffffffu);
      }
    }
    if constexpr (!Q) {
#pragma unroll
      for (uint32_t i = 0; i < G; i++) {
        const uint32_t c = first + S * i;
        put_run<4>(a.y, a.y_type, (int64_t)(row * a.dim) + c, left_of(c, a.dim), t[i]);
      }
    } else {
      const float top = a.y_type == POTS_OP_E4M3 ? 448.f : 127.f;
      const uint32_t lanes = min(a.block / 4, L);  // of a group
      uint32_t sizes[G];
#pragma unroll
      for (uint32_t i = 0; i < G; i++) {
        sizes[i] = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++)
          sizes[i] = max(sizes[i], __float_as_uint(t[i][j]) & 0x7fffffffu);
      }
      for (uint32_t m = 1; m < lanes; m *= 2)
#pragma unroll
        for (uint32_t i = 0; i < G; i++)
          sizes[i] = max(sizes[i], (uint32_t)__shfl_xor((int)sizes[i], (int)m));
      const uint32_t groups = a.block ? (a.dim + a.block - 1) / a.block : 1;
      if (!a.block) most = R::most(most, s_most, turn_most);
#pragma unroll
      for (uint32_t i = 0; i < G; i++) {
        const uint32_t c = first + S * i, left = left_of(c, a.dim);
        if (a.block) most = sizes[i];
        float scale = __uint_as_float(most);
        if (scale < INFINITY) scale = fmaxf(divided(scale, top, 1.f / top), kLeast);
        const float inv = __builtin_amdgcn_rcpf(scale), divisor = scale < INFINITY ? scale : 0.f;
        if (a.block ? left && lane % lanes == 0 : c == 0)
          gstore<float>(a.scales + row * groups + (a.block ? c / a.block : 0), scale);
        uint8_t* const q = reinterpret_cast<uint8_t*>(a.y) + row * a.dim + c;
        uint32_t b;
        float v[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) v[j] = divided(t[i][j], divisor, inv);
        if (a.y_type == POTS_OP_E4M3) {  // (v is at most 448 and a rounding: no overflow but NaN's)
          b = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
          b = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], (int)b, true);
        } else {
          b = 0;
#pragma unroll
          for (uint32_t j = 0; j < 4; j++)  // 1 to 255 for -127 to 127 (and 0, -128, for a NaN)
            b = __builtin_amdgcn_cvt_pk_u8_f32(rintf(v[j]) + 128.f, j, b);
          b ^= 0x80808080u;
        }
        if (left >= 4) {
          store_any(q, b);
        } else {
#pragma unroll
          for (uint32_t j = 0; j < 3; j++)
            if (j < left) gstore<uint8_t>(q + j, (uint8_t)(b >> 8 * j));
        }
      }
    }
  }
}

// part: [block][dim] sums of dy·h, where a.dweight is there.
template <class Y, class T, class R>
__global__ __launch_bounds__(R::kThreads) void norm_grad(pots_rms_norm a, float* __restrict__ part) {
  constexpr uint32_t G = R::kRuns, W = R::kWaves, L = R::kLanes, S = R::kStep;
  __shared__ float s_sum[2][W];
  __shared__ float s_dw[W == 1 ? R::kRows * S * G : 1];
  uint32_t turn = 0;
  const uint32_t lane = threadIdx.x % (L * W), own = threadIdx.x / (L * W), first = 4 * lane;
  const float over = 1.f / (float)a.dim;
  float dw[G][4] = {};
  AnyRuns<G> gain;
  gain.load(a.weight, a.weight_type, first, S, a.dim);
  const uint32_t step = gridDim.x * R::kRows;
  for (uint64_t row = blockIdx.x * R::kRows + own; row < a.rows; row += step) {
    Run<Y, 4> y[G];
    Run<T, 4> r[G], d[G];
    const typename T::elem* const dt =
        reinterpret_cast<const typename T::elem*>(a.dtotal) + (int64_t)row * a.dtotal_row;
    const float s = gload<float>(a.rstd + row);
    load_runs<Y, 4, G>(reinterpret_cast<const typename Y::elem*>(a.dy) + (int64_t)row * a.dy_row, first,
                       S, a.dim, y);
    load_runs<T, 4, G>(
        reinterpret_cast<const typename T::elem*>(a.total) + (int64_t)row * a.total_row, first,
        S, a.dim, r);
    // (sixteen waves have no registers for it before the sum)
    if (W < 16 && a.dtotal) load_runs<T, 4, G>(dt, first, S, a.dim, d);
    float sum = 0.f;
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      float w[4];
      gain.get(a.weight_type, i, w);
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const float h = T::get(r[i][j]) * s, dy = Y::get(y[i][j]);
        sum = fmaf(dy * w[j], h, sum);
        dw[i][j] = fmaf(dy, h, dw[i][j]);
      }
    }
    const float mean = R::sum(sum, s_sum, turn) * over;
    if (W == 16 && a.dtotal) load_runs<T, 4, G>(dt, first, S, a.dim, d);
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      const uint32_t c = first + S * i, left = left_of(c, a.dim);
      const int64_t at = (int64_t)(row * a.dim) + c;
      float v[4], w[4];
      gain.get(a.weight_type, i, w);
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) {
        const float h = T::get(r[i][j]) * s;
        v[j] = s * fmaf(-h, mean, Y::get(y[i][j]) * w[j]);
        if (a.dtotal) v[j] += T::get(d[i][j]);
      }
      if (a.dresidual)
        store_run<T, 4>(reinterpret_cast<typename T::elem*>(a.dresidual) + at, left, v);
      if (a.dx) put_run<4>(a.dx, a.x_type, at, left, v);
    }
  }
  if (!a.dweight) return;
  float* const sums = part + (uint64_t)blockIdx.x * a.dim;
  if constexpr (W == 1) {  // (each of the block's rows has had sums of its own)
#pragma unroll
    for (uint32_t i = 0; i < G; i++)
#pragma unroll
      for (uint32_t j = 0; j < 4; j++) s_dw[own * S * G + S * i + first + j] = dw[i][j];
    __syncthreads();
    for (uint32_t c = threadIdx.x; c < a.dim; c += 256) {
      float v = 0.f;
#pragma unroll
      for (uint32_t r = 0; r < R::kRows; r++) v += s_dw[r * S * G + c];
      sums[c] = v;
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      const uint32_t c = first + S * i;
      put_run<4>(sums, POTS_OP_F32, c, left_of(c, a.dim), dw[i]);
    }
  }
}

// dweight from `parts` rows of sums: 32 columns a block, a 32nd of the rows to each group of lanes.
__global__ __launch_bounds__(1024) void norm_join(const float* __restrict__ part, void* dweight,
                                                  uint32_t parts, uint32_t dim, uint32_t type) {
  __shared__ float s_sum[32][33];
  const uint32_t x = threadIdx.x % 32, g = threadIdx.x / 32, c = blockIdx.x * 32 + x;
  float sum = 0.f;
  if (c < dim) {
    for (uint32_t p = g; p < parts; p += 256) {
      float v[8];
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) {
        const uint32_t at = p + 32 * u;
        v[u] = at < parts ? gload<float>(part + (uint64_t)at * dim + c) : 0.f;
      }
#pragma unroll
      for (uint32_t u = 0; u < 8; u++) sum += v[u];
    }
  }
  s_sum[g][x] = sum;
  __syncthreads();
  if (g != 0 || c >= dim) return;
  for (uint32_t i = 1; i < 32; i++) sum += s_sum[i][x];
  if (type == POTS_OP_BF16)
    gstore<uint16_t>(reinterpret_cast<uint16_t*>(dweight) + c, f32_to_bf16(sum));
  else
    gstore<float>(reinterpret_cast<float*>(dweight) + c, sum);
}

namespace {

bool bad(const pots_rms_norm* a) {
  return !a || a->dim == 0 || a->dim > kMaxDim || a->rows > 0x7fffffffu ||
         a->x_type > POTS_OP_BF16 || a->total_type > POTS_OP_BF16 ||
         a->weight_type > POTS_OP_BF16 || !(a->eps >= kLeast) || !isfinite(a->eps);
}

// Rows of up to 1024 columns are a wave's or a part of one: the sum over a row then needs no barrier.
// Wider ones are shared by four to sixteen waves, so that a lane holds 16 values at most: in a wave of
// its own a row of 2048 leaves room for few waves, and forward and backward of 6144 such rows took 84 us
// where four waves to a row take 71. (8192 columns: 80 us with eight waves, 90 with four. 65536 rows of
// 64: 85 us in a wave each, 32 in a quarter of one.)
template <class F>
int by_width(uint32_t dim, F&& f) {
  if (dim <= 64) return f(Row<1, 1, 16>{});
  if (dim <= 128) return f(Row<1, 1, 32>{});
  if (dim <= 256) return f(Row<1, 1>{});
  if (dim <= 512) return f(Row<2, 1>{});
  if (dim <= 768) return f(Row<3, 1>{});
  if (dim <= 1024) return f(Row<4, 1>{});
  if (dim <= 2048) return f(Row<2, 4>{});
  if (dim <= 4096) return f(Row<4, 4>{});
  if (dim <= 8192) return f(Row<4, 8>{});
  return f(Row<4, 16>{});
}

template <class F>
int by_type(uint32_t type, F&& f) {
  return type == POTS_OP_BF16 ? f(Bf16{}) : f(Fp32{});
}

template <bool Q>
int forward(const pots_rms_norm* a, hipStream_t s) {
  return by_width(a->dim, [&](auto r) {
    typedef decltype(r) R;
    const uint32_t want = (uint32_t)(((uint64_t)a->rows + R::kRows - 1) / R::kRows);
    const uint32_t nb = want < 4096 ? want : 4096;
    return by_type(a->x_type, [&](auto x) {
      return by_type(a->total_type, [&](auto t) {
        typedef decltype(x) X;
        typedef decltype(t) T;
        if (a->residual) {
          hipLaunchKernelGGL((norm_rows<X, T, true, Q, R>), dim3(nb), dim3(R::kThreads), 0, s, *a);
        } else {
          hipLaunchKernelGGL((norm_rows<X, X, false, Q, R>), dim3(nb), dim3(R::kThreads), 0, s, *a);
        }
        POTS_HIP(hipGetLastError());
        return POTS_E_OK;
      });
    });
  });
}

// Blocks of the gradient's kernel. Each leaves a row of sums of dw for norm_join, so they are few, two to a
// compute unit; more where a lane has few runs on their way (49152 rows of 256 columns, both
// directions: 92 us with 512 blocks, 69 with 1536, 77 with 4096; 8192 rows of 1536: 71 with 1024, 78
// with 2048).
template <class R>
uint32_t grad_blocks(const pots_rms_norm* a) {
  constexpr uint32_t most = R::kWaves == 1 ? (R::kRuns == 1   ? 1536
                                              : R::kRuns == 2 ? 1024
                                              : R::kRuns == 3 ? 768
                                                              : 512)
                            : R::kRuns == 2  ? 1024
                                             : 512;
  const uint64_t want = ((uint64_t)a->rows + R::kRows - 1) / R::kRows;
  return (uint32_t)(want < most ? want : most);
}

bool bad_back(const pots_rms_norm* a) { return bad(a) || a->y_type > POTS_OP_BF16; }

}  // namespace

}  // namespace pots

using namespace pots;

static int forward_checked(const pots_rms_norm* a, bool quantized, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (quantized) {
    if (a->y_type != POTS_OP_E4M3 && a->y_type != POTS_OP_INT8) return POTS_E_ARG;
    if (a->block != 0 && a->block != 32 && a->block != 64 && a->block != 128 && a->block != 256)
      return POTS_E_ARG;
  } else if (a->y_type > POTS_OP_BF16) {
    return POTS_E_ARG;
  }
  if (a->rows == 0) return POTS_E_OK;
  if (!a->x || !a->weight || !a->y || (quantized ? !a->scales : !a->rstd) ||
      (a->residual && !a->total))
    return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return quantized ? forward<true>(a, s) : forward<false>(a, s);
}

extern "C" int pots_rms_norm_forward(const pots_rms_norm* a, void* stream) {
  return forward_checked(a, false, stream);
}

extern "C" int pots_rms_norm_quantized(const pots_rms_norm* a, void* stream) {
  return forward_checked(a, true, stream);
}

extern "C" uint64_t pots_rms_norm_backward_work(const pots_rms_norm* a) {
  if (bad_back(a) || !a->dweight) return 0;
  uint64_t blocks = 0;
  (void)by_width(a->dim, [&](auto r) {
    blocks = grad_blocks<decltype(r)>(a);
    return POTS_E_OK;
  });
  return blocks * a->dim * 4;
}

extern "C" int pots_rms_norm_backward(const pots_rms_norm* a, void* work, void* stream) {
  if (bad_back(a)) return POTS_E_ARG;
  if (a->rows && (!a->dy || !a->total || !a->weight || !a->rstd)) return POTS_E_ARG;
  if (a->rows && a->dweight && !work) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  float* const part = static_cast<float*>(work);
  uint32_t blocks = 0;
  const int rc = by_width(a->dim, [&](auto r) {
    typedef decltype(r) R;
    blocks = grad_blocks<R>(a);
    if (!blocks) return POTS_E_OK;
    return by_type(a->y_type, [&](auto y) {
      return by_type(a->total_type, [&](auto t) {
        typedef decltype(y) Y;
        typedef decltype(t) T;
        hipLaunchKernelGGL((norm_grad<Y, T, R>), dim3(blocks), dim3(R::kThreads), 0, s, *a, part);
        POTS_HIP(hipGetLastError());
        return POTS_E_OK;
      });
    });
  });
  if (rc != POTS_E_OK || !a->dweight) return rc;
  hipLaunchKernelGGL(norm_join, dim3((a->dim + 31) / 32), dim3(1024), 0, s, part, a->dweight,
                     blocks, a->dim, a->weight_type);
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}
