// The gated activation of a decoder's MLP, with its gradient.
//
//   out = silu(g)·u,  silu(g) = g·σ(g),  σ(g) = 1 / (1 + e^−g)
//   dg = dout·u·(σ(g) + g·(1 − σ(g))·σ(g)),  du = dout·silu(g)
//
// Bound by memory: three tensors forward, five backward, each once, 16 bytes a lane (8192 x 8960 in bf16
// 75 us and 106, 5.9 and 6.9 TB/s). The arithmetic is fp32, rounded once. σ and 1 − σ come from e^−|g|,
// which is at most 1, so that neither loses its last bits to the other.
#include <math.h>

#include "common.h"
#include "gmem.h"
#include "tiles.h"
#include "values.h"

namespace pots {

template <class T>
constexpr uint32_t kValues = 16 / sizeof(typename T::elem);

// σ(g) and 1 − σ(g): one of them is q = 1 / (1 + e^−|g|), the other e^−|g| q. What the exact quotient of the
// exact sum has over q is q times `over`, to first order.
struct Sigma {
  float one, rest, over;
};
// From e^−|g| = 2^n·2^f, n + f = −|g|·log2 e with the constant in two parts (Cody and Waite, 1980), the hardware's 2^f,
// and a reciprocal between 1/2 and 1 improved once by Newton's step. (With the library's exponential and an exact division the vector units are busy for
// 0.87 of a large call, so for 0.62, and a call that the cache holds takes a tenth longer: 1024 x 4864 in
// bf16 forward 9.9 us, so 9.0.) |g| past 200 is 200, since e^−200 is zero; a NaN comes back with g, by which all is
// multiplied.
__device__ __forceinline__ Sigma sigma(float g) {
  constexpr float kLog2e = 1.44269502f, kRest = 1.92596299e-8f;  // log2 e in fp32, and what is left
  const float a = fminf(fabsf(g), 200.f), hi = -a * kLog2e;
  const float lo = fmaf(-a, kRest, fmaf(-a, kLog2e, -hi)), n = rintf(hi);
  const float e = __builtin_ldexpf(__builtin_amdgcn_exp2f(hi - n + lo), (int)n);
  const float d = 1.f + e, r = __builtin_amdgcn_rcpf(d), q = fmaf(fmaf(-d, r, 1.f), r, r);
  const float over = fmaf(d - 1.f - e, q, fmaf(-d, q, 1.f));  // (both differences are exact)
  return g >= 0.f ? Sigma{q, e * q, over} : Sigma{e * q, q, over};
}

// σ(g) + g(1 − σ(g))σ(g), the slope of silu, in one rounding fewer than σ(1 + g(1 − σ)) has. Both factors carry q's
// error, so that it counts up to one and a half times; an fp32 result takes it out again (of normal values dg's error is
// 5.5e-8 of its size so, 6.4e-8 without, and 6.9e-8 with the other rounding).
template <class T>
__device__ __forceinline__ float slope(float g, const Sigma& s) {
  const float x = g * s.rest, v = fmaf(x, s.one, s.one);
  return sizeof(typename T::elem) == 4 ? fmaf(s.over, fmaf(x, 2.f * s.one, s.one), v) : v;
}

// A call whose tensors the last cache does not hold writes past it, and the gradient, which is the last
// to read them, reads past it too (8192 x 8960 in bf16, both directions: 205 us through it, 183 so).
// A smaller one leaves its results there for the product that reads them (with the products around it,
// 1024 x 4864: 98 us, past it 102).
constexpr uint64_t kCache = 256ull << 20;

template <class T, bool GRAD, bool PAST>
__global__ __launch_bounds__(256) void gated(pots_gated_silu a, Divisor runs, uint32_t all) {
  typedef typename T::elem elem;
  constexpr uint32_t N = kValues<T>;
  const uint32_t e = blockIdx.x * 256 + threadIdx.x;
  if (e >= all) return;
  const uint32_t row = runs.of(e), c = (e - row * runs.by) * N;
  Run<T, N> g[1], u[1], d[1];
  load_runs<T, N, 1, GRAD && PAST>(reinterpret_cast<const elem*>(a.gate) + row * a.gate_row, c, 0, a.columns, g);
  load_runs<T, N, 1, GRAD && PAST>(reinterpret_cast<const elem*>(a.up) + row * a.up_row, c, 0, a.columns, u);
  if (GRAD)
    load_runs<T, N, 1, GRAD && PAST>(reinterpret_cast<const elem*>(a.dout) + row * a.dout_row, c, 0, a.columns, d);
  float y[N], z[N];
#pragma unroll
  for (uint32_t j = 0; j < N; j++) {
    const float x = T::get(g[0][j]), v = T::get(u[0][j]);
    const Sigma s = sigma(x);
    if (GRAD) {
      const float dy = T::get(d[0][j]);
      y[j] = dy * v * slope<T>(x, s);
      z[j] = dy * (x * s.one);
    } else {
      y[j] = x * s.one * v;
    }
  }
  const int64_t at = (int64_t)row * a.columns + c;
  store_run<T, N, PAST>(reinterpret_cast<elem*>(GRAD ? a.dgate : a.out) + at, a.columns - c, y);
  if (GRAD) store_run<T, N, PAST>(reinterpret_cast<elem*>(a.dup) + at, a.columns - c, z);
}

namespace {

bool bad(const pots_gated_silu* a) {
  return !a || a->dtype > POTS_OP_BF16 || (uint64_t)a->rows * a->columns > 1ull << 40;
}

// Values of a launch, at the most: below 2^32 threads, and 32 bits hold a column.
constexpr uint32_t kLaunch = 1u << 30;

template <class T, bool GRAD>
int run(const pots_gated_silu* call, hipStream_t s) {
  typedef typename T::elem elem;
  pots_gated_silu a = *call;
  // Rows that follow each other everywhere are one row, as long as it is one.
  const int64_t c = a.columns;
  if ((uint64_t)a.rows * a.columns <= kLaunch && a.gate_row == c && a.up_row == c &&
      (!GRAD || a.dout_row == c)) {
    a.columns *= a.rows;
    a.rows = 1;
  }
  const uint64_t bytes = (uint64_t)a.rows * a.columns * sizeof(elem) * (GRAD ? 5 : 3);
  const auto kernel = bytes > kCache ? gated<T, GRAD, true> : gated<T, GRAD, false>;
  // Some rows a launch, or of longer rows a piece of one.
  const uint32_t wide = a.columns < kLaunch ? a.columns : kLaunch;
  const uint32_t most = a.columns > kLaunch ? 1 : kLaunch / ((wide + kValues<T> - 1) / kValues<T>);
  for (uint64_t r0 = 0; r0 < a.rows; r0 += most) {
    for (uint64_t c0 = 0; c0 < a.columns; c0 += wide) {
      pots_gated_silu part = a;
      part.rows = (uint32_t)(a.rows - r0 < most ? a.rows - r0 : most);
      part.columns = (uint32_t)(a.columns - c0 < wide ? a.columns - c0 : wide);
      part.gate = reinterpret_cast<const elem*>(a.gate) + (int64_t)r0 * a.gate_row + c0;
      part.up = reinterpret_cast<const elem*>(a.up) + (int64_t)r0 * a.up_row + c0;
      const uint64_t at = r0 * a.columns + c0;
      if (GRAD) {
        part.dout = reinterpret_cast<const elem*>(a.dout) + (int64_t)r0 * a.dout_row + c0;
        part.dgate = reinterpret_cast<elem*>(a.dgate) + at;
        part.dup = reinterpret_cast<elem*>(a.dup) + at;
      } else {
        part.out = reinterpret_cast<elem*>(a.out) + at;
      }
      const uint32_t per = (part.columns + kValues<T> - 1) / kValues<T>, all = part.rows * per;
      hipLaunchKernelGGL(kernel, dim3((all + 255) / 256), dim3(256), 0, s, part, Divisor(per), all);
      POTS_HIP(hipGetLastError());
    }
  }
  return POTS_E_OK;
}

}  // namespace

}  // namespace pots

using namespace pots;

extern "C" int pots_gated_silu_forward(const pots_gated_silu* a, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (a->rows == 0 || a->columns == 0) return POTS_E_OK;
  if (!a->gate || !a->up || !a->out) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == POTS_OP_BF16 ? run<Bf16, false>(a, s) : run<Fp32, false>(a, s);
}

extern "C" int pots_gated_silu_backward(const pots_gated_silu* a, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (a->rows == 0 || a->columns == 0) return POTS_E_OK;
  if (!a->gate || !a->up || !a->dout || !a->dgate || !a->dup) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == POTS_OP_BF16 ? run<Bf16, true>(a, s) : run<Fp32, true>(a, s);
}
