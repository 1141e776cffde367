// Runs of values of rows that start anywhere, as the memory-bound operators read and write them.
//
// The GPU's global loads and stores take 16 bytes at any address of an element, so a row of odd width
// or offset is read and written as wide as an aligned one, but for the run that crosses its end.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gmem.h"
#include "tiles.h"

namespace pots {

// Quotients by a number that is the same for the launch, of numbers below 2^31: a multiplication by its reciprocal rounded
// up and a shift (Granlund and Montgomery, 1994).
struct Divisor {
  uint32_t by, factor, shift;

  explicit Divisor(uint32_t d) : by(d), shift(0) {
    while (shift < 31 && (1u << shift) < d) shift++;
    factor = (uint32_t)(((1ull << (31 + shift)) + d - 1) / d);  // (2^31 for d = 1)
  }
  __device__ __forceinline__ uint32_t of(uint32_t n) const {
    return (uint32_t)((uint64_t)n * factor >> 31 >> shift);
  }
};

// N values of a row, one lane's share.
template <class T, uint32_t N>
using Run = typename T::elem __attribute__((ext_vector_type(N)));

// Loads and stores of a V that is aligned as an E alone.
template <class V, class E>
struct __attribute__((packed, aligned(alignof(E)))) Loose {
  V v;
};
template <class V, class E>
__device__ __forceinline__ V load_any(const E* p) {
  return ((const POTS_GLOBAL Loose<V, E>*)p)->v;
}
template <class V, class E>
__device__ __forceinline__ void store_any(E* p, V v) {
  ((POTS_GLOBAL Loose<V, E>*)p)->v = v;
}

// The same past the caches: for what nobody reads soon, or again.
template <class V, class E>
__device__ __forceinline__ V load_past(const E* p) {
  return __builtin_nontemporal_load(&((const POTS_GLOBAL Loose<V, E>*)p)->v);
}
template <class V, class E>
__device__ __forceinline__ void store_past(E* p, V v) {
  __builtin_nontemporal_store(v, &((POTS_GLOBAL Loose<V, E>*)p)->v);
}

// A run's values from the one numbered `by` (0 to N - 1) on, zeros behind them.
template <class T, uint32_t N>
__device__ __forceinline__ Run<T, N> shifted(Run<T, N> x, uint32_t by) {
  if constexpr (sizeof(x) == 8) {
    return __builtin_bit_cast(Run<T, N>, __builtin_bit_cast(uint64_t, x) >> 8 * sizeof(x[0]) * by);
  } else if constexpr (sizeof(x) == 16) {
    return __builtin_bit_cast(
        Run<T, N>, __builtin_bit_cast(unsigned __int128, x) >> 8 * (uint32_t)sizeof(x[0]) * by);
  } else {
#pragma unroll
    for (uint32_t m = 1; m < N; m *= 2) {
      Run<T, N> y = {};
#pragma unroll
      for (uint32_t j = 0; j + m < N; j++) y[j] = x[j + m];
      x = by & m ? y : x;
    }
    return x;
  }
}

// A lane's G runs of a row of `dim` values: those from first + i·step on, zeros past the row's end. A
// run that crosses the end is read as the row's last N values and shifted, so that all loads are on
// their way before the first is waited for. (dim is the same for all lanes, and one of the three ways
// is taken.)
template <class T, uint32_t N, uint32_t G, bool PAST = false>
__device__ __forceinline__ void load_runs(const typename T::elem* row, uint32_t first, uint32_t step,
                                          uint32_t dim, Run<T, N> (&x)[G]) {
  if (dim % N == 0) {
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      x[i] = Run<T, N>{};
      if (first + i * step < dim)
        x[i] = PAST ? load_past<Run<T, N>>(row + first + i * step)
                    : load_any<Run<T, N>>(row + first + i * step);
    }
  } else if (dim > N) {
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      x[i] = Run<T, N>{};
      if (first + i * step < dim) x[i] = load_any<Run<T, N>>(row + min(first + i * step, dim - N));
    }
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      const uint32_t c = first + i * step;
      x[i] = shifted<T, N>(x[i], c < dim ? c - min(c, dim - N) : 0);
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < G; i++) {
      x[i] = Run<T, N>{};
#pragma unroll
      for (uint32_t j = 0; j < N; j++)
        if (first + i * step + j < dim) x[i][j] = gload<typename T::elem>(row + first + i * step + j);
    }
  }
}

// N values from p on, of which the row has `left`.
template <class T, uint32_t N, bool PAST = false>
__device__ __forceinline__ void store_run(typename T::elem* p, uint32_t left,
                                          const float (&v)[N]) {
  if (left >= N) {
    Run<T, N> x;
#pragma unroll
    for (uint32_t j = 0; j < N; j++) x[j] = T::put(v[j]);
    if (PAST)
      store_past(p, x);
    else
      store_any(p, x);
  } else {
#pragma unroll
    for (uint32_t j = 0; j + 1 < N; j++)
      if (j < left) gstore<typename T::elem>(p + j, T::put(v[j]));
  }
}

// The same for a type that is the call's.
template <uint32_t N, bool PAST = false>
__device__ __forceinline__ void put_run(void* p, uint32_t type, int64_t at, uint32_t left,
                                        const float (&v)[N]) {
  if (type == POTS_OP_BF16)
    store_run<Bf16, N, PAST>(reinterpret_cast<uint16_t*>(p) + at, left, v);
  else
    store_run<Fp32, N, PAST>(reinterpret_cast<float*>(p) + at, left, v);
}

// Runs of four whose type is the call's: held as they lie in memory, made fp32 where they are used.
template <uint32_t G>
struct AnyRuns {
  Run<Fp32, 4> raw[G];

  __device__ __forceinline__ void load(const void* p, uint32_t type, uint32_t first, uint32_t step,
                                       uint32_t dim) {
    if (type == POTS_OP_BF16) {
      Run<Bf16, 4> x[G];
      load_runs<Bf16, 4, G>(reinterpret_cast<const uint16_t*>(p), first, step, dim, x);
#pragma unroll
      for (uint32_t i = 0; i < G; i++) {
        const u32x2v bits = __builtin_bit_cast(u32x2v, x[i]);
        raw[i][0] = __uint_as_float(bits[0]);
        raw[i][1] = __uint_as_float(bits[1]);
      }
    } else {
      load_runs<Fp32, 4, G>(reinterpret_cast<const float*>(p), first, step, dim, raw);
    }
  }
  // (The empty statements keep the conversion here, where it does not wait for other loads, and in a
  // branch, which is the same for all lanes.)
  __device__ __forceinline__ void get(uint32_t type, uint32_t i, float (&v)[4]) const {
    float lo = raw[i][0], hi = raw[i][1];
    asm volatile("" : "+v"(lo), "+v"(hi));
    v[0] = lo;
    v[1] = hi;
    v[2] = raw[i][2];
    v[3] = raw[i][3];
    if (type == POTS_OP_BF16) {
      asm volatile("");
      v[0] = __uint_as_float(__float_as_uint(lo) << 16);
      v[1] = __uint_as_float(__float_as_uint(lo) & 0xffff0000u);
      v[2] = __uint_as_float(__float_as_uint(hi) << 16);
      v[3] = __uint_as_float(__float_as_uint(hi) & 0xffff0000u);
    }
  }
};

}  // namespace pots
