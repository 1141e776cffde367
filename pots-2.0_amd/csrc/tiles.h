// Fragments of the 32x32 matrix-core products that attention.hip and vocab_loss.hip share.
//
// A 32x32x16 product D += A·B has, in lane l of a wave with i = l mod 32 and h = l / 32:
//   A: row i, eight values of the contraction (slots j = 0..7),  B: column i, the same slots,
//   D: column i, rows 8(r / 4) + 4h + r mod 4 of its registers r = 0..15.
// Which member of the contraction a slot stands for is free as long as A and B agree. A result
// D can therefore be the B operand of a next product without leaving its lanes: registers
// 8t .. 8t + 7 of D are, for its contraction step t, the rows 16t + 4h + (0..3) and
// 16t + 8 + 4h + (0..3). Softmax rows are kept as D's columns, so their maximum and sum are
// over a lane's own registers and one exchange between the halves.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gmem.h"

namespace pots {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2v __attribute__((ext_vector_type(2)));

#define POTS_LDS __attribute__((address_space(3)))

__device__ __forceinline__ f32x16 zero16() {
  f32x16 z;
#pragma unroll
  for (int r = 0; r < 16; r++) z[r] = 0.f;
  return z;
}

// The row of D that register r holds in the half h.
__device__ __forceinline__ constexpr uint32_t d_row(uint32_t r, uint32_t h) {
  return 8 * (r / 4) + 4 * h + r % 4;
}

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}

// The same product of fp32 values: eight 32x32x2 steps, step j contracting slot j of the two
// halves.
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; j++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// Four rows of 16 columns of bf16 in LDS, transposed: within each 16 lanes, lane m passes the
// address of row m / 4 at column 4(m mod 4) and receives the four rows of column m.
__device__ __forceinline__ i16x4 read_tr(const void* p) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((POTS_LDS i16x4*)(p));
}

__device__ __forceinline__ bf16x8 join(i16x4 lo, i16x4 hi) {
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ float bf16_to_f32(uint16_t x) {
  return __uint_as_float((uint32_t)x << 16);
}

__device__ __forceinline__ uint16_t f32_to_bf16(float x) {  // to nearest, ties to even
  return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// A buffer of `range` bytes: loads past it read zero.
__device__ __forceinline__ brsrc make_rsrc(const void* base, uint32_t range) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), (short)0, range, 0x00020000);
}

// Sixteen (or four) bytes a lane from a buffer to consecutive places from `lds` on, which is the
// same for the wave. (The host's pass of the compiler knows no such builtin.)
__device__ __forceinline__ void load_lds16(brsrc rsrc, void* lds, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (POTS_LDS void*)lds, 16, off, 0, 0, 0);
#endif
}
__device__ __forceinline__ void load_lds4(brsrc rsrc, void* lds, uint32_t off) {
#if defined(__HIP_DEVICE_COMPILE__)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (POTS_LDS void*)lds, 4, off, 0, 0, 0);
#endif
}

// Waits until at most LEFT of the wave's own loads (the last ones) are on their way, then for the
// block: the stages loaded before those are complete after it.
template <uint32_t LEFT = 0>
__device__ __forceinline__ void loads_done() {
  static_assert(LEFT < 64, "vmcnt has six bits");
  // (a barrier of its own, since __syncthreads waits for every load into LDS; the empty statements
  // keep the compiler from moving accesses over it)
  __builtin_amdgcn_s_waitcnt(0x0070 | (LEFT & 15) | (LEFT >> 4) << 14);  // vmcnt(LEFT) lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Element types of the operators' tensors.
struct Bf16 {
  typedef uint16_t elem;
  typedef bf16x8 frag;
  static __device__ __forceinline__ float get(elem x) { return bf16_to_f32(x); }
  static __device__ __forceinline__ elem put(float x) { return f32_to_bf16(x); }
  static __device__ __forceinline__ float at(const frag& f, int j) { return (float)f[j]; }
  template <typename V>
  static __device__ __forceinline__ frag pack(const V& v, int first) {
    frag f;
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = (__bf16)v[first + j];
    return f;
  }
  // four consecutive elements at an address aligned to them
  static __device__ __forceinline__ void store4(elem* p, float a, float b, float c, float d) {
    bf16x4 v = {(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
    *reinterpret_cast<bf16x4*>(p) = v;
  }
};

struct Fp32 {
  typedef float elem;
  typedef f32x8 frag;
  static __device__ __forceinline__ float get(elem x) { return x; }
  static __device__ __forceinline__ elem put(float x) { return x; }
  static __device__ __forceinline__ float at(const frag& f, int j) { return f[j]; }
  template <typename V>
  static __device__ __forceinline__ frag pack(const V& v, int first) {
    frag f;
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = v[first + j];
    return f;
  }
  static __device__ __forceinline__ void store4(elem* p, float a, float b, float c, float d) {
    f32x4 v = {a, b, c, d};
    *reinterpret_cast<f32x4*>(p) = v;
  }
};

}  // namespace pots
