// Softmax cross entropy of feature rows against a vocabulary matrix, with its gradient, for
// passes that keep no logits.
//
//   s_rv = x_r·w_v,  lse_r = log Σ_v e^{s_rv},  loss_r = lse_r − s_{r,t_r}
//   g_rv = weight_r (e^{s_rv − lse_r} − [v = t_r]),  dx = G·W,  dW = Gᵀ·X
//
// Forward: a tile of S is a product whose epilogue leaves a maximum and a sum of exponentials
// per row and 32·MB vocabulary rows; loss_rows joins them. Backward, in pieces of the
// vocabulary: S again with the epilogue that writes the piece of G, then that piece's rows of
// dW, and its share of dx added to fp32 sums. Rows that carry no weight are left out of the
// products first (live_rows: prompts, rows without a target), and so is whatever they hold.
//
// All three products are one tiled kernel over the matrix cores (Tile), each operand stored
// either with the contraction along its rows or with its rows along the contraction (W of dx,
// G and X of dW); the latter are read transposed from LDS. bf16 is multiplied as it is. An fp32
// value is the exact sum of three bf16 terms of eight bits each (split3), and a product of two
// takes the six products of terms that reach 2^-24 of it: at six bf16 products' cost that is
// 2.6 times the rate of the fp32 matrix instructions, with their accuracy (the three products
// left out are below 2^-24 of |x||w|). G is rounded to the inputs' type as an operand: half a
// step of bf16, 2^-9 of each term of sums that are rounded to bf16 themselves.
#include <math.h>

#include "common.h"
#include "gmem.h"
#include "tiles.h"

namespace pots {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t BK = 64;  // contraction per stage: 128 bytes of a row

// A matrix of bf16 terms: rows `ld` elements apart, term planes `plane` elements apart.
struct Mat {
  const uint16_t* p;
  int64_t ld, plane;
};


__device__ __forceinline__ void pair_of(uint32_t pairs, uint32_t t, uint32_t* pa, uint32_t* pb) {
  // (0,2) (1,1) (2,0) (0,1) (1,0) (0,0); one pair of plane 0 for bf16
  const uint32_t j = pairs == 1 ? 5 : t;
  *pa = (0x010210u >> (4 * j)) & 15;
  *pb = (0x001012u >> (4 * j)) & 15;
}

// T rows of an operand and BK of the contraction in LDS, in 16-byte chunks that one
// instruction brings in for 64 lanes, straight from memory. TR: stored [contraction][rows], so
// a stage is BK rows of T columns; else T rows of BK columns. A chunk is exchanged within its
// row by the row's number, so that the reads of a fragment fall on different banks: eight
// lanes' 16-byte reads of eight rows, or 32 lanes' transposing reads of four rows.
template <bool TR, uint32_t T, uint32_t NT>
struct Stage {
  static constexpr uint32_t kChunks = T * BK / 8 / NT;
  static_assert(T * BK / 8 % NT == 0, "a stage is whole instructions");
  static_assert(!TR || T >= 128, "the exchange of a transposed tile needs 16 chunks a row");

  // r0, rows: the tile's first row and their number (for TR: columns, a multiple of 8); k0,
  // ks: the contraction's. Rows and contraction past the end repeat the last.
  static __device__ __forceinline__ void load(uint16_t* lds, const Mat& m, uint32_t plane,
                                              uint32_t r0, uint32_t rows, uint32_t k0,
                                              uint32_t ks) {
    const uint16_t* base = m.p + (int64_t)plane * m.plane;
    const uint32_t wave = threadIdx.x / 64;
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++) {
      const uint32_t first = (u * NT / 64 + wave) * 64, c = first + threadIdx.x % 64;
      const uint16_t* src;
      if constexpr (TR) {
        const uint32_t r = c / (T / 8), at = (c % (T / 8)) ^ (4 * (r & 3));
        src = base + (int64_t)min(k0 + r, ks - 1) * m.ld + min(r0 + 8 * at, rows - 8);
      } else {
        const uint32_t r = c / (BK / 8), at = (c % (BK / 8)) ^ (r & 7);
        src = base + (int64_t)min(r0 + r, rows - 1) * m.ld + k0 + 8 * at;
      }
      __builtin_amdgcn_global_load_lds((const POTS_GLOBAL void*)src,
                                       (POTS_LDS void*)(lds + first * 8), 16, 0, 0);
    }
  }

  // Rows c .. c + 31 at step ks of the stage: contraction 16ks + 8h + (0..7).
  static __device__ __forceinline__ bf16x8 frag(const uint16_t* lds, uint32_t c, uint32_t ks,
                                                uint32_t lane) {
    const uint32_t h = lane / 32;
    if constexpr (TR) {
      const uint32_t m = lane % 16, r = 16 * ks + 8 * h + m / 4;
      const uint32_t col = c + (lane & 16) + 4 * (m % 4);
      const uint16_t* p = lds + r * T + (((col / 8) ^ (4 * (r & 3))) * 8 + col % 8);
      return join(read_tr(p), read_tr(p + 4 * T));
    } else {
      const uint32_t r = c + lane % 32;
      return *reinterpret_cast<const bf16x8*>(lds + r * BK + (((2 * ks + h) ^ (r & 7)) * 8));
    }
  }
};

// Waits for the wave's own loads into LDS, then for the block: a stage is complete after it.
__device__ __forceinline__ void loads_done() {
  __builtin_amdgcn_s_waitcnt(0x0F70);  // vmcnt(0)
  __syncthreads();
}

// A block's TM x TN of A·Bᵀ over K (a multiple of BK), WM x WN waves of MB x NB products of 32.
template <bool ATR, bool BTR, uint32_t TM_, uint32_t TN_, uint32_t WM, uint32_t WN>
struct Tile {
  static constexpr uint32_t TM = TM_, TN = TN_, NT = 64 * WM * WN;
  static constexpr uint32_t MB = TM / WM / 32, NB = TN / WN / 32;
  typedef Stage<ATR, TM, NT> SA;
  typedef Stage<BTR, TN, NT> SB;
  f32x16 acc[MB][NB];
  uint32_t wm, wn, lane;

  __device__ __forceinline__ void step(const uint16_t* a, const uint16_t* b) {
#pragma unroll
    for (uint32_t ks = 0; ks < BK / 16; ks++) {
      bf16x8 fa[MB], fb[NB];
#pragma unroll
      for (uint32_t m = 0; m < MB; m++) fa[m] = SA::frag(a, wm + 32 * m, ks, lane);
#pragma unroll
      for (uint32_t n = 0; n < NB; n++) fb[n] = SB::frag(b, wn + 32 * n, ks, lane);
#pragma unroll
      for (uint32_t m = 0; m < MB; m++)
#pragma unroll
        for (uint32_t n = 0; n < NB; n++) acc[m][n] = mma(fa[m], fb[n], acc[m][n]);
    }
  }

  // ka: the contraction's length where an operand is stored along it and may end inside K.
  __device__ __forceinline__ void run(const Mat& A, const Mat& B, uint32_t m0, uint32_t M,
                                      uint32_t n0, uint32_t N, uint32_t K, uint32_t ka,
                                      uint32_t kb, uint32_t pairs) {
    __shared__ __attribute__((aligned(16))) uint16_t s_a0[TM * BK], s_b0[TN * BK];
    __shared__ __attribute__((aligned(16))) uint16_t s_a1[TM * BK], s_b1[TN * BK];
    lane = threadIdx.x % 64;
    wm = threadIdx.x / 64 / WN * (TM / WM);
    wn = threadIdx.x / 64 % WN * (TN / WN);
#pragma unroll
    for (uint32_t m = 0; m < MB; m++)
#pragma unroll
      for (uint32_t n = 0; n < NB; n++) acc[m][n] = zero16();
    const uint32_t steps = K / BK * pairs;
    uint32_t k = 0, pair = 0;
    auto load = [&](uint16_t* a, uint16_t* b) {
      uint32_t pa, pb;
      pair_of(pairs, pair, &pa, &pb);
      SA::load(a, A, pa, m0, M, k, ka);
      SB::load(b, B, pb, n0, N, k, kb);
      k += BK;
      if (k == K) {
        k = 0;
        pair++;
      }
    };
    if (steps) load(s_a0, s_b0);
    for (uint32_t t = 0; t < steps; t += 2) {
      loads_done();
      if (t + 1 < steps) load(s_a1, s_b1);
      step(s_a0, s_b0);
      if (t + 1 == steps) break;
      loads_done();
      if (t + 2 < steps) load(s_a0, s_b0);
      step(s_a1, s_b1);
    }
  }

  // f(m, n, acc, row of A of register 0 of the lane, row of B of the lane)
  template <class F>
  __device__ __forceinline__ void each(uint32_t m0, uint32_t n0, F f) {
#pragma unroll
    for (uint32_t n = 0; n < NB; n++)
#pragma unroll
      for (uint32_t m = 0; m < MB; m++)
        f(acc[m][n], m0 + wm + 32 * m + 4 * (lane / 32), n0 + wn + 32 * n + lane % 32);
  }
};

// Tiles of a launch: an XCD's blocks are neighbours, groups of eight tiles of B by all of A's,
// so that the 32 that run at once read four and eight tiles' operands through their L2.
__device__ __forceinline__ void tile_of(uint32_t mt, uint32_t nt, uint32_t* m, uint32_t* n) {
  const uint32_t u = xcd_block(blockIdx.x, mt * nt), g = u / (8 * mt), in = u % (8 * mt);
  const uint32_t w = min(8u, nt - 8 * g);
  *m = in / w;
  *n = 8 * g + in % w;
}

// ---- laying operands out --------------------------------------------------------------------

__device__ __forceinline__ void split3(float x, uint16_t* t) {
  const uint32_t u = __float_as_uint(x);
  if ((u & 0x7F800000u) == 0x7F800000u) {  // one term; a NaN keeps a bit of its fraction
    t[0] = (u >> 16) | ((u & 0x7FFFFFu) ? 0x40 : 0);
    t[1] = t[2] = 0;
    return;
  }
  const float r = x - __uint_as_float(u & 0xFFFF0000u);  // the lower 16 bits, exact
  const uint32_t v = __float_as_uint(r);
  const float q = r - __uint_as_float(v & 0xFFFF0000u);  // eight bits at most
  t[0] = u >> 16;
  t[1] = v >> 16;
  t[2] = __float_as_uint(q) >> 16;
}

// dst [terms][rows_pad][dp] of src rows (through idx where given, rows from *count on zero).
template <class T>
__global__ __launch_bounds__(256) void lay_out(const typename T::elem* __restrict__ src,
                                               int64_t ld, uint32_t d, uint32_t rows,
                                               const uint32_t* __restrict__ idx,
                                               const uint32_t* __restrict__ count,
                                               uint16_t* __restrict__ dst, uint32_t dp,
                                               uint64_t plane, uint32_t rows_pad) {
  const uint32_t live = count ? gload<uint32_t>(count) : rows;
  const uint64_t total = (uint64_t)rows_pad * (dp / 4);
  for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < total;
       e += (uint64_t)gridDim.x * 256) {
    const uint32_t r = e / (dp / 4), c = e % (dp / 4) * 4;
    constexpr uint32_t kTerms = sizeof(typename T::elem) == 4 ? 3 : 1;
    uint16_t t[4][3] = {};
    if (r < live) {
      const typename T::elem* p = src + (int64_t)(idx ? idx[r] : r) * ld;
#pragma unroll
      for (uint32_t j = 0; j < 4; j++)
        if (c + j < d) {
          if constexpr (kTerms == 3)
            split3(p[c + j], t[j]);
          else
            t[j][0] = p[c + j];
        }
    }
#pragma unroll
    for (uint32_t x = 0; x < kTerms; x++) {
      u32x2v v = {(uint32_t)t[0][x] | (uint32_t)t[1][x] << 16,
                  (uint32_t)t[2][x] | (uint32_t)t[3][x] << 16};
      *reinterpret_cast<u32x2v*>(dst + x * plane + (uint64_t)r * dp + c) = v;
    }
  }
}

// The rows that carry a gradient, in order: idx, their number, each row's place (or ~0), and
// their weights, targets and lse (in units of log2) gathered.
__global__ __launch_bounds__(1024) void live_rows(pots_vocab_loss a, uint32_t* __restrict__ idx,
                                                  uint32_t* __restrict__ pos,
                                                  uint32_t* __restrict__ count,
                                                  float* __restrict__ weight,
                                                  float* __restrict__ lse2,
                                                  uint32_t* __restrict__ target) {
  __shared__ uint32_t s_wave[16];
  uint32_t base = 0;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  for (uint32_t r0 = 0; r0 < a.rows; r0 += 1024) {
    const uint32_t r = r0 + threadIdx.x;
    const float w = r < a.rows ? a.weights[r] : 0.f;
    const int64_t t = r < a.rows ? a.targets[r] : -1;
    const bool live = w != 0.f && t >= 0;  // a NaN weight counts
    const uint64_t mask = __ballot(live);
    if (lane == 0) s_wave[wave] = __popcll(mask);
    __syncthreads();
    uint32_t at = base, all = 0;
    for (uint32_t v = 0; v < 16; v++) {
      if (v < wave) at += s_wave[v];
      all += s_wave[v];
    }
    __syncthreads();
    at += __popcll(mask & ((1ull << lane) - 1));
    if (r < a.rows) pos[r] = live ? at : ~0u;
    if (live) {
      idx[at] = r;
      weight[at] = t < a.vocab ? w : NAN;
      lse2[at] = a.lse[r] * kLog2e;
      target[at] = (uint32_t)t;
    }
    base += all;
  }
  if (threadIdx.x == 0) *count = base;
}

// ---- the products ---------------------------------------------------------------------------

// A piece of the vocabulary from v0 on, `nv` rows of it, against rows of x: a maximum (times
// log2 e) and a sum of 2^(s - maximum) per row and wave, part[chunk][row], and the targets' s.
template <class C>
__global__ __launch_bounds__(C::NT) void loss_scores(Mat W, Mat X, uint32_t v0, uint32_t nv,
                                                     uint32_t rows, uint32_t K, uint32_t pairs,
                                                     uint32_t mt, uint32_t nt,
                                                     const int64_t* __restrict__ targets,
                                                     float2* __restrict__ part,
                                                     uint32_t part_ld,
                                                     float* __restrict__ hit) {
  uint32_t m, n;
  tile_of(mt, nt, &m, &n);
  C c;
  const uint32_t m0 = m * C::TM, n0 = n * C::TN;
  c.run(W, X, m0, nv, n0, rows, K, 0, 0, pairs);
  const uint32_t mw = m0 + c.wm;  // the wave's vocabulary rows: 32·MB of them
  if (mw + 32 * C::MB > nv)
    c.each(m0, n0, [&](f32x16& s, uint32_t v, uint32_t) {
#pragma unroll
      for (uint32_t r = 0; r < 16; r++)
        if (v + d_row(r, 0) >= nv) s[r] = -INFINITY;
    });
#pragma unroll
  for (uint32_t b = 0; b < C::NB; b++) {
    const uint32_t row = n0 + c.wn + 32 * b + c.lane % 32;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (uint32_t x = 0; x < C::MB; x++)
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) top = fmaxf(top, c.acc[x][b][r]);
    top = fmaxf(top, __shfl_xor(top, 32));
    const float tc = top == -INFINITY ? 0.f : top * kLog2e;
#pragma unroll
    for (uint32_t x = 0; x < C::MB; x++)
#pragma unroll
      for (uint32_t r = 0; r < 16; r++)
        sum += __builtin_amdgcn_exp2f(__builtin_fmaf(c.acc[x][b][r], kLog2e, -tc));
    sum += __shfl_xor(sum, 32);
    if (row < rows && c.lane < 32)
      part[(uint64_t)((v0 + mw) / (32 * C::MB)) * part_ld + row] = {tc, sum};
    const int64_t t = row < rows ? targets[row] - v0 - mw : -1;
    const bool here = t >= 0 && t < 32 * C::MB && mw + t < nv;
    if (__any(here)) {
#pragma unroll
      for (uint32_t x = 0; x < C::MB; x++)
#pragma unroll
        for (uint32_t r = 0; r < 16; r++)
          if (here && t == 32 * x + d_row(r, c.lane / 32)) hit[row] = c.acc[x][b][r];
    }
  }
}

// 32 rows a block, the chunks over 32 groups of lanes, joined in a fixed order.
__global__ __launch_bounds__(1024) void loss_rows(const float2* __restrict__ part,
                                                  uint32_t part_ld, uint32_t chunks,
                                                  const float* __restrict__ hit,
                                                  pots_vocab_loss a) {
  __shared__ float2 s_part[32][33];
  const uint32_t i = threadIdx.x % 32, g = threadIdx.x / 32, row = blockIdx.x * 32 + i;
  float m = -INFINITY, l = 0.f;
  if (row < a.rows)
    for (uint32_t c = g; c < chunks; c += 32) {
      const float2 p = part[(uint64_t)c * part_ld + row];
      if (p.x > m) {
        l *= __builtin_amdgcn_exp2f(m - p.x);
        m = p.x;
      }
      l += p.y * __builtin_amdgcn_exp2f(p.x - m);
    }
  s_part[g][i] = {m, l};
  __syncthreads();
  if (g != 0 || row >= a.rows) return;
  for (uint32_t x = 0; x < 32; x++) m = fmaxf(m, s_part[x][i].x);
  l = 0.f;
  for (uint32_t x = 0; x < 32; x++) {
    const float2 p = s_part[x][i];
    if (p.x != -INFINITY) l += p.y * __builtin_amdgcn_exp2f(p.x - m);
  }
  const float lse = (m + __builtin_amdgcn_logf(l)) * kLn2;
  const int64_t t = a.targets[row];
  a.lse[row] = lse;
  a.loss[row] = t < 0 ? 0.f : t < a.vocab ? lse - hit[row] : NAN;
}

// The piece's G, [terms][live rows][ld], zero past the live rows and the vocabulary.
template <class T, class C>
__global__ __launch_bounds__(C::NT) void loss_grad(Mat W, Mat X, uint32_t v0, uint32_t nv,
                                                   const uint32_t* __restrict__ count,
                                                   uint32_t K, uint32_t pairs, uint32_t mt,
                                                   uint32_t nt,
                                                   const float* __restrict__ weight,
                                                   const float* __restrict__ lse2,
                                                   const uint32_t* __restrict__ target,
                                                   uint16_t* __restrict__ g, uint32_t ld,
                                                   uint64_t plane) {
  uint32_t m, n;
  tile_of(mt, nt, &m, &n);
  const uint32_t live = gload<uint32_t>(count);
  const uint32_t m0 = m * C::TM, n0 = n * C::TN;
  if (n0 >= live) return;
  C c;
  c.run(W, X, m0, nv, n0, live, K, 0, 0, pairs);
  c.each(m0, n0, [&](f32x16& s, uint32_t v, uint32_t row) {
    const bool on = row < live;
    const float w = on ? weight[row] : 0.f, l2 = on ? lse2[row] : 0.f;
    const uint32_t t = on ? target[row] - v0 : ~0u;
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      uint16_t e[4][3];
#pragma unroll
      for (uint32_t x = 0; x < 4; x++) {
        const uint32_t at = v + 8 * q + x;
        const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[4 * q + x], kLog2e, -l2));
        const float y = on && at < nv ? w * (at == t ? p - 1.f : p) : 0.f;
        if constexpr (sizeof(typename T::elem) == 4)
          split3(y, e[x]);
        else
          e[x][0] = f32_to_bf16(y);
      }
#pragma unroll
      for (uint32_t k = 0; k < (sizeof(typename T::elem) == 4 ? 3 : 1); k++) {
        const u32x2v o = {(uint32_t)e[0][k] | (uint32_t)e[1][k] << 16,
                          (uint32_t)e[2][k] | (uint32_t)e[3][k] << 16};
        *reinterpret_cast<u32x2v*>(g + k * plane + (uint64_t)row * ld + v + 8 * q) = o;
      }
    }
  });
}

// dx's share of the piece: Wᵀ (stored along the contraction) by G, added to sums [rows][dp].
template <class C>
__global__ __launch_bounds__(C::NT) void loss_dx(Mat W, Mat G, uint32_t dp, uint32_t nv,
                                                 const uint32_t* __restrict__ count, uint32_t K,
                                                 uint32_t pairs, uint32_t mt, uint32_t nt,
                                                 float* __restrict__ sums, bool first) {
  uint32_t m, n;
  tile_of(mt, nt, &m, &n);
  const uint32_t live = gload<uint32_t>(count);
  const uint32_t m0 = m * C::TM, n0 = n * C::TN;
  if (n0 >= live) return;
  C c;
  c.run(W, G, m0, dp, n0, live, K, nv, 0, pairs);
  c.each(m0, n0, [&](f32x16& s, uint32_t col, uint32_t row) {
    if (row >= live) return;
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      if (col + 8 * q >= dp) continue;
      f32x4* p = reinterpret_cast<f32x4*>(sums + (uint64_t)row * dp + col + 8 * q);
      f32x4 y = {s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
      if (!first) y += *p;
      *p = y;
    }
  });
}

// The piece's rows of dW: Xᵀ by Gᵀ, both stored along the contraction (the live rows).
template <class T, class C>
__global__ __launch_bounds__(C::NT) void loss_dw(Mat X, Mat G, uint32_t dp, uint32_t nv,
                                                 const uint32_t* __restrict__ count,
                                                 uint32_t pairs, uint32_t mt, uint32_t nt,
                                                 uint32_t d, typename T::elem* __restrict__ dw,
                                                 int64_t ld, bool vec) {
  uint32_t m, n;
  tile_of(mt, nt, &m, &n);
  const uint32_t live = gload<uint32_t>(count);
  const uint32_t m0 = m * C::TM, n0 = n * C::TN, K = (live + BK - 1) / BK * BK;
  C c;
  c.run(X, G, m0, dp, n0, (nv + 7) & ~7u, K, K, K, pairs);
  c.each(m0, n0, [&](f32x16& s, uint32_t col, uint32_t v) {
    if (v >= nv) return;
    typename T::elem* p = dw + (int64_t)v * ld;
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      const uint32_t at = col + 8 * q;
      if (at >= d) continue;
      if (vec) {
        T::store4(p + at, s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]);
      } else {
#pragma unroll
        for (uint32_t x = 0; x < 4; x++)
          if (at + x < d) p[at + x] = T::put(s[4 * q + x]);
      }
    }
  });
}

// dx from the sums: a block a row, zero for the rows left out.
template <class T>
__global__ __launch_bounds__(256) void loss_dx_rows(const float* __restrict__ sums, uint32_t dp,
                                                    const uint32_t* __restrict__ pos,
                                                    uint32_t d, typename T::elem* dx,
                                                    int64_t ld) {
  const uint32_t row = blockIdx.x, at = pos[row];
  for (uint32_t c = threadIdx.x; c < d; c += 256)
    dx[(int64_t)row * ld + c] = T::put(at == ~0u ? 0.f : sums[(uint64_t)at * dp + c]);
}

namespace {

typedef Tile<false, false, 128, 128, 2, 2> Scores;
typedef Tile<true, false, 128, 128, 2, 2> DxTile;
typedef Tile<true, true, 128, 128, 2, 2> DwTile;

uint32_t cdiv(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

// Sizes and the workspace's parts.
struct Plan {
  uint32_t dp, terms, pairs, rows_pad, piece;
  bool copy_w, copy_x;
  uint64_t w, x, part, hit, idx, pos, count, weight, lse2, target, g, sums, bytes;
};

uint64_t take(Plan* p, uint64_t bytes) {
  const uint64_t at = p->bytes;
  p->bytes += align_up(bytes, 256);
  return at;
}

bool as_is(const pots_vocab_loss* a, const void* p, int64_t row) {
  return a->dtype == POTS_OP_BF16 && a->dim % BK == 0 &&
         reinterpret_cast<uint64_t>(p) % 16 == 0 && row % 8 == 0;
}

Plan plan(const pots_vocab_loss* a, bool backward) {
  Plan p = {};
  p.terms = a->dtype == POTS_OP_BF16 ? 1 : 3;
  p.pairs = a->dtype == POTS_OP_BF16 ? 1 : 6;
  p.dp = cdiv(a->dim, BK) * BK;
  p.rows_pad = cdiv(a->rows, 128) * 128;
  p.copy_w = !as_is(a, a->w, a->w_row);
  p.copy_x = backward || !as_is(a, a->x, a->x_row);
  const uint32_t all = cdiv(a->vocab, 128) * 128;
  p.piece = backward || p.copy_w ? min(all, 16384u) : all;
  if (p.copy_w) p.w = take(&p, 2ull * p.terms * p.piece * p.dp);
  if (p.copy_x) p.x = take(&p, 2ull * p.terms * p.rows_pad * p.dp);
  if (!backward) {
    p.part = take(&p, 8ull * (all / (32 * Scores::MB)) * a->rows);
    p.hit = take(&p, 4ull * a->rows);
  } else {
    for (uint64_t* q : {&p.idx, &p.pos, &p.weight, &p.lse2, &p.target})
      *q = take(&p, 4ull * p.rows_pad);
    p.count = take(&p, 4);
    p.g = take(&p, 2ull * p.terms * p.rows_pad * p.piece);
    p.sums = take(&p, 4ull * p.rows_pad * p.dp);
  }
  return p;
}

bool bad(const pots_vocab_loss* a) {
  return !a || a->dtype > POTS_OP_BF16 || a->dim == 0 || a->vocab == 0 || a->dim > 65536 ||
         a->rows > (1u << 24) || a->vocab > (1u << 24);
}

template <class T>
int lay(const void* src, int64_t ld, uint32_t d, uint32_t rows, const uint32_t* idx,
        const uint32_t* count, uint16_t* dst, const Plan& p, uint64_t plane, uint32_t rows_pad,
        hipStream_t s) {
  const uint64_t nb = ((uint64_t)rows_pad * (p.dp / 4) + 255) / 256;
  hipLaunchKernelGGL((lay_out<T>), dim3((uint32_t)(nb < 8192 ? nb : 8192)), dim3(256), 0, s,
                     reinterpret_cast<const typename T::elem*>(src), ld, d, rows, idx, count,
                     dst, p.dp, plane, rows_pad);
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}

// The piece's rows of w as an operand, copied into the workspace where they cannot be read as
// they lie (fp32, or rows that are not whole 128-byte stages).
template <class T>
int piece_of_w(const pots_vocab_loss* a, const Plan& p, char* work, uint32_t v0, uint32_t nv,
               Mat* W, hipStream_t s) {
  const typename T::elem* src =
      reinterpret_cast<const typename T::elem*>(a->w) + (int64_t)v0 * a->w_row;
  if (!p.copy_w) {
    *W = Mat{reinterpret_cast<const uint16_t*>(src), a->w_row, 0};
    return POTS_E_OK;
  }
  uint16_t* dst = reinterpret_cast<uint16_t*>(work + p.w);
  *W = Mat{dst, (int64_t)p.dp, (int64_t)p.piece * p.dp};
  return lay<T>(src, a->w_row, a->dim, nv, nullptr, nullptr, dst, p, W->plane, nv, s);
}

template <class T>
int forward(const pots_vocab_loss* a, char* work, hipStream_t s) {
  const Plan p = plan(a, false);
  Mat X = {reinterpret_cast<const uint16_t*>(a->x), a->x_row, 0};
  if (p.copy_x) {
    uint16_t* dst = reinterpret_cast<uint16_t*>(work + p.x);
    X = Mat{dst, (int64_t)p.dp, (int64_t)p.rows_pad * p.dp};
    const int rc = lay<T>(a->x, a->x_row, a->dim, a->rows, nullptr, nullptr, dst, p, X.plane,
                          a->rows, s);
    if (rc) return rc;
  }
  float2* part = reinterpret_cast<float2*>(work + p.part);
  float* hit = reinterpret_cast<float*>(work + p.hit);
  for (uint32_t v0 = 0; v0 < a->vocab; v0 += p.piece) {
    const uint32_t nv = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;
    Mat W;
    const int rc = piece_of_w<T>(a, p, work, v0, nv, &W, s);
    if (rc) return rc;
    const uint32_t mt = cdiv(nv, Scores::TM), nt = cdiv(a->rows, Scores::TN);
    hipLaunchKernelGGL((loss_scores<Scores>), dim3(mt * nt), dim3(Scores::NT), 0, s, W, X, v0,
                       nv, a->rows, p.dp, p.pairs, mt, nt, a->targets, part, a->rows, hit);
    POTS_HIP(hipGetLastError());
  }
  hipLaunchKernelGGL(loss_rows, dim3(cdiv(a->rows, 32)), dim3(1024), 0, s, part, a->rows,
                     cdiv(a->vocab, Scores::TM) * (Scores::TM / (32 * Scores::MB)), hit, *a);
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}

template <class T>
int backward(const pots_vocab_loss* a, char* work, hipStream_t s) {
  const Plan p = plan(a, true);
  auto u32 = [&](uint64_t at) { return reinterpret_cast<uint32_t*>(work + at); };
  auto f32 = [&](uint64_t at) { return reinterpret_cast<float*>(work + at); };
  uint32_t* count = u32(p.count);
  hipLaunchKernelGGL(live_rows, dim3(1), dim3(1024), 0, s, *a, u32(p.idx), u32(p.pos), count,
                     f32(p.weight), f32(p.lse2), u32(p.target));
  POTS_HIP(hipGetLastError());
  uint16_t* xs = reinterpret_cast<uint16_t*>(work + p.x);
  const Mat X = {xs, (int64_t)p.dp, (int64_t)p.rows_pad * p.dp};
  int rc = a->rows == 0 ? POTS_E_OK
                        : lay<T>(a->x, a->x_row, a->dim, a->rows, u32(p.idx), count, xs, p,
                                 X.plane, p.rows_pad, s);
  if (rc) return rc;
  uint16_t* g = reinterpret_cast<uint16_t*>(work + p.g);
  const Mat G = {g, (int64_t)p.piece, (int64_t)p.rows_pad * p.piece};
  const int64_t esize = sizeof(typename T::elem);
  const bool vec = a->dim % 4 == 0 && a->dw_row % 4 == 0 &&
                   reinterpret_cast<uint64_t>(a->dw) % (4 * esize) == 0;
  for (uint32_t v0 = 0; v0 < a->vocab; v0 += p.piece) {
    const uint32_t nv = a->vocab - v0 < p.piece ? a->vocab - v0 : p.piece;
    const uint32_t wmt = cdiv(p.dp, DwTile::TM), wnt = cdiv(nv, DwTile::TN);
    const uint32_t mt = cdiv(nv, Scores::TM), nt = cdiv(a->rows, Scores::TN);
    const uint32_t dmt = cdiv(p.dp, DxTile::TM), dnt = cdiv(a->rows, DxTile::TN);
    if (a->rows) {
    Mat W;
    rc = piece_of_w<T>(a, p, work, v0, nv, &W, s);
    if (rc) return rc;
    hipLaunchKernelGGL((loss_grad<T, Scores>), dim3(mt * nt), dim3(Scores::NT), 0, s, W, X, v0,
                       nv, count, p.dp, p.pairs, mt, nt, f32(p.weight), f32(p.lse2),
                       u32(p.target), g, p.piece, G.plane);
    POTS_HIP(hipGetLastError());
    hipLaunchKernelGGL((loss_dx<DxTile>), dim3(dmt * dnt), dim3(DxTile::NT), 0, s, W, G, p.dp,
                       nv, count, cdiv(nv, BK) * BK, p.pairs, dmt, dnt, f32(p.sums), v0 == 0);
    POTS_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL((loss_dw<T, DwTile>), dim3(wmt * wnt), dim3(DwTile::NT), 0, s, X, G,
                       p.dp, nv, count, p.pairs, wmt, wnt, a->dim,
                       reinterpret_cast<typename T::elem*>(a->dw) + (int64_t)v0 * a->dw_row,
                       a->dw_row, vec);
    POTS_HIP(hipGetLastError());
  }
  if (a->rows == 0) return POTS_E_OK;
  hipLaunchKernelGGL((loss_dx_rows<T>), dim3(a->rows), dim3(256), 0, s, f32(p.sums), p.dp,
                     u32(p.pos), a->dim, reinterpret_cast<typename T::elem*>(a->dx), a->dx_row);
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}

}  // namespace

}  // namespace pots

using namespace pots;

extern "C" uint64_t pots_vocab_loss_forward_work(const pots_vocab_loss* a) {
  return bad(a) || a->rows == 0 ? 0 : plan(a, false).bytes;
}

extern "C" int pots_vocab_loss_forward(const pots_vocab_loss* a, void* work, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (a->rows == 0) return POTS_E_OK;
  if (!a->x || !a->w || !a->targets || !a->loss || !a->lse || !work) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* w = static_cast<char*>(work);
  return a->dtype == POTS_OP_BF16 ? forward<Bf16>(a, w, s) : forward<Fp32>(a, w, s);
}

extern "C" uint64_t pots_vocab_loss_backward_work(const pots_vocab_loss* a) {
  return bad(a) ? 0 : plan(a, true).bytes;
}

extern "C" int pots_vocab_loss_backward(const pots_vocab_loss* a, void* work, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (!a->w || !a->dw || !work) return POTS_E_ARG;
  if (a->rows && (!a->x || !a->targets || !a->lse || !a->weights || !a->dx)) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* w = static_cast<char*>(work);
  return a->dtype == POTS_OP_BF16 ? backward<Bf16>(a, w, s) : backward<Fp32>(a, w, s);
}
