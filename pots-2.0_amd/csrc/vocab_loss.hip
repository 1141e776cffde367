// Softmax cross entropy of feature rows against a vocabulary matrix, with its gradient, for
// passes that keep no logits.
//
//   s_rv = x_r·w_v,  lse_r = log Σ_v e^{s_rv},  loss_r = lse_r − s_{r,t_r}
//   g_rv = weight_r (e^{s_rv − lse_r} − [v = t_r]),  dx = G·W,  dW = Gᵀ·X
//
// Forward: a tile of S is a product whose epilogue leaves a maximum and a sum of exponentials per
// row of x; loss_rows joins the tiles. Backward, in pieces of the vocabulary: S again with the
// epilogue that writes the piece of G (1.1 PFLOP/s without its writes, 0.9 with them), then that
// piece's rows of dW, and its share of dx added to fp32 sums (1.0 PFLOP/s together). Rows that
// carry no weight are left out of the products first (live_rows: prompts, rows without a target),
// and so is whatever they hold.
//
// All three products are one tiled kernel over the matrix cores (Tile), each operand stored
// either with the contraction along its rows or with its rows along the contraction (W of dx,
// G and X of dW); the latter are read transposed from LDS. bf16 is multiplied as it is. An fp32
// value is the exact sum of three bf16 terms (take_term), the second at most 2^-8 and the third 2^-16
// of it. A product of two takes the six products of terms above 2^-24 of it; the three left out are
// together below 2^-23. At six bf16 products' cost that is 1.3 times as fast as the library's
// fp32 product (154 TFLOP/s); few rows forward are multiplied as fp32. (An infinite value meets zero
// terms: its rows' scores are NaN, not infinite, where they are made of terms.) G is rounded to the inputs'
// type as an operand: half a step of bf16, 2^-8, of each term of sums that are rounded to bf16
// themselves.
//
// Bound by the matrix cores and what feeds them: a block's 256 x 256 tile needs 64 KiB a stage of 64,
// and the loads alone (multiplications taken out, in a copy) take four fifths of the time;
// multiplications alone two thirds. 8192 rows of 1536 against 151936 in bf16: 3.4 ms, 1.14 PFLOP/s,
// of which exponentials and sums are about a tenth (the library's product without them:
// 3.1 ms). What did not help: four stages of 32 (3.7 ms), four waves of 128 x 128 (4.0), one
// operand past the LDS in fragments (3.7), loads issued later in a stage (3 to 7 % slower).
#include <math.h>

#include <type_traits>

#include "common.h"
#include "gmem.h"
#include "tiles.h"

namespace pots {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

constexpr uint32_t BK = 64;  // contraction per stage, 128 bytes of a row; lengths are padded to it

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
// row by the row's number, so that the reads of a fragment fall on different banks: 16 lanes'
// 16-byte reads of 16 rows, or 32 lanes' transposing reads of four rows (64 banks of four bytes). A lane's
// offsets are the same at every stage; the stage moves the buffer's base, in scalar registers.
template <bool TR, uint32_t T, uint32_t NT>
struct Stage {
  static constexpr uint32_t kAll = T * BK / 8, kChunks = (kAll + NT - 1) / NT;
  static_assert(kAll % 64 == 0 && (kAll % NT == 0 || NT % kAll == 0), "whole waves' loads");
  static_assert(!TR || (T % 64 == 0 && T > 64), "the exchange stays within a transposed row");
  uint32_t off[kChunks], wide;

  // What row r's chunks are exchanged by.
  static __device__ __forceinline__ uint32_t swap(uint32_t r) {
    return !TR ? (r >> 1) & 7 : T % 128 == 0 ? 4 * (r & 3) : 2 * (r & 2);
  }

  // r0, rows: the tile's first row and their number; rows past it repeat the last (for TR:
  // columns, whose last eight repeat).
  __device__ __forceinline__ void init(const Mat& m, uint32_t r0, uint32_t rows) {
    wide = 2 * min(T, rows - r0);
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++) {
      // (a tile of less than a load for each wave is loaded by several, so that all wait alike)
      const uint32_t c = (u * NT + threadIdx.x) % kAll;
      if constexpr (TR) {
        const uint32_t r = c / (T / 8), at = (c % (T / 8)) ^ swap(r);
        off[u] = 2 * (r * (uint32_t)m.ld + min(r0 + 8 * at, rows - 8) - r0);
      } else {
        const uint32_t r = c / (BK / 8), at = (c % (BK / 8)) ^ swap(r);
        off[u] = 2 * (min(r, rows - 1 - r0) * (uint32_t)m.ld + 8 * at);
      }
    }
  }

  // The stage of contraction k0 .. k0 + BK; for TR, zero from `ks` on. Not `on`: zeros, and no
  // memory is read.
  __device__ __forceinline__ void load(uint16_t* lds, const Mat& m, uint32_t plane, uint32_t r0,
                                       uint32_t k0, uint32_t ks, bool on) const {
    const uint16_t* base = m.p + (int64_t)plane * m.plane +
                           (TR ? (int64_t)k0 * m.ld + r0 : (int64_t)r0 * m.ld + k0);
    const uint32_t range =
        TR ? (min(BK, ks - k0) - 1) * (uint32_t)m.ld * 2 + wide : 0x7FFFFFFF;
    const brsrc rsrc = make_rsrc(base, on ? range : 0);
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++)
      load_lds16(rsrc, lds + (u * NT + wave * 64) % kAll * 8, off[u]);
  }

  // Rows c .. c + 31 at step ks of the stage: contraction 16ks + 8h + (0..7).
  static __device__ __forceinline__ void read(const uint16_t* lds, uint32_t c, uint32_t ks,
                                              uint32_t lane, bf16x8* f) {
    const uint32_t h = lane / 32;
    if constexpr (TR) {
      const uint32_t m = lane % 16, r = 16 * ks + 8 * h + m / 4;
      const uint32_t col = c + (lane & 16) + 4 * (m % 4);
      const uint16_t* p = lds + r * T + (((col / 8) ^ swap(m / 4)) * 8 + 4 * (m % 2));
      *f = join(read_tr(p), read_tr(p + 4 * T));
    } else {
      const uint32_t r = c + lane % 32;
      *f = *reinterpret_cast<const bf16x8*>(lds + r * BK + (((2 * ks + h) ^ swap(lane % 32)) * 8));
    }
  }
  // The same of a stage of fp32 rows, two of its chunks.
  static __device__ __forceinline__ void read(const uint16_t* lds, uint32_t c, uint32_t ks,
                                              uint32_t lane, f32x8* f) {
    const uint16_t* row = lds + (c + lane % 32) * BK;
    const uint32_t at = 4 * ks + 2 * (lane / 32), by = swap(lane % 32);
    *f = __builtin_shufflevector(*reinterpret_cast<const f32x4*>(row + (at ^ by) * 8),
                                 *reinterpret_cast<const f32x4*>(row + ((at + 1) ^ by) * 8), 0, 1,
                                 2, 3, 4, 5, 6, 7);
  }
};

// The stages in LDS: objects of their own, so that the compiler knows a load into one from the
// reads of another and need not wait for it; one set for all the products of a kernel.
template <uint32_t WHICH, uint32_t SIZE>
__device__ __forceinline__ uint16_t* lds_buffer() {
  __shared__ __attribute__((aligned(16))) uint16_t s_buf[SIZE];
  return s_buf;
}

// A block's TM x TN of A·Bᵀ over K (a multiple of BK), WM x WN waves of MB x NB products of 32.
// NBUF stages in LDS: NBUF - 1 are on their way while one is multiplied.
// F32: the operands are fp32, as stored, of twice the length and the distance in Mat's units, and go
// through the fp32 matrix instructions.
template <bool ATR, bool BTR, uint32_t TM_, uint32_t TN_, uint32_t WM_, uint32_t WN_,
          uint32_t NBUF, bool F32 = false>
struct Tile {
  static_assert(!F32 || (!ATR && !BTR), "no transposing reads of fp32");
  typedef std::conditional_t<F32, f32x8, bf16x8> frag;
  static constexpr uint32_t TM = TM_, TN = TN_, WM = WM_, WN = WN_, NT = 64 * WM * WN;
  static constexpr uint32_t MB = TM / WM / 32, NB = TN / WN / 32;
  typedef Stage<ATR, TM, NT> SA;
  typedef Stage<BTR, TN, NT> SB;
  f32x16 acc[MB][NB];
  uint32_t wm, wn, lane;

  __device__ __forceinline__ void step(const uint16_t* a, const uint16_t* b) {
#pragma unroll
    for (uint32_t ks = 0; ks < BK / (F32 ? 32 : 16); ks++) {
      frag fa[MB], fb[NB];
#pragma unroll
      for (uint32_t m = 0; m < MB; m++) SA::read(a, wm + 32 * m, ks, lane, &fa[m]);
#pragma unroll
      for (uint32_t n = 0; n < NB; n++) SB::read(b, wn + 32 * n, ks, lane, &fb[n]);
#pragma unroll
      for (uint32_t m = 0; m < MB; m++)
#pragma unroll
        for (uint32_t n = 0; n < NB; n++) acc[m][n] = mma(fa[m], fb[n], acc[m][n]);
    }
  }

  // The contraction is k0 .. k0 + K; ka, kb: its end where an operand is stored along it.
  __device__ __forceinline__ void run(const Mat& A, const Mat& B, uint32_t m0, uint32_t M,
                                      uint32_t n0, uint32_t N, uint32_t k0, uint32_t K,
                                      uint32_t ka, uint32_t kb, uint32_t pairs) {
    uint16_t* const s_a[4] = {lds_buffer<0, TM * BK>(), lds_buffer<1, TM * BK>(),
                              lds_buffer<NBUF == 4 ? 2 : 0, TM * BK>(),
                              lds_buffer<NBUF == 4 ? 3 : 1, TM * BK>()};
    uint16_t* const s_b[4] = {lds_buffer<4, TN * BK>(), lds_buffer<5, TN * BK>(),
                              lds_buffer<NBUF == 4 ? 6 : 4, TN * BK>(),
                              lds_buffer<NBUF == 4 ? 7 : 5, TN * BK>()};
    lane = threadIdx.x % 64;
    wm = threadIdx.x / 64 / WN * (TM / WM);
    wn = threadIdx.x / 64 % WN * (TN / WN);
#pragma unroll
    for (uint32_t m = 0; m < MB; m++)
#pragma unroll
      for (uint32_t n = 0; n < NB; n++) acc[m][n] = zero16();
    const uint32_t steps = K / BK * pairs;
    uint32_t k = k0, pair = 0, ahead = 0;
    SA sa;
    SB sb;
    sa.init(A, m0, M);
    sb.init(B, n0, N);
    auto load = [&](uint32_t j) {  // the next stage; past the last, nothing
      const bool on = ahead < steps;
      uint32_t pa, pb;
      pair_of(pairs, on ? pair : 0, &pa, &pb);
      sa.load(s_a[j], A, pa, m0, k, ka, on);
      sb.load(s_b[j], B, pb, n0, k, kb, on);
      ahead++;
      k += BK;
      if (k == k0 + K) {
        k = k0;
        pair++;
      }
    };
#pragma unroll
    for (uint32_t j = 0; j + 1 < NBUF; j++) load(j);
    constexpr uint32_t kLeft = (NBUF - 2) * (SA::kChunks + SB::kChunks);  // of later stages
    for (uint32_t t = 0; t < steps; t += NBUF) {
#pragma unroll
      for (uint32_t j = 0; j < NBUF; j++) {
        loads_done<kLeft>();
        if (NBUF > 2 || ahead < steps) load((j + NBUF - 1) % NBUF);
        if (t + j < steps) step(s_a[j], s_b[j]);
      }
    }
    loads_done();
  }

  // A part of A's stages for each wave to itself, after run().
  static constexpr uint32_t kScratch = TM * BK * 2 / (WM_ * WN_);  // values
  __device__ __forceinline__ uint16_t* scratch() const {
    constexpr uint32_t half = WM * WN / 2;
    const uint32_t w = threadIdx.x / 64, in = w % half * kScratch;
    return w < half ? lds_buffer<0, TM * BK>() + in : lds_buffer<1, TM * BK>() + in;
  }

  // f(acc, row of A of register 0 of the lane, row of B of the lane)
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
__device__ __forceinline__ void tile_of(uint32_t block, uint32_t mt, uint32_t nt, uint32_t* m,
                                        uint32_t* n) {
  const uint32_t u = xcd_block(block, mt * nt), g = u / (8 * mt), in = u % (8 * mt);
  const uint32_t w = min(8u, nt - 8 * g);
  *m = in / w;
  *n = 8 * g + in % w;
}

// ---- laying operands out --------------------------------------------------------------------

// x to eight bits as bf16 (to nearest; down where that would be infinite); x is left with the
// rest, exactly, at most 2^-8 of it.
__device__ __forceinline__ uint16_t take_term(float* x) {
  const uint32_t u = __float_as_uint(*x);
  if ((u & 0x7F800000u) == 0x7F800000u) {  // one term; a NaN keeps a bit of its fraction
    *x = 0.f;
    return (u >> 16) | ((u & 0x7FFFFFu) ? 0x40 : 0);
  }
  uint16_t t = f32_to_bf16(*x);
  if ((t & 0x7F80u) == 0x7F80u) t = u >> 16;
  *x = *x - bf16_to_f32(t);
  return t;
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
          if constexpr (kTerms == 3) {
            float x = p[c + j];
#pragma unroll
            for (uint32_t k = 0; k < 3; k++) t[j][k] = take_term(&x);
          } else {
            t[j][0] = p[c + j];
          }
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
// their weights, targets and lse (in units of log2) gathered. G is held in units of the largest
// weight, `unit`, which its products are multiplied by at the end: rows that weigh the same (a
// mean over the batch) then have a weight of 1, which rounds no entry of G.
__global__ __launch_bounds__(1024) void live_rows(pots_vocab_loss a, uint32_t* __restrict__ idx,
                                                  uint32_t* __restrict__ pos,
                                                  uint32_t* __restrict__ count,
                                                  float* __restrict__ weight,
                                                  float* __restrict__ lse2,
                                                  uint32_t* __restrict__ target,
                                                  float* __restrict__ unit) {
  __shared__ uint32_t s_wave[16];
  __shared__ float s_top[16];
  uint32_t base = 0;
  const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  float top = 0.f;
  for (uint32_t r = threadIdx.x; r < a.rows; r += 1024) top = fmaxf(top, fabsf(a.weights[r]));
  for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o));
  if (lane == 0) s_top[wave] = top;
  __syncthreads();
  for (uint32_t v = 0; v < 16; v++) top = fmaxf(top, s_top[v]);
  if (!(top >= 0x1p-100f && top <= 0x1p100f)) top = 1.f;
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
      weight[at] = t < a.vocab ? w / top : NAN;
      lse2[at] = a.lse[r] * kLog2e;
      target[at] = (uint32_t)t;
    }
    base += all;
  }
  if (threadIdx.x == 0) {
    *count = base;
    *unit = top;
  }
}

// ---- the products ---------------------------------------------------------------------------

// A piece of the vocabulary from v0 on, `nv` rows of it, against rows of x: a maximum (times
// log2 e) and a sum of 2^(s - maximum) per row and tile, part[chunk][row], and the targets' s.
template <class C>
__global__ __launch_bounds__(C::NT) void loss_scores(Mat W, Mat X, uint32_t v0, uint32_t nv,
                                                     uint32_t rows, uint32_t K, uint32_t pairs,
                                                     uint32_t mt, uint32_t nt,
                                                     const int64_t* __restrict__ targets,
                                                     float2* __restrict__ part,
                                                     float* __restrict__ hit) {
  __shared__ float2 s_part[C::WM][C::TN];
  uint32_t m, n;
  tile_of(blockIdx.x, mt, nt, &m, &n);
  C c;
  const uint32_t m0 = m * C::TM, n0 = n * C::TN;
  c.run(W, X, m0, nv, n0, rows, 0, K, 0, 0, pairs);
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
    if (c.lane < 32)
      s_part[c.wm / (C::TM / C::WM)][c.wn + 32 * b + c.lane] =
          make_float2(top == -INFINITY ? -INFINITY : tc, sum);
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
  __syncthreads();
  for (uint32_t x = threadIdx.x; x < C::TN && n0 + x < rows; x += C::NT) {
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < C::WM; w++) top = fmaxf(top, s_part[w][x].x);
#pragma unroll
    for (uint32_t w = 0; w < C::WM; w++)
      sum += s_part[w][x].y *
             __builtin_amdgcn_exp2f(s_part[w][x].x == top ? 0.f : s_part[w][x].x - top);
    part[(uint64_t)(v0 / C::TM + m) * rows + n0 + x] = make_float2(top, sum);
  }
}

// RB rows a block, the chunks over 1024 / RB groups of lanes, joined in a fixed order.
template <uint32_t RB>
__global__ __launch_bounds__(1024) void loss_rows(const float2* __restrict__ part,
                                                  uint32_t chunks,
                                                  const float* __restrict__ hit,
                                                  pots_vocab_loss a) {
  constexpr uint32_t G = 1024 / RB;
  __shared__ float2 s_part[G][RB + 1];
  const uint32_t i = threadIdx.x % RB, g = threadIdx.x / RB, row = blockIdx.x * RB + i;
  float m = -INFINITY, l = 0.f;
  auto join = [&](float2 p) {
    const float top = fmaxf(m, p.x);
    if (top == -INFINITY) {  // no finite score yet; a NaN among them stays in the sum
      l += p.y;
      return;
    }
    l = l * __builtin_amdgcn_exp2f(m - top) + p.y * __builtin_amdgcn_exp2f(p.x - top);
    m = top;
  };
  if (row < a.rows)
    for (uint32_t c = g; c < chunks; c += G) join(part[(uint64_t)c * a.rows + row]);
  for (uint32_t half = G / 2; half > 0; half /= 2) {
    s_part[g][i] = make_float2(m, l);
    __syncthreads();
    if (g < half) join(s_part[g + half][i]);
    __syncthreads();
  }
  if (g != 0 || row >= a.rows) return;
  const float lse = (m + __builtin_amdgcn_logf(l)) * kLn2;
  const int64_t t = a.targets[row];
  a.lse[row] = lse;
  a.loss[row] = t < 0 ? 0.f : t < a.vocab ? lse - hit[row] : NAN;
}

// The piece's G in units of the largest weight, [terms][live rows][ld], zero past the live rows
// and the vocabulary. A lane's results are four vocabulary rows at a time of a row of G; they
// are gathered in LDS to whole 256-byte spans.
template <class T, class C>
__global__ __launch_bounds__(C::NT) void loss_grad(Mat W, Mat X, uint32_t v0, uint32_t nv,
                                                   const uint32_t* __restrict__ count,
                                                   uint32_t K, uint32_t pairs, uint32_t mt,
                                                   const float* __restrict__ weight,
                                                   const float* __restrict__ lse2,
                                                   const uint32_t* __restrict__ target,
                                                   uint16_t* __restrict__ g, uint32_t ld,
                                                   uint64_t plane) {
  uint32_t m, n;
  const uint32_t live = gload<uint32_t>(count), nt = (live + C::TN - 1) / C::TN;
  if (blockIdx.x >= mt * nt) return;
  tile_of(blockIdx.x, mt, nt, &m, &n);
  const uint32_t m0 = m * C::TM, n0 = n * C::TN;
  C c;
  c.run(W, X, m0, nv, n0, live, 0, K, 0, 0, pairs);
  constexpr uint32_t kTerms = sizeof(typename T::elem) == 4 ? 3 : 1;
  constexpr uint32_t CW = 4 * C::MB;  // 16-byte chunks of a wave's row of G
  static_assert(CW * 8 * 32 <= C::kScratch, "a wave's 32 rows fit");
  uint16_t* const s = c.scratch();
  const uint32_t i = c.lane % 32, h = c.lane / 32;
#pragma unroll
  for (uint32_t b = 0; b < C::NB; b++) {
    const uint32_t row = n0 + c.wn + 32 * b + i;
    const bool on = row < live;
    const float w = on ? weight[row] : 0.f, l2 = on ? lse2[row] : 0.f;
    const uint32_t t = on ? target[row] - v0 - m0 - c.wm : ~0u;
    const uint32_t left = on && nv > m0 + c.wm ? nv - m0 - c.wm : 0;
#pragma unroll
    for (uint32_t x = 0; x < C::MB; x++)
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) {
        const uint32_t at = 32 * x + d_row(r, h);
        const float p =
            __builtin_amdgcn_exp2f(__builtin_fmaf(c.acc[x][b][r], kLog2e, -l2));
        c.acc[x][b][r] = at < left ? w * (at == t ? p - 1.f : p) : 0.f;
      }
#pragma unroll
    for (uint32_t k = 0; k < kTerms; k++) {
#pragma unroll
      for (uint32_t x = 0; x < C::MB; x++)
#pragma unroll
        for (uint32_t q = 0; q < 4; q++) {
          uint16_t e[4];
#pragma unroll
          for (uint32_t y = 0; y < 4; y++) {
            if constexpr (kTerms == 3) {
              float v = c.acc[x][b][4 * q + y];
              e[y] = take_term(&v);
              c.acc[x][b][4 * q + y] = v;
            } else {
              e[y] = f32_to_bf16(c.acc[x][b][4 * q + y]);
            }
          }
          const u32x2v o = {(uint32_t)e[0] | (uint32_t)e[1] << 16,
                            (uint32_t)e[2] | (uint32_t)e[3] << 16};
          *reinterpret_cast<u32x2v*>(s + i * 8 * CW + ((4 * x + q) ^ (i % CW)) * 8 + 4 * h) = o;
        }
      // (a wave's own LDS: its writes and reads are in order)
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (uint32_t y = 0; y < CW / 2; y++) {
        const uint32_t r = (c.lane + 64 * y) / CW, ch = c.lane % CW;
        const u32x4v o = *reinterpret_cast<const u32x4v*>(s + r * 8 * CW + (ch ^ (r % CW)) * 8);
        gstore<u32x4v>(g + k * plane + (uint64_t)(n0 + c.wn + 32 * b + r) * ld + m0 + c.wm +
                           8 * ch,
                       o);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  }
}

// Both products of a piece of G in one launch, so that the tiles of one fill the GPU's places
// beside the other's. Blocks below mt·nt·splits: a share of dx, Wᵀ (stored along the
// contraction, the piece's vocabulary) by G, added to the split's sums [rows][dp]. The others:
// the piece's rows of dW, Xᵀ by Gᵀ, both stored along the contraction (the live rows), or a
// share of their contraction to sums of its own where there are few tiles (or dW's rows are not
// whole fours of values).
template <class T, class CX, class CW>
__global__ __launch_bounds__(CX::NT) void loss_products(
    Mat W, Mat X, Mat G, uint32_t dp, uint32_t nv, const uint32_t* __restrict__ count,
    const float* __restrict__ unit, uint32_t pairs, uint32_t mt, uint32_t splits,
    uint32_t per, float* __restrict__ sums, uint64_t slice, bool first, uint32_t wmt,
    uint32_t wnt, uint32_t wsplits, uint32_t wper, float* __restrict__ wsums, uint64_t wslice,
    uint32_t d, typename T::elem* __restrict__ dw, int64_t ld) {
  // (the tiles of the live rows alone, dealt over all XCDs; the launch has room for every row)
  const uint32_t live = gload<uint32_t>(count), nt = (live + CX::TN - 1) / CX::TN;
  uint32_t m, n;
  if (blockIdx.x < mt * nt * splits) {
    const uint32_t split = blockIdx.x / (mt * nt);
    tile_of(blockIdx.x % (mt * nt), mt, nt, &m, &n);
    const uint32_t m0 = m * CX::TM, n0 = n * CX::TN, k0 = split * per;
    CX c;
    const uint32_t all = (nv + BK - 1) / BK * BK;
    c.run(W, G, m0, dp, n0, live, k0, k0 < all ? min(per, all - k0) : 0, nv, 0, pairs);
    float* out = sums + split * slice;
    c.each(m0, n0, [&](f32x16& s, uint32_t col, uint32_t row) {
      if (row >= live) return;
#pragma unroll
      for (uint32_t q = 0; q < 4; q++) {
        if (col + 8 * q >= dp) continue;
        f32x4* p = reinterpret_cast<f32x4*>(out + (uint64_t)row * dp + col + 8 * q);
        f32x4 y = {s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
        if (!first) y += *p;
        *p = y;
      }
    });
    return;
  }
  const uint32_t unit_w = blockIdx.x - mt * nt * splits;
  if (unit_w >= wmt * wnt * wsplits) return;
  tile_of(unit_w % (wmt * wnt), wmt, wnt, &m, &n);
  const uint32_t m0 = m * CW::TM, n0 = n * CW::TN, all = (live + BK - 1) / BK * BK;
  const uint32_t wsplit = unit_w / (wmt * wnt), k0 = wsplit * wper;
  CW c;
  c.run(X, G, m0, dp, n0, (nv + 7) & ~7u, k0, k0 < all ? min(wper, all - k0) : 0, live, live,
        pairs);
  if (wsums) {
    float* out = wsums + wsplit * wslice;
    c.each(m0, n0, [&](f32x16& s, uint32_t col, uint32_t v) {
      if (v >= nv) return;
#pragma unroll
      for (uint32_t q = 0; q < 4; q++) {
        const f32x4 y = {s[4 * q], s[4 * q + 1], s[4 * q + 2], s[4 * q + 3]};
        if (col + 8 * q < dp) *reinterpret_cast<f32x4*>(out + (uint64_t)v * dp + col + 8 * q) = y;
      }
    });
    return;
  }
  const float mul = *unit;
  c.each(m0, n0, [&](f32x16& s, uint32_t col, uint32_t v) {
    if (v >= nv) return;
    typename T::elem* p = dw + (int64_t)v * ld;
#pragma unroll
    for (uint32_t q = 0; q < 4; q++) {
      const uint32_t at = col + 8 * q;
      if (at < d)
        T::store4(p + at, s[4 * q] * mul, s[4 * q + 1] * mul, s[4 * q + 2] * mul,
                  s[4 * q + 3] * mul);
    }
  });
}

// Rows of dx or dW from the shares' sums, a block a row (two where 2^24 rows would be 2^32 threads):
// row pos[r] of them (r without pos), zero for the rows left out.
template <class T>
__global__ __launch_bounds__(256) void loss_join(const float* __restrict__ sums, uint32_t dp,
                                                 uint32_t splits, uint64_t slice,
                                                 const uint32_t* __restrict__ pos,
                                                 const float* __restrict__ unit, uint32_t d,
                                                 typename T::elem* __restrict__ out, int64_t ld,
                                                 uint32_t rows) {
  const float mul = *unit;
  for (uint32_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const uint32_t at = pos ? pos[row] : row;
    typename T::elem* const to = out + (int64_t)row * ld;
    for (uint32_t c = threadIdx.x * 4; c < d; c += 1024) {
      f32x4 y = {0.f, 0.f, 0.f, 0.f};
      if (at != ~0u)
        for (uint32_t s = 0; s < splits; s++)
          y += gload<f32x4>(sums + s * slice + (uint64_t)at * dp + c);
#pragma unroll
      for (uint32_t x = 0; x < 4; x++)
        if (c + x < d) to[c + x] = T::put(y[x] * mul);
    }
  }
}

namespace {

// Tiles. Large ones read each operand half as often, where there are enough of them for the GPU
// (8192 rows of 1536: 3.4 ms, 4.0 in medium ones); up to 32 rows the product is bound by reading W,
// and a tile as narrow as the rows leaves its multiplications out of the way (seven rows of 896
// against 151936: 51 us, 5.3 TB/s).
template <bool ATR, bool BTR>
using Large = Tile<ATR, BTR, 256, 256, 2, 4, 2>;
template <bool ATR, bool BTR>
using Trimmed = Tile<ATR, BTR, 192, 256, 2, 4, 2>;  // products' rows of 576 or 896 columns, say
template <bool ATR, bool BTR>
using Medium = Tile<ATR, BTR, 128, 128, 2, 2, 2>;
template <bool ATR, bool BTR>
using Narrow = Tile<ATR, BTR, 256, 32, 8, 1, 4>;
template <bool ATR, bool BTR>
using NarrowX = Tile<ATR, BTR, 256, 32, 8, 1, 2>;  // beside Large in one kernel's LDS
// fp32 rows as they are, through the fp32 matrix instructions: see kDirectRows. Tiles of 128 rows
// of w, three blocks to a compute unit, against 256 and one: 96 rows 226 us and 268, 512 753 and 763.
using Direct = Tile<false, false, 128, 64, 4, 1, 2, true>;
using NarrowDirect = Tile<false, false, 256, 32, 8, 1, 4, true>;
enum Shape { kLarge, kTrimmed, kMedium, kNarrow };

constexpr uint32_t kCus = 256;
constexpr uint32_t kMostJoined = 1u << 23;  // blocks of loss_join

uint32_t cdiv(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

Shape scores_shape(uint32_t rows, uint32_t piece) {
  if (rows <= 32) return kNarrow;
  return rows > 128 && (uint64_t)cdiv(rows, 256) * cdiv(piece, 256) >= kCus ? kLarge : kMedium;
}

// Sizes and the workspace's parts.
struct Plan {
  uint32_t dp, terms, pairs, rows_pad, piece;
  Shape scores, products;
  uint32_t splits, per, wsplits, wper;  // shares of dx's and of dW's contractions
  bool copy_w, copy_x, join_w, direct;
  uint64_t w, x, part, hit, idx, pos, count, unit, weight, lse2, target, g, sums, wsums, bytes;
};

uint64_t take(Plan* p, uint64_t bytes) {
  const uint64_t at = p->bytes;
  p->bytes += align_up(bytes, 256);
  return at;
}

// Whether a matrix can be read where it lies: whole stages on 16-byte borders, and a tile of 256 of
// its rows within 31 bits of offset.
bool lies_well(const pots_vocab_loss* a, const void* p, int64_t row) {
  const int64_t size = a->dtype == POTS_OP_BF16 ? 2 : 4;
  return size * a->dim % (2 * BK) == 0 && reinterpret_cast<uint64_t>(p) % 16 == 0 &&
         row * size % 16 == 0 && row >= 0 && row * size < 1 << 23;
}
bool as_is(const pots_vocab_loss* a, const void* p, int64_t row) {
  return a->dtype == POTS_OP_BF16 && lies_well(a, p, row);
}

// Up to so many fp32 rows the forward pass reads operands where they lie and multiplies with the
// fp32 instructions: laying w out as three terms and reading them for six products costs more than
// the slower multiplications. us at 2048 columns against 46432, laid out and where they lie: 40 rows
// 604 and 148, 96 rows 596 and 226, 210 rows 634 and 412, 512 rows 925 and 753, 769 and
// 768 rows 1345 and 1105; at 576 against 49152: 133 and 48, 135 and 69, 167 and 121, 243 and 222,
// 349 and 325; 1024 rows laid out, 1374 and 357, are where the fp32 instructions would be slower.
// Up to 32 rows bound by reading w (three rows 89 us, 4.3 TB/s), then by the fp32 instructions
// (256 rows: 117 TFLOP/s).
constexpr uint32_t kDirectRows = 768;

Plan plan(const pots_vocab_loss* a, bool backward) {
  constexpr uint64_t kRoom = 512ull << 20;  // bytes of a piece of G, and of a copied one of W
  Plan p = {};
  p.terms = a->dtype == POTS_OP_BF16 ? 1 : 3;
  p.pairs = a->dtype == POTS_OP_BF16 ? 1 : 6;
  p.dp = cdiv(a->dim, BK) * BK;
  p.rows_pad = cdiv(a->rows, 256) * 256;
  p.direct = !backward && a->dtype == POTS_OP_F32 && a->rows <= kDirectRows &&
             lies_well(a, a->w, a->w_row) && lies_well(a, a->x, a->x_row);
  if (p.direct) p.dp = 2 * a->dim, p.terms = p.pairs = 1;  // in units of two bytes
  p.copy_w = !p.direct && !as_is(a, a->w, a->w_row);
  p.copy_x = !p.direct && (backward || !as_is(a, a->x, a->x_row));
  const uint32_t all = cdiv(a->vocab, 256) * 256;
  uint64_t most = all;
  if (p.copy_w) most = min(most, kRoom / (2ull * p.terms * p.dp));
  if (backward && a->rows) most = min(most, kRoom / (2ull * p.terms * p.rows_pad));
  most = max(most, (uint64_t)2048);
  // (a launch has less than 2^32 threads: 2^22 large tiles are half of them)
  most = min(most, 256ull * max((1u << 22) / max(p.rows_pad / 256, 1u), 1u));
  const uint32_t pieces = (uint32_t)((all + most - 1) / most);
  p.piece = cdiv(cdiv(all, pieces), 256) * 256;
  p.scores = p.direct && a->rows > 32 ? kMedium : scores_shape(a->rows, p.piece);
  if (p.copy_w) p.w = take(&p, 2ull * p.terms * p.piece * p.dp);
  if (p.copy_x) p.x = take(&p, 2ull * p.terms * p.rows_pad * p.dp);
  if (!backward) {
    p.part = take(&p, 8ull * (all / 128) * a->rows);
    p.hit = take(&p, 4ull * a->rows);
    return p;
  }
  for (uint64_t* q : {&p.idx, &p.pos, &p.weight, &p.lse2, &p.target})
    *q = take(&p, 4ull * p.rows_pad);
  p.count = take(&p, 4);
  p.unit = take(&p, 4);
  p.g = take(&p, 2ull * p.terms * p.rows_pad * p.piece);
  // Shares of dx's contraction about as long as dW's, so that the launch's blocks are alike, and
  // shorter ones where the GPU would not be full; each share has sums of its own.
  p.products = p.scores;
  if (p.products == kLarge && cdiv(p.dp, 192) * 192 < cdiv(p.dp, 256) * 256)
    p.products = kTrimmed;  // fewer columns past the end
  const uint32_t tn = p.products == kNarrow ? 32 : p.products == kMedium ? 128 : 256;
  const uint32_t tm = p.products == kTrimmed ? 192 : p.products == kMedium ? 128 : 256;
  const uint32_t k_dx = p.piece / BK, k_dw = cdiv(a->rows, BK);
  const uint32_t most_splits = p.products == kNarrow ? 64 : 16;
  const uint32_t dx_tiles = cdiv(p.dp, tm) * cdiv(a->rows, tn);
  const uint32_t dw_tiles = cdiv(p.dp, tm) * cdiv(p.piece, p.products == kMedium ? 128 : 256);
  p.splits = k_dw ? min(max((k_dx + k_dw / 2) / k_dw, 1u), 16u) : 1;
  while (p.splits < most_splits && dx_tiles * p.splits + dw_tiles < 2 * kCus &&
         k_dx * p.pairs / p.splits > 8)
    p.splits++;
  p.per = cdiv(k_dx, p.splits) * BK;
  p.splits = cdiv(p.piece, p.per);
  p.sums = take(&p, 4ull * p.splits * p.rows_pad * p.dp);
  // dW's contraction in shares too, where its few tiles would be the launch's long end
  p.wsplits = 1;
  while (p.wsplits < 16 && dx_tiles * p.splits + dw_tiles * p.wsplits < kCus &&
         k_dw * p.pairs / p.wsplits > 8)
    p.wsplits *= 2;
  p.wper = cdiv(max(k_dw, 1u), p.wsplits) * BK;
  p.wsplits = max(cdiv(k_dw * BK, p.wper), 1u);
  const uint64_t esize = a->dtype == POTS_OP_BF16 ? 2 : 4;
  p.join_w = p.wsplits > 1 || a->dim % 4 || a->dw_row % 4 ||
             reinterpret_cast<uint64_t>(a->dw) % (4 * esize);
  if (p.join_w) p.wsums = take(&p, 4ull * p.wsplits * p.piece * p.dp);
  return p;
}

bool bad(const pots_vocab_loss* a) {
  return !a || a->dtype > POTS_OP_BF16 || a->dim == 0 || a->vocab == 0 || a->dim > 65536 ||
         a->rows > (1u << 24) || a->vocab > (1u << 24) ||
         (uint64_t)cdiv(a->rows, 32) * cdiv(a->vocab, 128) > 0x7FFFFFFFu;
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
    *W = Mat{reinterpret_cast<const uint16_t*>(src), a->w_row * (int64_t)(sizeof(*src) / 2), 0};
    return POTS_E_OK;
  }
  uint16_t* dst = reinterpret_cast<uint16_t*>(work + p.w);
  *W = Mat{dst, (int64_t)p.dp, (int64_t)p.piece * p.dp};
  return lay<T>(src, a->w_row, a->dim, nv, nullptr, nullptr, dst, p, W->plane, nv, s);
}

template <class C>
int scores(const pots_vocab_loss* a, const Plan& p, const Mat& W, const Mat& X, uint32_t v0,
           uint32_t nv, char* work, hipStream_t s) {
  const uint32_t mt = cdiv(nv, C::TM), nt = cdiv(a->rows, C::TN);
  hipLaunchKernelGGL((loss_scores<C>), dim3(mt * nt), dim3(C::NT), 0, s, W, X, v0, nv, a->rows,
                     p.dp, p.pairs, mt, nt, a->targets, reinterpret_cast<float2*>(work + p.part),
                     reinterpret_cast<float*>(work + p.hit));
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}

template <class T>
int forward(const pots_vocab_loss* a, char* work, hipStream_t s) {
  const Plan p = plan(a, false);
  Mat X = {reinterpret_cast<const uint16_t*>(a->x),
           a->x_row * (int64_t)(sizeof(typename T::elem) / 2), 0};
  if (p.copy_x) {
    uint16_t* dst = reinterpret_cast<uint16_t*>(work + p.x);
    X = Mat{dst, (int64_t)p.dp, (int64_t)p.rows_pad * p.dp};
    const int rc = lay<T>(a->x, a->x_row, a->dim, a->rows, nullptr, nullptr, dst, p, X.plane,
                          a->rows, s);
    if (rc) return rc;
  }
  for (uint32_t v0 = 0; v0 < a->vocab; v0 += p.piece) {
    const uint32_t nv = min(a->vocab - v0, p.piece);
    Mat W;
    int rc = piece_of_w<T>(a, p, work, v0, nv, &W, s);
    if (rc) return rc;
    rc = p.direct              ? a->rows > 32 ? scores<Direct>(a, p, W, X, v0, nv, work, s)
                                              : scores<NarrowDirect>(a, p, W, X, v0, nv, work, s)
         : p.scores == kLarge  ? scores<Large<false, false>>(a, p, W, X, v0, nv, work, s)
         : p.scores == kMedium ? scores<Medium<false, false>>(a, p, W, X, v0, nv, work, s)
                               : scores<Narrow<false, false>>(a, p, W, X, v0, nv, work, s);
    if (rc) return rc;
  }
  const float2* part = reinterpret_cast<const float2*>(work + p.part);
  const float* hit = reinterpret_cast<const float*>(work + p.hit);
  const uint32_t chunks = cdiv(a->vocab, p.scores == kMedium ? 128 : 256);
  // four rows a block, in 32-byte reads, where blocks of 32 would be few (seven rows: 28 us and 4)
  if (a->rows < 2048)
    hipLaunchKernelGGL(loss_rows<4>, dim3(cdiv(a->rows, 4)), dim3(1024), 0, s, part, chunks, hit,
                       *a);
  else
    hipLaunchKernelGGL(loss_rows<32>, dim3(cdiv(a->rows, 32)), dim3(1024), 0, s, part, chunks,
                       hit, *a);
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}

template <class T, template <bool, bool> class S, template <bool, bool> class SX,
          template <bool, bool> class SW>
int piece_grads(const pots_vocab_loss* a, const Plan& p, const Mat& W, const Mat& X, uint32_t v0,
                uint32_t nv, char* work, hipStream_t s) {
  auto f32 = [&](uint64_t at) { return reinterpret_cast<float*>(work + at); };
  const uint32_t* count = reinterpret_cast<const uint32_t*>(work + p.count);
  typedef S<false, false> C;
  typedef SX<true, false> CX;
  typedef SW<true, true> CW;
  uint16_t* g = reinterpret_cast<uint16_t*>(work + p.g);
  const Mat G = {g, (int64_t)p.piece, (int64_t)p.rows_pad * p.piece};
  const uint32_t mt = cdiv(nv, C::TM), nt = cdiv(a->rows, C::TN);
  if (mt * nt) {
    hipLaunchKernelGGL((loss_grad<T, C>), dim3(mt * nt), dim3(C::NT), 0, s, W, X, v0, nv, count,
                       p.dp, p.pairs, mt, f32(p.weight), f32(p.lse2),
                       reinterpret_cast<const uint32_t*>(work + p.target), g, p.piece, G.plane);
    POTS_HIP(hipGetLastError());
  }
  typedef typename T::elem elem;
  elem* const dw = reinterpret_cast<elem*>(a->dw) + (int64_t)v0 * a->dw_row;
  const uint32_t xmt = cdiv(p.dp, CX::TM), wmt = cdiv(p.dp, CW::TM), wnt = cdiv(nv, CW::TN);
  hipLaunchKernelGGL((loss_products<T, CX, CW>), dim3(xmt * nt * p.splits + wmt * wnt * p.wsplits),
                     dim3(CX::NT), 0, s, W, X, G, p.dp, nv, count, f32(p.unit), p.pairs, xmt,
                     p.splits, p.per, f32(p.sums), (uint64_t)p.rows_pad * p.dp, v0 == 0, wmt,
                     wnt, p.wsplits, p.wper, p.join_w ? f32(p.wsums) : nullptr,
                     (uint64_t)p.piece * p.dp, a->dim, dw, a->dw_row);
  POTS_HIP(hipGetLastError());
  if (p.join_w) {
    hipLaunchKernelGGL((loss_join<T>), dim3(min(nv, kMostJoined)), dim3(256), 0, s, f32(p.wsums),
                       p.dp, p.wsplits, (uint64_t)p.piece * p.dp, nullptr, f32(p.unit), a->dim,
                       dw, a->dw_row, nv);
    POTS_HIP(hipGetLastError());
  }
  return POTS_E_OK;
}

template <class T>
int backward(const pots_vocab_loss* a, char* work, hipStream_t s) {
  const Plan p = plan(a, true);
  auto u32 = [&](uint64_t at) { return reinterpret_cast<uint32_t*>(work + at); };
  auto f32 = [&](uint64_t at) { return reinterpret_cast<float*>(work + at); };
  hipLaunchKernelGGL(live_rows, dim3(1), dim3(1024), 0, s, *a, u32(p.idx), u32(p.pos),
                     u32(p.count), f32(p.weight), f32(p.lse2), u32(p.target), f32(p.unit));
  POTS_HIP(hipGetLastError());
  uint16_t* xs = reinterpret_cast<uint16_t*>(work + p.x);
  const Mat X = {xs, (int64_t)p.dp, (int64_t)p.rows_pad * p.dp};
  if (a->rows) {
    const int rc = lay<T>(a->x, a->x_row, a->dim, a->rows, u32(p.idx), u32(p.count), xs, p,
                          X.plane, p.rows_pad, s);
    if (rc) return rc;
  }
  for (uint32_t v0 = 0; v0 < a->vocab; v0 += p.piece) {
    const uint32_t nv = min(a->vocab - v0, p.piece);
    Mat W = {};
    int rc = a->rows ? piece_of_w<T>(a, p, work, v0, nv, &W, s) : POTS_E_OK;
    if (rc) return rc;
    rc = p.products == kLarge
             ? piece_grads<T, Large, Large, Large>(a, p, W, X, v0, nv, work, s)
         : p.products == kTrimmed
             ? piece_grads<T, Large, Trimmed, Trimmed>(a, p, W, X, v0, nv, work, s)
         : p.products == kMedium
             ? piece_grads<T, Medium, Medium, Medium>(a, p, W, X, v0, nv, work, s)
             : piece_grads<T, Narrow, NarrowX, Large>(a, p, W, X, v0, nv, work, s);
    if (rc) return rc;
  }
  if (a->rows == 0) return POTS_E_OK;
  hipLaunchKernelGGL((loss_join<T>), dim3(min(a->rows, kMostJoined)), dim3(256), 0, s,
                     f32(p.sums), p.dp, p.splits, (uint64_t)p.rows_pad * p.dp, u32(p.pos),
                     f32(p.unit), a->dim, reinterpret_cast<typename T::elem*>(a->dx), a->dx_row,
                     a->rows);
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
