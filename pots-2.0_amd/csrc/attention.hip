// Softmax attention of a batch of sequences over their own keys, with its gradient, for
// passes that keep no probabilities.
//
//   s_ij = scale·q_i·k_j over the j that i sees, lse_i = log Σ_j e^{s_ij}, p_ij = e^{s_ij − lse_i}
//   o_i = Σ_j p_ij v_j
//   D_i = do_i·o_i,  dp_ij = do_i·v_j,  ds_ij = p_ij (dp_ij − D_i)
//   dq_i = scale Σ_j ds_ij k_j,  dk_j = scale Σ_i ds_ij q_i,  dv_j = Σ_i p_ij do_i
//
// with k and v shared by heads / kv_heads query heads, over which dk and dv are summed.
//
// Forward: one pass over the keys with a running maximum and sum. A wave holds 32 query rows as
// the columns of its products (tiles.h): Sᵀ = K·Qᵀ leaves a row's scores in one lane and its
// other half, and those registers are the right operand of Oᵀ += Vᵀ·Pᵀ as they are. K and V go
// through LDS, shared by a block's waves; V is read transposed from it.
//
// Backward: the probabilities are recomputed from lse. dq sums over keys and dk, dv over
// queries, so each has a kernel of its own whose sums stay in registers (attn_dq, which also
// makes D, and attn_dkv): seven products of a tile (eight for wide heads) where one kernel with
// atomics on dq would take five, for results that do not depend on the order of blocks. Few key
// heads leave attn_dkv with few blocks: then the query heads of a group are split over blocks, each
// with fp32 sums of its own that attn_fold adds in order.
//
// Bound, for long sequences in bf16, by no unit alone: the 1.5B shape (48 sequences of 2048 x 128,
// causal; products of the half that is seen) keeps the matrix cores busy for 0.31 of the cycles in
// attn_fwd, 0.38 in attn_dq and 0.32 in attn_dkv, issues vector instructions for about 0.43, 0.31
// and 0.24 (an exponential as four; in attn_fwd the maximum and its rescale too), and reads LDS
// for 0.16 to 0.21, without bank conflicts. Two waves a SIMD take turns at them, and in attn_dkv
// they wait for a tile or for each other for half of their time. attn_fwd 74 us, 0.70 PFLOP/s; attn_dq 95 us,
// 0.81; attn_dkv 190 us, 0.68; the 0.5B shape (112 of 1024 x 64): 29, 39 and 57 us. fp32 is bound by
// its matrix instructions, a sixteenth of bf16's rate, and small steps by how few blocks they have.
// Tiles that went through registers into padded LDS, with no tile on its way, took 159, 207 and
// 467 us.
//
// Roundings: bf16 p and ds (the right operands of the second products) are rounded to bf16, since the
// matrix cores take no product of bf16 and fp32: off by at most 2^-8 of each term of a sum whose
// result is rounded the same. The gradients of the 1.5B shape are off by 2.4e-3 of their norm, 1.7e-3
// with that last rounding alone, its output by 2.0e-3 and 1.6e-3. D is taken from out as it was
// rounded, but where a row sees few keys (attn_dq). Scores, statistics and sums are fp32.
//
// A value that is not finite, inside its sequence's length, may reach every row of its tile (zero
// times infinity); what lies past a length is never read.
#include <math.h>

#include "common.h"
#include "gmem.h"
#include "tiles.h"

namespace pots {

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Eight values of row r from column c on; zero for rows from `rows` and columns from `d` (a multiple
// of eight) on.
template <class T>
__device__ __forceinline__ typename T::frag load_frag(const typename T::elem* base,
                                                      int64_t stride, uint32_t r, uint32_t rows,
                                                      uint32_t c, uint32_t d) {
  typename T::frag f = {};
  if (r < rows && c < d) {
    const typename T::elem* p = base + (int64_t)r * stride + c;
    if constexpr (sizeof(typename T::elem) == 2) {
      f = gload<bf16x8>(p);
    } else {
      f = __builtin_shufflevector(gload<f32x4>(p), gload<f32x4>(p + 4), 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }
  return f;
}

// A tile of KT rows of DP columns in LDS, in 16-byte chunks, each exchanged within its row by
// swap(row) so that both of a tile's reads meet 64 different banks of four bytes: 16 lanes
// reading a chunk of 16 rows, and 32 lanes reading 64 bytes of four rows transposed.
template <class T, uint32_t DP, uint32_t KT, uint32_t NT>
struct Rows {
  typedef typename T::elem elem;
  typedef typename T::frag frag;
  static constexpr uint32_t CE = 16 / sizeof(elem), CPR = DP / CE, kAll = KT * CPR;
  static constexpr uint32_t kChunks = (kAll + NT - 1) / NT, kBytes = DP * sizeof(elem);
  uint32_t off[kChunks];

  static __device__ __forceinline__ uint32_t swap(uint32_t r) {
    const uint32_t low = (r >> 2) & 3;
    return kBytes % 256 == 0 ? (r & 3) << 2 | low : kBytes % 128 == 0 ? (r & 2) << 1 | low : low;
  }

  // A lane's offsets into a tile's rows; columns past d are out of any buffer's range.
  __device__ __forceinline__ void init(int64_t stride, uint32_t d) {
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++) {
      const uint32_t c = u * NT + threadIdx.x, r = c / CPR, col = ((c % CPR) ^ swap(r)) * CE;
      off[u] = col < d ? (r * (uint32_t)stride + col) * sizeof(elem) : 0x7FFFFFF0;
    }
  }

  // Rows r0 .. r0 + KT, straight into LDS (complete once the wave has waited for its loads); those
  // past `rows` and the columns past d are zero.
  __device__ __forceinline__ void load(elem* tile, const elem* base, int64_t stride, uint32_t r0,
                                       uint32_t rows, uint32_t d) const {
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    const uint32_t range = ((min(KT, rows - r0) - 1) * (uint32_t)stride + d) * sizeof(elem);
    const brsrc rsrc = make_rsrc(base + (int64_t)r0 * stride, range);
#pragma unroll
    for (uint32_t u = 0; u < kChunks; u++)
      if (kAll % NT == 0 || u * NT + wave * 64 < kAll)
        load_lds16(rsrc, tile + (u * NT + wave * 64) * CE, off[u]);
  }

  // Eight values of row r from column c on.
  static __device__ __forceinline__ frag row(const elem* tile, uint32_t r, uint32_t c) {
    const elem* p = tile + r * DP;
    if constexpr (sizeof(elem) == 2) {
      return *reinterpret_cast<const bf16x8*>(p + ((c / 8) ^ swap(r)) * 8);
    } else {
      const f32x4 a = *reinterpret_cast<const f32x4*>(p + ((c / 4) ^ swap(r)) * 4);
      const f32x4 b = *reinterpret_cast<const f32x4*>(p + ((c / 4 + 1) ^ swap(r)) * 4);
      return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
    }
  }

  // Column c + i at the rows that a D's registers 8t .. 8t + 7 hold: r0 + 4h + (0..3) and
  // r0 + 8 + 4h + (0..3), r0 = 16t.
  static __device__ __forceinline__ frag col(const elem* tile, uint32_t r0, uint32_t c,
                                             uint32_t lane) {
    const uint32_t h = lane / 32;
    if constexpr (sizeof(elem) == 2) {
      const uint32_t m = lane % 16, r = r0 + 4 * h + m / 4, at = c + (lane & 16) + 4 * (m % 4);
      const uint16_t* p = tile + at % 8;
      return join(read_tr(p + r * DP + ((at / 8) ^ swap(r)) * 8),
                  read_tr(p + (r + 8) * DP + ((at / 8) ^ swap(r + 8)) * 8));
    } else {
      f32x8 f;
#pragma unroll
      for (uint32_t j = 0; j < 8; j++) {
        const uint32_t r = r0 + 4 * h + j % 4 + 8 * (j / 4), at = c + lane % 32;
        f[j] = tile[r * DP + ((at / 4) ^ swap(r)) * 4 + at % 4];
      }
      return f;
    }
  }
};

template <class T>
struct Head {
  const typename T::elem* p;
  int64_t row;
  __device__ Head(const pots_heads& x, uint32_t b, uint32_t h)
      : p(reinterpret_cast<const typename T::elem*>(x.ptr) + b * x.batch + h * x.head),
        row(x.row) {}
};

__device__ __forceinline__ uint32_t length_of(const pots_attention& a, uint32_t b) {
  if (!a.lengths) return a.n;
  const int32_t l = gload<int32_t>(a.lengths + b);
  return l < 0 ? 0 : min((uint32_t)l, a.n);
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// A wave's D of [d_head × 32 rows] as rows of a tensor: lane (i, h) holds row r0 + i, four
// consecutive columns at a time (of the blocks of 32 columns `mine`, mine + step, ...).
template <class T, uint32_t NB>
__device__ __forceinline__ void store_rows(const pots_heads& x, uint32_t b, uint32_t head,
                                           uint32_t row, uint32_t n, uint32_t d,
                                           const f32x16 (&acc)[NB], float mul, uint32_t h,
                                           uint32_t step = 1, uint32_t mine = 0) {
  if (row >= n) return;
  typename T::elem* p = reinterpret_cast<typename T::elem*>(x.ptr) + b * x.batch +
                        head * x.head + (int64_t)row * x.row;
#pragma unroll
  for (uint32_t db = 0; db < NB; db++) {
    if (db % step != mine) continue;
#pragma unroll
    for (uint32_t g = 0; g < 4; g++) {
      const uint32_t c = 32 * db + 8 * g + 4 * h;
      if (c >= d) continue;
      const f32x16& v = acc[db];
      T::store4(p + c, v[4 * g] * mul, v[4 * g + 1] * mul, v[4 * g + 2] * mul,
                v[4 * g + 3] * mul);
    }
  }
}

// The sequence (of `seqs`) and the tile of a block, long tiles first: a launch's blocks start in
// order, and what is left at its end is short. Where the sequences divide over the XCDs, each
// XCD has some of its own, and their shared rows in its L2.
__device__ __forceinline__ void unit_of(uint32_t seqs, uint32_t* seq, uint32_t* place) {
  if (seqs % kXcds == 0) {
    const uint32_t per = seqs / kXcds, i = blockIdx.x / kXcds;
    *seq = blockIdx.x % kXcds * per + i % per;
    *place = i / per;
  } else {
    *seq = blockIdx.x % seqs;
    *place = blockIdx.x / seqs;
  }
}

// How a block divides its work. Rows: four waves of 32 rows each (queries; keys in attn_dkv) go
// through the other side's tiles of 64 (32 in fp32) together. Split: where that leaves compute
// units without a block, a block has 32 rows and each wave takes its own 32 of a tile's 128; the
// waves' sums are joined at the end, in order. A split block loads a tile when it has done with the
// one before: its sequences are short, and where two blocks fit a compute unit (bf16, but attn_dkv
// of heads past 96; fp32 heads to 64, in attn_dkv to 32) they cover for each other. Elsewhere the loads
// show, but a second tile would leave no room for four waves. The 135M decoder's layer (fp32, 36
// query heads' sequences of 256), us: blocks of one wave 24 (attn_fwd), 32 (attn_dq) and 47 (attn_dkv),
// split ones 14, 21 and 22; two sequences of 675 x 128 in fp32 56, 78 and 80 with two waves and a tile
// ahead, 37, 51 and 49.
template <class T, uint32_t DP, bool SPLIT>
struct Shape {
  static constexpr uint32_t kWide = DP * sizeof(typename T::elem);  // bytes of a row
  static constexpr uint32_t NW = 4, NT = 64 * NW;
  static constexpr uint32_t R = SPLIT ? 32 : 32 * NW;  // the block's rows
  static constexpr uint32_t KT = SPLIT ? 32 * NW : sizeof(typename T::elem) == 2 ? 64 : 32;
  static constexpr uint32_t U = SPLIT ? 1 : KT / 32;   // a wave's products in a tile
  static constexpr uint32_t KS = DP / 16, NB = DP / 32;
  static constexpr uint32_t kStat = KT < 64 ? 64 : KT;  // a tile's statistics, 64 to a load
  static constexpr bool kApart = DP > 64;               // dk and dv in blocks of their own
  typedef Rows<T, DP, KT, NT> Tile;
  typedef typename T::elem Lds[KT * DP];
  typedef typename T::elem Next[SPLIT ? 1 : KT * DP];  // the tile on its way; a split block has none
};

// The four waves' sums of a split block, joined in order: two waves' in each of its tiles, of which
// the caller's blocks of 32 columns, wave, wave + 4, ..., come back in acc. Between two barriers.
template <uint32_t NB>
__device__ __forceinline__ float* sums_of(void* a, void* b, uint32_t wave) {
  return reinterpret_cast<float*>(wave < 2 ? a : b) + wave % 2 * NB * 1024;
}
template <uint32_t NB>
__device__ __forceinline__ void put_sums(f32x16 (&acc)[NB], void* a, void* b, uint32_t wave,
                                         uint32_t lane) {
  float* p = sums_of<NB>(a, b, wave) + lane;
#pragma unroll
  for (uint32_t db = 0; db < NB; db++)
#pragma unroll
    for (uint32_t r = 0; r < 16; r++) p[(db * 16 + r) * 64] = acc[db][r];
}
template <uint32_t NB>
__device__ __forceinline__ void join_sums(f32x16 (&acc)[NB], void* a, void* b, uint32_t wave,
                                          uint32_t lane) {
#pragma unroll
  for (uint32_t db = 0; db < NB; db++) {
    if (db % 4 != wave) continue;
#pragma unroll
    for (uint32_t r = 0; r < 16; r++) {
      float sum = 0.f;
#pragma unroll
      for (uint32_t w = 0; w < 4; w++) sum += sums_of<NB>(a, b, w)[(db * 16 + r) * 64 + lane];
      acc[db][r] = sum;
    }
  }
}

template <class T, uint32_t DP, bool SPLIT>
__global__ __launch_bounds__((Shape<T, DP, SPLIT>::NT),
                             (!SPLIT && Shape<T, DP, SPLIT>::kWide <= 256 ? 2 : 1)) void attn_fwd(
    pots_attention a, uint32_t tiles) {
  typedef typename T::elem elem;
  typedef typename T::frag frag;
  typedef Shape<T, DP, SPLIT> S;
  typedef typename S::Tile R;
  constexpr uint32_t NW = S::NW, KT = S::KT, KS = S::KS, NB = S::NB, U = S::U;
  __shared__ __attribute__((aligned(16))) typename S::Lds s_k0, s_v0;
  __shared__ __attribute__((aligned(16))) typename S::Next s_k1, s_v1;
  uint32_t bh, place;
  unit_of(a.batch * a.heads, &bh, &place);
  const uint32_t tile = tiles - 1 - place, b = bh / a.heads, head = bh % a.heads;
  const uint32_t kvh = head / (a.heads / a.kv_heads);
  const uint32_t lane = threadIdx.x % 64, i = lane % 32, h = lane / 32;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t len = length_of(a, b), d = a.head_dim;
  const Head<T> Q(a.q, b, head), K(a.k, b, kvh), V(a.v, b, kvh);
  const uint32_t q0 = tile * S::R, qw = SPLIT ? q0 : q0 + 32 * wave, q = qw + i;
  // keys that the block's rows see, and the wave's
  const uint32_t end = q0 >= len ? 0 : a.causal ? min(len, q0 + S::R) : len;
  const uint32_t wend = qw >= len ? 0 : a.causal ? min(len, qw + 32) : len;
  const uint32_t seen = q >= len ? 0 : a.causal ? min(len, q + 1) : len;
  R rk, rv;
  rk.init(K.row, d);
  rv.init(V.row, d);
  auto load = [&](elem* k, elem* v, uint32_t k0) {
    rk.load(k, K.p, K.row, k0, len, d);
    rv.load(v, V.p, V.row, k0, len, d);
  };
  if (end) load(s_k0, s_v0, 0);
  frag qf[KS];
#pragma unroll
  for (uint32_t ks = 0; ks < KS; ks++)
    qf[ks] = load_frag<T>(Q.p, Q.row, q, len, 16 * ks + 8 * h, d);
  f32x16 o[NB];
#pragma unroll
  for (uint32_t db = 0; db < NB; db++) o[db] = zero16();
  const float c = a.scale * kLog2e;
  float m = -INFINITY, mc = 0.f, l = 0.f;
  auto step = [&](const elem* s_k, const elem* s_v, uint32_t t0) {
    const uint32_t at = SPLIT ? 32 * wave : 0, k0 = t0 + at;  // of the tile, the wave's part
    if (k0 >= wend) return;
    f32x16 s[U];
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
      s[u] = zero16();
#pragma unroll
      for (uint32_t ks = 0; ks < KS; ks++)
        s[u] = mma(R::row(s_k, at + 32 * u + i, 16 * ks + 8 * h), qf[ks], s[u]);
    }
    // a tile that some row sees in part, or rows that see nothing
    if (k0 + 32 * U > len || qw + 32 > len || (a.causal && k0 + 32 * U - 1 > qw)) {
#pragma unroll
      for (uint32_t u = 0; u < U; u++)
#pragma unroll
        for (uint32_t r = 0; r < 16; r++)
          if (k0 + 32 * u + d_row(r, h) >= seen) s[u][r] = -INFINITY;
    }
    float top = m;
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) top = fmaxf(top, s[u][r]);
    top = fmaxf(top, other_half(top));
    if (__any(top > m)) {
      const float tc = top == -INFINITY ? 0.f : top * c;
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mc - tc);
      m = top;
      mc = tc;
      l *= f;
#pragma unroll
      for (uint32_t db = 0; db < NB; db++)
#pragma unroll
        for (uint32_t r = 0; r < 16; r++) o[db][r] *= f;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) {
        s[u][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][r], c, -mc));
        l += s[u][r];
      }
#pragma unroll
      for (uint32_t t = 0; t < 2; t++) {
        const frag p = T::pack(s[u], 8 * t);
#pragma unroll
        for (uint32_t db = 0; db < NB; db++)
          o[db] = mma(R::col(s_v, at + 32 * u + 16 * t, 32 * db, lane), p, o[db]);
      }
    }
  };
  uint32_t k0 = 0;
  for (; SPLIT && k0 + KT < end; k0 += KT) {
    loads_done();
    step(s_k0, s_v0, k0);
    __syncthreads();
    load(s_k0, s_v0, k0 + KT);
  }
  for (; k0 + KT < end; k0 += 2 * KT) {  // the next tile is on its way while one is worked on
    loads_done();
    load(s_k1, s_v1, k0 + KT);
    step(s_k0, s_v0, k0);
    loads_done();
    if (k0 + 2 * KT < end) load(s_k0, s_v0, k0 + 2 * KT);
    step(s_k1, s_v1, k0 + KT);
  }
  if (k0 < end) {
    loads_done();
    step(s_k0, s_v0, k0);
  }
  l += other_half(l);
  if constexpr (SPLIT) {
    // each wave's sums in units of the largest maximum of all, then added up
    __shared__ float s_m[NW][32], s_l[NW][32];
    if (h == 0) s_m[wave][i] = m == -INFINITY ? -INFINITY : mc;
    __syncthreads();  // and every wave is done with its tiles
    float top = -INFINITY;
#pragma unroll
    for (uint32_t w = 0; w < NW; w++) top = fmaxf(top, s_m[w][i]);
    // (a sum without a finite maximum is zero, or NaN, which stays)
    const float f = m == -INFINITY || mc == top ? 1.f : __builtin_amdgcn_exp2f(mc - top);
    if (h == 0) s_l[wave][i] = l * f;
#pragma unroll
    for (uint32_t db = 0; db < NB; db++)
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) o[db][r] *= f;
    put_sums<NB>(o, s_k0, s_v0, wave, lane);
    __syncthreads();
    l = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < NW; w++) l += s_l[w][i];
    mc = top == -INFINITY ? 0.f : top;
    join_sums<NB>(o, s_k0, s_v0, wave, lane);
  }
  store_rows<T, NB>(a.out, b, head, q, a.n, d, o, l > 0.f || l != l ? 1.f / l : 0.f, h,
                    SPLIT ? NW : 1, SPLIT ? wave : 0);
  if (h == 0 && q < a.n && (!SPLIT || wave == 0))
    a.lse[(int64_t)bh * a.n + q] =
        l == 0.f ? -INFINITY : (mc + __builtin_amdgcn_logf(l)) * kLn2;
}

// dq, and for attn_dkv each row's lse in units of log2 and D: stat [2][batch·heads][n]. A wave
// holds 32 query rows as columns, as in the forward pass: Sᵀ = K·Qᵀ and dPᵀ = V·dOᵀ from the
// tiles' rows, dQᵀ += Kᵀ·dSᵀ with K read transposed.
//
// D = Σ dO·out carries the rounding of out, which counts where a row sees few keys, since its out is
// then as large as v and no average of many. Rows that see one product of 32 keys or less, the first
// of causal sequences, take D = Σ p·dp from their registers instead, in no time that shows (the
// gradients of the 0.5B shape are then off by 2.4e-3 of their norm, else 2.5e-3; with no rounding
// but their own 1.7e-3).
template <class T, uint32_t DP, bool SPLIT>
__global__ __launch_bounds__((Shape<T, DP, SPLIT>::NT),
                             (Shape<T, DP, SPLIT>::kWide <= 256 ? 2 : 1)) void attn_dq(
    pots_attention a, float* __restrict__ stat, uint32_t tiles) {
  typedef typename T::elem elem;
  typedef typename T::frag frag;
  typedef Shape<T, DP, SPLIT> S;
  typedef typename S::Tile R;
  constexpr uint32_t NW = S::NW, KT = S::KT, KS = S::KS, NB = S::NB, U = S::U;
  __shared__ __attribute__((aligned(16))) typename S::Lds s_k0, s_v0;
  __shared__ __attribute__((aligned(16))) typename S::Next s_k1, s_v1;
  uint32_t bh, place;
  unit_of(a.batch * a.heads, &bh, &place);
  const uint32_t tile = tiles - 1 - place, b = bh / a.heads, head = bh % a.heads;
  const uint32_t kvh = head / (a.heads / a.kv_heads);
  const uint32_t lane = threadIdx.x % 64, i = lane % 32, h = lane / 32;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t len = length_of(a, b), d = a.head_dim;
  const Head<T> Q(a.q, b, head), K(a.k, b, kvh), V(a.v, b, kvh), O(a.out, b, head),
      G(a.dout, b, head);
  const uint32_t q0 = tile * S::R, qw = SPLIT ? q0 : q0 + 32 * wave, q = qw + i;
  const uint32_t end = q0 >= len ? 0 : a.causal ? min(len, q0 + S::R) : len;
  const uint32_t wend = qw >= len ? 0 : a.causal ? min(len, qw + 32) : len;
  const uint32_t seen = q >= len ? 0 : a.causal ? min(len, q + 1) : len;
  R rk, rv;
  rk.init(K.row, d);
  rv.init(V.row, d);
  auto load = [&](elem* k, elem* v, uint32_t k0) {
    rk.load(k, K.p, K.row, k0, len, d);
    rv.load(v, V.p, V.row, k0, len, d);
  };
  if (end) load(s_k0, s_v0, 0);
  frag qf[KS], gf[KS];
  float dl = 0.f;
#pragma unroll
  for (uint32_t ks = 0; ks < KS; ks++) {
    qf[ks] = load_frag<T>(Q.p, Q.row, q, len, 16 * ks + 8 * h, d);
    gf[ks] = load_frag<T>(G.p, G.row, q, len, 16 * ks + 8 * h, d);
    const frag of = load_frag<T>(O.p, O.row, q, len, 16 * ks + 8 * h, d);
#pragma unroll
    for (int j = 0; j < 8; j++) dl = __builtin_fmaf(T::at(gf[ks], j), T::at(of, j), dl);
  }
  dl += other_half(dl);
  float lse2 = INFINITY;  // a row that sees nothing has probabilities of zero
  if (q < a.n) {
    const int64_t at = (int64_t)bh * a.n + q;
    const float x = q < len ? gload<float>(a.lse + at) : -INFINITY;
    if (x != -INFINITY) lse2 = x * kLog2e;
    if (h == 0 && (!SPLIT || wave == 0)) {
      stat[at] = lse2;
      stat[(int64_t)a.batch * a.heads * a.n + at] = dl;
    }
  }
  f32x16 acc[NB];
#pragma unroll
  for (uint32_t db = 0; db < NB; db++) acc[db] = zero16();
  const float c = a.scale * kLog2e;
  auto step = [&](const elem* s_k, const elem* s_v, uint32_t k0) {
#pragma unroll
    for (uint32_t x = 0; x < U; x++) {
      const uint32_t u = SPLIT ? wave : x, ku = k0 + 32 * u;
      if (ku >= wend) return;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (uint32_t ks = 0; ks < KS; ks++) {
        s = mma(R::row(s_k, 32 * u + i, 16 * ks + 8 * h), qf[ks], s);
        dp = mma(R::row(s_v, 32 * u + i, 16 * ks + 8 * h), gf[ks], dp);
      }
#pragma unroll
      for (uint32_t r = 0; r < 16; r++)
        s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -lse2));
      if (wend <= 32) {  // all the keys of these rows are here
        dl = 0.f;
#pragma unroll
        for (uint32_t r = 0; r < 16; r++)
          if (d_row(r, h) < seen) dl = __builtin_fmaf(s[r], dp[r], dl);
        dl += other_half(dl);
        if (h == 0 && q < a.n)
          stat[((int64_t)a.batch * a.heads + bh) * a.n + q] = dl;
      }
#pragma unroll
      for (uint32_t r = 0; r < 16; r++) s[r] *= dp[r] - dl;
      if (ku + 32 > len || qw + 32 > len || (a.causal && ku + 31 > qw)) {
#pragma unroll
        for (uint32_t r = 0; r < 16; r++)
          if (ku + d_row(r, h) >= seen) s[r] = 0.f;
      }
#pragma unroll
      for (uint32_t t = 0; t < 2; t++) {
        const frag p = T::pack(s, 8 * t);
#pragma unroll
        for (uint32_t db = 0; db < NB; db++)
          acc[db] = mma(R::col(s_k, 32 * u + 16 * t, 32 * db, lane), p, acc[db]);
      }
    }
  };
  uint32_t k0 = 0;
  for (; SPLIT && k0 + KT < end; k0 += KT) {
    loads_done();
    step(s_k0, s_v0, k0);
    __syncthreads();
    load(s_k0, s_v0, k0 + KT);
  }
  for (; k0 + KT < end; k0 += 2 * KT) {
    loads_done();
    load(s_k1, s_v1, k0 + KT);
    step(s_k0, s_v0, k0);
    loads_done();
    if (k0 + 2 * KT < end) load(s_k0, s_v0, k0 + 2 * KT);
    step(s_k1, s_v1, k0 + KT);
  }
  if (k0 < end) {
    loads_done();
    step(s_k0, s_v0, k0);
  }
  if constexpr (SPLIT) {
    __syncthreads();
    put_sums<NB>(acc, s_k0, s_v0, wave, lane);
    __syncthreads();
    join_sums<NB>(acc, s_k0, s_v0, wave, lane);
  }
  store_rows<T, NB>(a.dq, b, head, q, a.n, d, acc, a.scale, h, SPLIT ? NW : 1,
                    SPLIT ? wave : 0);
}

// dk and dv of a block's keys, over `per` query heads of their group and the queries that see
// them. A wave holds 32 keys as columns: S = Q·Kᵀ and dP = dO·Vᵀ from the tiles' rows, dVᵀ +=
// dOᵀ·P and dKᵀ += Qᵀ·dS from the same tiles read transposed. With `part`, the sums go to fp32
// slices [2][split][batch][kv_heads][n][d].
enum DkvWhat { kBoth, kOnlyDk, kOnlyDv };

template <class T, uint32_t DP, bool SPLIT, DkvWhat WHAT>
__device__ __forceinline__ void dkv_block(
    const pots_attention& a, const float* __restrict__ stat, float* __restrict__ part,
    uint32_t seq, uint32_t tile, uint32_t splits, uint32_t per, typename T::elem* s_q0,
    typename T::elem* s_q1, typename T::elem* s_g0, typename T::elem* s_g1, float* s_stat0,
    float* s_stat1) {
  typedef typename T::elem elem;
  typedef typename T::frag frag;
  typedef Shape<T, DP, SPLIT> S;
  typedef typename S::Tile R;
  constexpr uint32_t NW = S::NW, QT = S::KT, KS = S::KS, NB = S::NB, U = S::U;
  constexpr uint32_t kStat = S::kStat;
  constexpr bool kDk = WHAT != kOnlyDv, kDv = WHAT != kOnlyDk;
  const uint32_t split = seq % splits, bk = seq / splits, b = bk / a.kv_heads;
  const uint32_t kvh = bk % a.kv_heads, rep = a.heads / a.kv_heads;
  const uint32_t lane = threadIdx.x % 64, i = lane % 32, h = lane / 32;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const uint32_t len = length_of(a, b), d = a.head_dim;
  const Head<T> K(a.k, b, kvh), V(a.v, b, kvh);
  const uint32_t k0 = tile * S::R, kw = SPLIT ? k0 : k0 + 32 * wave, key = kw + i;
  // the block's steps: (head, tile of queries) in order
  const uint32_t first = a.causal ? k0 / QT * QT : 0, e0 = split * per;
  const uint32_t tiles_q = k0 < len ? (len - first + QT - 1) / QT : 0;
  const uint32_t steps = tiles_q * (min(rep, e0 + per) - e0);
  R rq, rg;
  rq.init(a.q.row, d);
  rg.init(a.dout.row, d);
  const float* const stat1 = stat + (int64_t)a.batch * a.heads * a.n;
  uint32_t le = e0, lq = first;  // the next step to load
  auto load = [&](elem* s_q, elem* s_g, float* s_stat) {
    const uint32_t head = kvh * rep + le;
    const Head<T> Q(a.q, b, head), G(a.dout, b, head);
    rq.load(s_q, Q.p, Q.row, lq, len, d);
    rg.load(s_g, G.p, G.row, lq, len, d);
    if (64 * wave < kStat) {  // lse and D of the tile's rows, 64 a wave; zero past the length
      const uint32_t q = lq + 64 * wave;
      const int64_t at = (int64_t)(b * a.heads + head) * a.n + q;
      const uint32_t range = q < len ? 4 * min(64u, len - q) : 0;
      load_lds4(make_rsrc(stat + at, range), s_stat + 64 * wave, 4 * lane);
      load_lds4(make_rsrc(stat1 + at, range), s_stat + kStat + 64 * wave, 4 * lane);
    }
    lq += QT;
    if (lq >= len) {
      lq = first;
      le++;
    }
  };
  if (steps) load(s_q0, s_g0, s_stat0);
  frag kf[KS], vf[KS];
#pragma unroll
  for (uint32_t ks = 0; ks < KS; ks++) {
    kf[ks] = load_frag<T>(K.p, K.row, key, len, 16 * ks + 8 * h, d);
    if (kDk) vf[ks] = load_frag<T>(V.p, V.row, key, len, 16 * ks + 8 * h, d);
  }
  f32x16 dk[NB], dv[NB];
#pragma unroll
  for (uint32_t db = 0; db < NB; db++) {
    dk[db] = zero16();
    dv[db] = zero16();
  }
  const float c = a.scale * kLog2e;
  uint32_t q0 = first;
  auto step = [&](const elem* s_q, const elem* s_g, const float* s_stat) {
#pragma unroll
    for (uint32_t y = 0; y < U; y++) {
      const uint32_t u = SPLIT ? wave : y, qu = q0 + 32 * u;
      if (qu >= len || kw >= len || (a.causal && qu + 31 < kw)) continue;
      f32x16 s = zero16(), dp = zero16();
#pragma unroll
      for (uint32_t ks = 0; ks < KS; ks++) {
        s = mma(R::row(s_q, 32 * u + i, 16 * ks + 8 * h), kf[ks], s);
        if (kDk) dp = mma(R::row(s_g, 32 * u + i, 16 * ks + 8 * h), vf[ks], dp);
      }
#pragma unroll
      for (uint32_t g = 0; g < 4; g++) {
        const float* st = s_stat + 32 * u + 8 * g + 4 * h;
        const f32x4 ls = *reinterpret_cast<const f32x4*>(st);
        const f32x4 dl = *reinterpret_cast<const f32x4*>(st + kStat);
#pragma unroll
        for (uint32_t x = 0; x < 4; x++) {
          const uint32_t r = 4 * g + x;
          s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], c, -ls[x]));
          if (kDk) dp[r] = s[r] * (dp[r] - dl[x]);
        }
      }
      if (kw + 32 > len || qu + 32 > len || (a.causal && qu < kw + 31)) {
#pragma unroll
        for (uint32_t r = 0; r < 16; r++) {
          const uint32_t q = qu + d_row(r, h);
          if (key >= len || q >= len || (a.causal && q < key)) s[r] = dp[r] = 0.f;
        }
      }
#pragma unroll
      for (uint32_t t = 0; t < 2; t++) {
        const frag p = T::pack(kDv ? s : dp, 8 * t), ds = T::pack(dp, 8 * t);
#pragma unroll
        for (uint32_t db = 0; db < NB; db++) {
          const uint32_t r0 = 32 * u + 16 * t;
          if (kDv) dv[db] = mma(R::col(s_g, r0, 32 * db, lane), p, dv[db]);
          if (kDk) dk[db] = mma(R::col(s_q, r0, 32 * db, lane), ds, dk[db]);
        }
      }
    }
    q0 = q0 + QT < len ? q0 + QT : first;
  };
  uint32_t t = 0;
  for (; SPLIT && t + 1 < steps; t++) {
    loads_done();
    step(s_q0, s_g0, s_stat0);
    __syncthreads();
    load(s_q0, s_g0, s_stat0);
  }
  for (; t + 2 <= steps; t += 2) {
    loads_done();
    load(s_q1, s_g1, s_stat1);
    step(s_q0, s_g0, s_stat0);
    loads_done();
    if (t + 2 < steps) load(s_q0, s_g0, s_stat0);
    step(s_q1, s_g1, s_stat1);
  }
  if (t < steps) {
    loads_done();
    step(s_q0, s_g0, s_stat0);
  }
  if constexpr (SPLIT) {
    auto join = [&](f32x16(&acc)[NB]) {
      __syncthreads();
      put_sums<NB>(acc, s_q0, s_g0, wave, lane);
      __syncthreads();
      join_sums<NB>(acc, s_q0, s_g0, wave, lane);
    };
    if (kDk) join(dk);
    if (kDv) join(dv);
  }
  constexpr uint32_t kOf = SPLIT ? NW : 1;
  const uint32_t mine = SPLIT ? wave : 0;
  if (part) {
    pots_heads x;
    x.row = d;
    x.head = (int64_t)a.n * d;
    x.batch = x.head * a.kv_heads;
    x.ptr = part + split * x.batch * a.batch;
    if (kDk) store_rows<Fp32, NB>(x, b, kvh, key, a.n, d, dk, a.scale, h, kOf, mine);
    x.ptr = part + (splits + split) * x.batch * a.batch;
    if (kDv) store_rows<Fp32, NB>(x, b, kvh, key, a.n, d, dv, 1.f, h, kOf, mine);
  } else {
    if (kDk) store_rows<T, NB>(a.dk, b, kvh, key, a.n, d, dk, a.scale, h, kOf, mine);
    if (kDv) store_rows<T, NB>(a.dv, b, kvh, key, a.n, d, dv, 1.f, h, kOf, mine);
  }
}


// Wide heads have a block for dk and one for dv, which both make S: five products of a tile, not
// four, but sums and fragments of one fit two waves a SIMD (1.5B shape: 194 us together, one
// wave a SIMD, 188 apart; two heads of 675 in fp32, a launch of few blocks: 121 and 80).
template <class T, uint32_t DP, bool SPLIT>
__global__ __launch_bounds__((Shape<T, DP, SPLIT>::NT),
                             (!SPLIT && Shape<T, DP, SPLIT>::kWide <= 256 ? 2 : 1)) void attn_dkv(
    pots_attention a, const float* __restrict__ stat, float* __restrict__ part, uint32_t splits,
    uint32_t per) {
  typedef Shape<T, DP, SPLIT> S;
  __shared__ __attribute__((aligned(16))) typename S::Lds s_q0, s_g0;
  __shared__ __attribute__((aligned(16))) typename S::Next s_q1, s_g1;
  __shared__ __attribute__((aligned(16))) float s_stat0[2 * S::kStat], s_stat1[2 * S::kStat];
  const uint32_t seqs = a.batch * a.kv_heads * splits;
  uint32_t seq, place;
  if constexpr (S::kApart) {
    unit_of(2 * seqs, &seq, &place);
    const uint32_t tile = place;
    if (seq % 2 == 0)
      dkv_block<T, DP, SPLIT, kOnlyDk>(a, stat, part, seq / 2, tile, splits, per, s_q0, s_q1,
                                       s_g0, s_g1, s_stat0, s_stat1);
    else
      dkv_block<T, DP, SPLIT, kOnlyDv>(a, stat, part, seq / 2, tile, splits, per, s_q0, s_q1,
                                       s_g0, s_g1, s_stat0, s_stat1);
  } else {
    unit_of(seqs, &seq, &place);
    dkv_block<T, DP, SPLIT, kBoth>(a, stat, part, seq, place, splits, per, s_q0, s_q1, s_g0, s_g1,
                                   s_stat0, s_stat1);
  }
}

// dk (blockIdx.y = 0) and dv (1) from the splits' sums, in order, four values a thread.
template <class T>
__global__ __launch_bounds__(256) void attn_fold(pots_attention a,
                                                 const float* __restrict__ part,
                                                 uint32_t splits) {
  const uint64_t each = (uint64_t)a.batch * a.kv_heads * a.n * a.head_dim;
  const float* p = part + blockIdx.y * splits * each;
  const pots_heads& x = blockIdx.y ? a.dv : a.dk;
  for (uint64_t e = ((uint64_t)blockIdx.x * 256 + threadIdx.x) * 4; e < each;
       e += (uint64_t)gridDim.x * 1024) {
    f32x4 sum = gload<f32x4>(p + e);
    for (uint32_t s = 1; s < splits; s++) sum += gload<f32x4>(p + s * each + e);
    const uint64_t row = e / a.head_dim, bk = row / a.n;
    T::store4(reinterpret_cast<typename T::elem*>(x.ptr) + (int64_t)(bk / a.kv_heads) * x.batch +
                  (int64_t)(bk % a.kv_heads) * x.head + (int64_t)(row - bk * a.n) * x.row +
                  (e - row * a.head_dim),
              sum[0], sum[1], sum[2], sum[3]);
  }
}

namespace {

bool bad(const pots_attention* a) {
  return !a || a->dtype > POTS_OP_BF16 || a->kv_heads == 0 || a->heads == 0 ||
         a->heads % a->kv_heads || a->head_dim == 0 || a->head_dim % 8 ||
         a->head_dim > POTS_ATTENTION_MAX_DIM ||
         !(a->scale > 0.f) || !isfinite(a->scale) || a->n > 0x40000000u ||
         (uint64_t)a->batch * a->heads > 0x100000u;
}

// Whether x's rows start on 16-byte borders, and a tile of them spans less than 2 GiB.
bool aligned(const pots_attention* a, const pots_heads& x) {
  const int64_t e = a->dtype == POTS_OP_BF16 ? 2 : 4;
  return reinterpret_cast<uint64_t>(x.ptr) % 16 == 0 && x.batch * e % 16 == 0 &&
         x.head * e % 16 == 0 && x.row * e % 16 == 0 && x.row >= 0 && x.row < (1 << 22);
}

uint32_t cdiv(uint32_t a, uint32_t b) { return a / b + (a % b != 0); }

constexpr uint64_t kMostBlocks = (1u << 24) - 1;  // of 256 threads: less than 2^32 in a launch

// Whether blocks of 128 rows leave compute units without one: blocks of 32 then.
bool few(uint64_t sequences, uint32_t n) { return sequences * cdiv(n, 128) < 256; }

struct Cut {
  bool split;
  uint32_t tiles, splits, per;  // of keys; of a group's query heads in attn_dkv
};

// The query heads of a group are shared out over blocks while there are fewer blocks than
// compute units and a block has more than two tiles of queries to go through, or fewer than
// three for each (causal tiles differ in length, and the launch ends with the short ones) and
// more than eight tiles. us, attn_dkv and attn_fold, with half as many blocks asked for and so: the
// 0.5B shape 75 + 7 and 57 + 8, the 1.5B shape 266 + 9 and 200 + 12; with twice as many no faster.
Cut cut(const pots_attention* a) {
  Cut c;
  const uint32_t rep = a->heads / a->kv_heads;
  c.split = few((uint64_t)a->batch * a->heads, a->n);
  c.tiles = cdiv(a->n, c.split ? 32 : 128);
  const uint64_t blocks = (uint64_t)a->batch * a->kv_heads * c.tiles * (a->head_dim > 64 ? 2 : 1);
  const uint32_t steps = cdiv(a->n, c.split ? 128 : 64);
  c.splits = 1;
  while (c.splits < rep) {
    const uint64_t now = blocks * c.splits, left = (uint64_t)steps * cdiv(rep, c.splits);
    if (!(now < 256 && left > 2) && !(now < 768 && left > 8)) break;
    c.splits++;
  }
  c.per = cdiv(rep, c.splits);
  c.splits = cdiv(rep, c.per);
  return c;
}

template <class T, uint32_t DP, bool SPLIT>
int forward(const pots_attention* a, hipStream_t s) {
  typedef Shape<T, DP, SPLIT> S;
  const uint32_t tiles = cdiv(a->n, S::R);
  const uint64_t blocks = (uint64_t)a->batch * a->heads * tiles;
  if (blocks > kMostBlocks) return POTS_E_ARG;
  hipLaunchKernelGGL((attn_fwd<T, DP, SPLIT>), dim3((uint32_t)blocks), dim3(S::NT), 0, s, *a,
                     tiles);
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}

template <class T, uint32_t DP, bool SPLIT>
int backward(const pots_attention* a, char* work, hipStream_t s) {
  typedef Shape<T, DP, SPLIT> S;
  const Cut c = cut(a);
  const uint64_t qblocks = (uint64_t)a->batch * a->heads * c.tiles;
  const uint64_t kblocks =
      (uint64_t)a->batch * a->kv_heads * c.tiles * c.splits * (S::kApart ? 2 : 1);
  if (qblocks > kMostBlocks || kblocks > kMostBlocks) return POTS_E_ARG;
  float* stat = reinterpret_cast<float*>(work);
  float* part = nullptr;
  if (c.splits > 1)
    part = reinterpret_cast<float*>(work +
                                    align_up((size_t)a->batch * a->heads * a->n * 8, 256));
  hipLaunchKernelGGL((attn_dq<T, DP, SPLIT>), dim3((uint32_t)qblocks), dim3(S::NT), 0, s, *a,
                     stat, c.tiles);
  POTS_HIP(hipGetLastError());
  hipLaunchKernelGGL((attn_dkv<T, DP, SPLIT>), dim3((uint32_t)kblocks), dim3(S::NT), 0, s, *a,
                     stat, part, c.splits, c.per);
  POTS_HIP(hipGetLastError());
  if (part) {
    const uint64_t each = (uint64_t)a->batch * a->kv_heads * a->n * a->head_dim;
    const uint64_t nb = (each + 1023) / 1024;
    hipLaunchKernelGGL((attn_fold<T>), dim3((uint32_t)(nb < 4096 ? nb : 4096), 2), dim3(256), 0,
                       s, *a, part, c.splits);
    POTS_HIP(hipGetLastError());
  }
  return POTS_E_OK;
}

#define POTS_SPLIT(T, DP, F, ...) \
  (split ? F<T, DP, true>(__VA_ARGS__) : F<T, DP, false>(__VA_ARGS__))
#define POTS_DIMS(T, F, ...)                                     \
  (a->head_dim <= 32   ? POTS_SPLIT(T, 32, F, __VA_ARGS__)       \
   : a->head_dim <= 64 ? POTS_SPLIT(T, 64, F, __VA_ARGS__)       \
   : a->head_dim <= 96 ? POTS_SPLIT(T, 96, F, __VA_ARGS__)       \
                       : POTS_SPLIT(T, 128, F, __VA_ARGS__))

}  // namespace

}  // namespace pots

using namespace pots;

extern "C" int pots_attention_forward(const pots_attention* a, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (a->batch == 0 || a->n == 0) return POTS_E_OK;
  if (!a->q.ptr || !a->k.ptr || !a->v.ptr || !a->out.ptr || !a->lse) return POTS_E_ARG;
  for (const pots_heads* x : {&a->q, &a->k, &a->v, &a->out})
    if (!aligned(a, *x)) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool split = few((uint64_t)a->batch * a->heads, a->n);
  return a->dtype == POTS_OP_BF16 ? POTS_DIMS(Bf16, forward, a, s)
                                  : POTS_DIMS(Fp32, forward, a, s);
}

extern "C" uint64_t pots_attention_backward_work(const pots_attention* a) {
  if (bad(a) || a->batch == 0 || a->n == 0) return 0;
  const Cut c = cut(a);
  uint64_t bytes = align_up((size_t)a->batch * a->heads * a->n * 8, 256);
  if (c.splits > 1)
    bytes += 2ull * c.splits * a->batch * a->kv_heads * a->n * a->head_dim * 4;
  return bytes;
}

extern "C" int pots_attention_backward(const pots_attention* a, void* work, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (a->batch == 0 || a->n == 0) return POTS_E_OK;
  if (!a->q.ptr || !a->k.ptr || !a->v.ptr || !a->out.ptr || !a->lse || !a->dout.ptr ||
      !a->dq.ptr || !a->dk.ptr || !a->dv.ptr || !work)
    return POTS_E_ARG;
  for (const pots_heads* x : {&a->q, &a->k, &a->v, &a->out, &a->dout, &a->dq, &a->dk, &a->dv})
    if (!aligned(a, *x)) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool split = cut(a).split;
  char* w = static_cast<char*>(work);
  return a->dtype == POTS_OP_BF16 ? POTS_DIMS(Bf16, backward, a, w, s)
                                  : POTS_DIMS(Fp32, backward, a, w, s);
}
