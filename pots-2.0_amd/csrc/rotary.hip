// Rotary positions of queries and keys, on one axis or several.
//
//   (u, v) -> (u cos θ − v sin θ, u sin θ + v cos θ),  θ = position · frequency of the pair
//
// The gradient is the turn by −θ. Bound by memory: q and k are read and written once, in one
// launch. θ is taken in whole turns and their fraction in 64 bits, so that far positions lose
// nothing that fp32 would hold (frequency / 2π is off by 2^-53 and 2^-54 of its size, so θ by at most 2^-35 of a turn
// up to position 2^20 at frequencies up to 1); the sine and cosine of the fraction, less than
// an eighth of a turn, are fp32. A block computes them for a few tokens into LDS, once for all heads; its
// lanes then go over the tokens' heads, 16 bytes of u and 16 of v at a time, the first of them on their
// way meanwhile (those 8192 tokens in bf16 12.4 us a call, 4.7 TB/s; with angles of each lane's own and no
// LDS 16). Where the pairs are no multiple of such a run, the last run overlaps the one before it
// and writes the same values.
#include <math.h>

#include "common.h"
#include "gmem.h"
#include "tiles.h"
#include "values.h"

namespace pots {

constexpr uint32_t kMaxWidth = 1024, kMaxHeads = 1u << 16;
constexpr uint32_t kAngles = 1024, kTokens = 64;  // of a block, at the most
constexpr uint32_t kAhead = 2;  // runs that a lane has on their way

struct Turn {
  float c, s;
};

__device__ __forceinline__ Turn turn_of(double position, double frequency, bool inverse) {
  const double f = frequency * 0.15915494309189535;  // 1 / 2π
  const double r = fma(position, f, -rint(position * f));
  const double quarter = rint(4.0 * r);
  float s, c;
  sincospif((float)(2.0 * fma(quarter, -0.25, r)), &s, &c);
  const int q = (int)quarter & 3;  // a quarter turn: (c, s) to (-s, c)
  Turn t;
  t.c = q == 0 ? c : q == 1 ? -s : q == 2 ? -c : s;
  t.s = q == 0 ? s : q == 1 ? c : q == 2 ? -s : -c;
  if (inverse) t.s = -t.s;
  return t;
}

// A lane's part of a head: P pairs, of the two halves or beside each other, or 2P columns that are
// copied. lo and hi lie `apart`.
template <class T, uint32_t P, bool ADJACENT>
struct Piece {
  Run<T, P> lo, hi;

  __device__ __forceinline__ void load(const typename T::elem* p, uint32_t at, uint32_t apart) {
    lo = load_any<Run<T, P>>(p + at);
    hi = load_any<Run<T, P>>(p + at + apart);
  }
  __device__ __forceinline__ void store(typename T::elem* p, uint32_t at, uint32_t apart) const {
    store_any(p + at, lo);
    store_any(p + at + apart, hi);
  }
  // Fewer pairs than P, value by value.
  __device__ __forceinline__ void load_pairs(const typename T::elem* p, uint32_t apart,
                                             uint32_t pairs) {
#pragma unroll
    for (uint32_t j = 0; j + 1 < P; j++) {
      if (j >= pairs) break;
      if (ADJACENT) {
        Run<T, P>& r = j < P / 2 ? lo : hi;
        r[2 * j % P] = gload<typename T::elem>(p + 2 * j);
        r[2 * j % P + 1] = gload<typename T::elem>(p + 2 * j + 1);
      } else {
        lo[j] = gload<typename T::elem>(p + j);
        hi[j] = gload<typename T::elem>(p + apart + j);
      }
    }
  }
  __device__ __forceinline__ void store_pairs(typename T::elem* p, uint32_t apart,
                                              uint32_t pairs) const {
#pragma unroll
    for (uint32_t j = 0; j + 1 < P; j++) {
      if (j >= pairs) break;
      if (ADJACENT) {
        const Run<T, P>& r = j < P / 2 ? lo : hi;
        gstore<typename T::elem>(p + 2 * j, r[2 * j % P]);
        gstore<typename T::elem>(p + 2 * j + 1, r[2 * j % P + 1]);
      } else {
        gstore<typename T::elem>(p + j, lo[j]);
        gstore<typename T::elem>(p + apart + j, hi[j]);
      }
    }
  }
  // Fewer columns than 2P, in pieces of P, P / 2, ... 1 of them, as their count has them.
  template <uint32_t N, bool LOAD, class E>
  __device__ __forceinline__ void columns(E* p, uint32_t rest) {
    Run<T, P>& r = N == P ? lo : hi;
    constexpr uint32_t at = N == P ? 0 : P - 2 * N;
    if (rest & N) {
      E* const q = p + (rest & ~(2 * N - 1));
      Run<T, N> x;
      if constexpr (LOAD) {
        x = load_any<Run<T, N>>(q);
#pragma unroll
        for (uint32_t j = 0; j < N; j++) r[at + j] = x[j];
      } else {
#pragma unroll
        for (uint32_t j = 0; j < N; j++) x[j] = r[at + j];
        store_any(q, x);
      }
    }
    if constexpr (N > 1) columns<N / 2, LOAD>(p, rest);
  }
  __device__ __forceinline__ void turn(const Turn* t) {
#pragma unroll
    for (uint32_t j = 0; j < P; j++) {
      const Turn x = t[j];
      if (ADJACENT) {
        Run<T, P>& r = j < P / 2 ? lo : hi;
        const uint32_t at = 2 * j % P;
        const float u = T::get(r[at]), v = T::get(r[at + 1]);
        r[at] = T::put(fmaf(u, x.c, -(v * x.s)));
        r[at + 1] = T::put(fmaf(u, x.s, v * x.c));
      } else {
        const float u = T::get(lo[j]), v = T::get(hi[j]);
        lo[j] = T::put(fmaf(u, x.c, -(v * x.s)));
        hi[j] = T::put(fmaf(u, x.s, v * x.c));
      }
    }
  }
};

// FEW: a head has fewer pairs than P, or fewer other columns than 2P.
template <class T, uint32_t P, bool ADJACENT, bool FEW>
__global__ __launch_bounds__(256) void rotary_turn(pots_rotary a, uint32_t tokens, uint32_t from,
                                                   Divisor by_heads, Divisor by_pairs) {
  typedef typename T::elem elem;
  __shared__ Turn s_turn[kAngles + P];  // (a head of fewer pairs than P reads past its last one)
  // (fewer than 2^31 tokens in all)
  const uint32_t all = a.batch * a.n, t0 = from + blockIdx.x * tokens, here = min(all - t0, tokens);
  const uint32_t heads = a.heads + a.kv_heads, items = here * heads;
  const uint32_t b0 = t0 / a.n, n0 = t0 - b0 * a.n;
  // The block's token t: its sequence and its place there. (One division less where all are of one.)
  auto token = [&](uint32_t t, uint32_t& b, uint32_t& n) {
    b = b0, n = n0 + t;
    if (n >= a.n) {
      b += n / a.n;
      n %= a.n;
    }
  };
  auto place = [&](uint32_t item, uint32_t& t, const elem*& in, elem*& out) {
    t = by_heads.of(item);
    uint32_t h = item - t * heads, b, n;
    token(t, b, n);
    const bool key = h >= a.heads;
    if (key) h -= a.heads;
    const pots_heads& i = key ? a.k : a.q;
    const pots_heads& o = key ? a.k_out : a.q_out;
    in = reinterpret_cast<const elem*>(i.ptr) + b * i.batch + n * i.row + h * i.head;
    out = reinterpret_cast<elem*>(o.ptr) + b * o.batch + n * o.row + h * o.head;
  };
  // A head's runs: those of its pairs, then those of the columns that are copied.
  const uint32_t turned = a.pairs < P ? 1 : (a.pairs + P - 1) / P;
  const uint32_t rest = a.head_dim - 2 * a.pairs;
  const uint32_t runs = turned + (rest < 2 * P ? rest != 0 : (rest + 2 * P - 1) / (2 * P));
  const uint32_t slots = 256 / runs, slot = threadIdx.x / runs, run = threadIdx.x - slot * runs;
  const bool turns = run < turned, whole = !FEW || (turns ? a.pairs >= P : rest >= 2 * P);
  const uint32_t i0 = a.pairs >= P ? min(run * P, a.pairs - P) : 0;
  const uint32_t c0 = rest >= 2 * P ? min((run - turned) * 2 * P, rest - 2 * P) : 0;
  const uint32_t at = !turns ? 2 * a.pairs + c0 : ADJACENT ? 2 * i0 : i0;
  const uint32_t apart = turns && !ADJACENT ? a.pairs : P;
  const uint32_t first = slot < slots ? slot : items;  // (lanes past the last slot have no item)
  Piece<T, P, ADJACENT> x[kAhead];
  if (FEW)
    for (uint32_t j = 0; j < kAhead; j++) x[j] = {};
  elem* out[kAhead];
  uint32_t t[kAhead];
  auto load = [&](uint32_t item) {
#pragma unroll
    for (uint32_t j = 0; j < kAhead; j++) {
      const elem* in;  // (past the last item: that one again, and nothing is stored)
      place(min(item + j * slots, items - 1), t[j], in, out[j]);
      if (whole)
        x[j].load(in, at, apart);
      else if (turns)
        x[j].load_pairs(in, apart, a.pairs);
      else
        x[j].template columns<P, true>(in + at, rest);
    }
  };
  if (first < items) load(first);  // on their way while the angles are taken
  for (uint32_t e = threadIdx.x; e < here * a.pairs; e += 256) {
    const uint32_t t = by_pairs.of(e), i = e - t * a.pairs;
    uint32_t b, n, axis = 0;
    token(t, b, n);
    for (uint32_t x = 0; x + 1 < a.axes; x++) axis += i >= a.ends[x];
    const int64_t at = axis * a.position_axis + b * a.position_batch + n * a.position_token;
    const double position =
        a.position_bits == 64
            ? (double)gload<int64_t>(reinterpret_cast<const int64_t*>(a.positions) + at)
            : (double)gload<int32_t>(reinterpret_cast<const int32_t*>(a.positions) + at);
    const double f = a.frequency_type == POTS_OP_F64
                         ? gload<double>(reinterpret_cast<const double*>(a.frequencies) + i)
                         : (double)gload<float>(reinterpret_cast<const float*>(a.frequencies) + i);
    s_turn[e] = turn_of(position, f, a.inverse);
  }
  __syncthreads();
  for (uint32_t item = first; item < items; item += kAhead * slots) {
    if (item != first) load(item);
#pragma unroll
    for (uint32_t j = 0; j < kAhead; j++) {
      if (turns) x[j].turn(s_turn + t[j] * a.pairs + i0);
      if (item + j * slots >= items) continue;
      if (whole)
        x[j].store(out[j], at, apart);
      else if (turns)
        x[j].store_pairs(out[j], apart, a.pairs);
      else
        x[j].template columns<P, false>(out[j] + at, rest);
    }
  }
}

namespace {

bool bad(const pots_rotary* a) {
  if (!a || a->dtype > POTS_OP_BF16 || a->head_dim == 0 || a->head_dim > kMaxWidth ||
      a->pairs == 0 || 2 * a->pairs > a->head_dim || a->pairs > kMaxWidth || a->axes == 0 ||
      a->axes > 4 || a->heads == 0 || a->kv_heads == 0 || a->heads > kMaxHeads ||
      a->kv_heads > kMaxHeads || (uint64_t)a->batch * a->n > 0x7fffffffu)
    return true;
  if (a->frequency_type != POTS_OP_F32 && a->frequency_type != POTS_OP_F64) return true;
  if (a->position_bits != 32 && a->position_bits != 64) return true;
  for (uint32_t x = 1; x < a->axes; x++)
    if (a->ends[x] < a->ends[x - 1]) return true;
  return a->ends[a->axes - 1] != a->pairs;
}

template <class T, uint32_t P>
int turn(const pots_rotary* a, hipStream_t s) {
  // Tokens of a block: few enough for eight blocks to a compute unit (8192 tokens of 14 heads of 128, two
  // calls in a graph: 30.5 us; four blocks 32.7, sixteen 34.1), as many as their angles allow.
  const uint64_t all = (uint64_t)a->batch * a->n;
  uint64_t tokens = all / 2048;
  const uint32_t most = kAngles / a->pairs < kTokens ? kAngles / a->pairs : kTokens;
  tokens = tokens < 1 ? 1 : tokens > most ? most : tokens;
  const uint32_t rest = a->head_dim - 2 * a->pairs;
  const bool few = a->pairs < P || (rest && rest < 2 * P);
  const auto kernel =
      few ? (a->adjacent ? rotary_turn<T, P, true, true> : rotary_turn<T, P, false, true>)
          : (a->adjacent ? rotary_turn<T, P, true, false> : rotary_turn<T, P, false, false>);
  constexpr uint64_t kLaunch = 1u << 23;  // blocks: a launch has less than 2^32 threads
  for (uint64_t from = 0; from < all; from += kLaunch * tokens) {
    const uint64_t blocks = (all - from + tokens - 1) / tokens;
    hipLaunchKernelGGL(kernel, dim3((uint32_t)(blocks < kLaunch ? blocks : kLaunch)), dim3(256), 0, s,
                       *a, (uint32_t)tokens, (uint32_t)from, Divisor(a->heads + a->kv_heads), Divisor(a->pairs));
    POTS_HIP(hipGetLastError());
  }
  return POTS_E_OK;
}

}  // namespace

}  // namespace pots

using namespace pots;

extern "C" int pots_rotary_turn(const pots_rotary* a, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (a->batch == 0 || a->n == 0) return POTS_E_OK;
  if (!a->q.ptr || !a->k.ptr || !a->q_out.ptr || !a->k_out.ptr || !a->positions || !a->frequencies)
    return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (a->dtype != POTS_OP_BF16) return turn<Fp32, 4>(a, s);
  return a->pairs >= 8 ? turn<Bf16, 8>(a, s) : turn<Bf16, 4>(a, s);
}
