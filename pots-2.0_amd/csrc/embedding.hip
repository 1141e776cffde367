// Rows of a table by token, scaled, and the table's gradient by sorted tokens.
//
//   out_i = scale·table[id_i]        dtable_v (+)= scale · Σ_{i: id_i = v} dout_i
//
// Both are bound by memory: 8192 rows of 1536 in fp32 out of a table of 151936 take 14.6 us (6.9
// TB/s, part of it out of the last cache), the dense gradient of the same 185 us (983 MB, 5.3 TB/s,
// which a copy does not exceed). Few tokens are bound by the launches, 5 us each.
//
// No result depends on atomics: the tokens are sorted by (id, position), the sorted list is cut into
// equal pieces whatever the ids' frequencies, and each piece adds up its rows in registers, in the
// order of the positions. A row whose tokens lie within one piece is written right away; one that
// crosses pieces leaves fp32 sums that embed_join adds in order. (A dense gradient's pieces may be
// longer than those of one that is added to a table: cut. The same tokens' sums may then differ in
// their last bits.)
//
// Sorting: the keys (id above position, so all differ) are placed by counting. A block holds 32 of
// them and counts the smaller ones of their run, two instructions a pair: up to 16384 tokens are
// one run (8192 tokens 14 us; sorting networks of 2048 in LDS and a merge took 24). More are runs
// of 2048, merged up to 32 at a time, where a key's place is its own index plus, for each other
// run, the number of smaller keys there. A dense
// gradient's zeros are written beside the sums, to the rows that no token has.
#include <math.h>

#include "common.h"
#include "gmem.h"
#include "tiles.h"

namespace pots {

constexpr uint32_t kFew = 256;                    // tokens that every block orders for itself
constexpr uint32_t kOneRun = 16384, kRun = 2048;  // tokens of a single run; else of each run
constexpr uint32_t kMerge = 32;    // runs a pass merges
constexpr uint32_t kPiece = 16;    // sorted keys that a wave adds up, at the least
constexpr uint32_t kFill = 16;     // rows that a block writes zeros to
// The last cache before memory: a table that it holds is written through it (191 MB 25 us, past it
// 31), a larger one past it, which leaves it to the sums' reads (933 MB 208 us through it, 201 past).
constexpr uint64_t kCache = 256ull << 20;
constexpr uint32_t kNoRow = ~0u;   // the id of a token outside the table; sorts last

template <class T>
constexpr uint32_t kPer = 16 / sizeof(typename T::elem);  // values in a 16-byte chunk

template <class T>
using Chunk = typename T::elem __attribute__((ext_vector_type(kPer<T>)));

// A chunk from column c of a row of d, zero past its end.
template <class T>
__device__ __forceinline__ Chunk<T> load_chunk(const typename T::elem* p, uint32_t c, uint32_t d,
                                               bool vec) {
  if (vec) return gload<Chunk<T>>(p + c);
  Chunk<T> x;
#pragma unroll
  for (uint32_t j = 0; j < kPer<T>; j++)
    x[j] = c + j < d ? gload<typename T::elem>(p + c + j) : typename T::elem(0);
  return x;
}

template <class T>
__device__ __forceinline__ void get_chunk(const typename T::elem* p, uint32_t c, uint32_t d,
                                          bool vec, float (&v)[kPer<T>]) {
  const Chunk<T> x = load_chunk<T>(p, c, d, vec);
#pragma unroll
  for (uint32_t j = 0; j < kPer<T>; j++) v[j] = T::get(x[j]);
}

template <class T>
__device__ __forceinline__ void put_chunk(typename T::elem* p, uint32_t c, uint32_t d, bool vec,
                                          const float (&v)[kPer<T>]) {
  if (vec) {
    Chunk<T> x;
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++) x[j] = T::put(v[j]);
    gstore<Chunk<T>>(p + c, x);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++)
      if (c + j < d) gstore<typename T::elem>(p + c + j, T::put(v[j]));
  }
}

template <class T>
__global__ __launch_bounds__(256) void embed_rows(pots_embedding a, uint32_t cpr, bool vec) {
  const uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x;
  if (e >= (uint64_t)a.tokens * cpr) return;
  const uint32_t i = e / cpr, c = (e - (uint64_t)i * cpr) * kPer<T>;
  const int64_t id = gload<int64_t>(a.ids + i);
  float v[kPer<T>];
  if (id >= 0 && id < a.vocab) {
    get_chunk<T>(reinterpret_cast<const typename T::elem*>(a.table) + id * a.table_row, c, a.dim,
                 vec, v);
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++) v[j] *= a.scale;
  } else {
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++) v[j] = NAN;
  }
  put_chunk<T>(reinterpret_cast<typename T::elem*>(a.rows) + (int64_t)i * a.rows_row, c, a.dim,
               vec, v);
}

// Zeros to rows r0 .. r0 + kFill of a dense gradient (those before `end`), by a block; with keys,
// only to the rows that no token has, each looked up in the sorted list by one lane.
template <class T, uint32_t NT, bool PAST>
__device__ __forceinline__ void fill_rows_as(const pots_embedding& a, const uint64_t* keys,
                                             uint32_t r0, uint32_t end, uint32_t cpr,
                                             bool vec) {
  __shared__ uint32_t s_has[kFill];
  const uint32_t n = r0 < end ? min(kFill, end - r0) : 0;
  if (threadIdx.x < n) {
    const uint64_t key = (uint64_t)(r0 + threadIdx.x) << 32;
    uint32_t lo = 0, hi = keys ? a.tokens : 0;
    while (lo < hi) {
      const uint32_t mid = lo + (hi - lo) / 2;
      if (keys[mid] < key)
        lo = mid + 1;
      else
        hi = mid;
    }
    s_has[threadIdx.x] =
        keys && lo < a.tokens && (uint32_t)(keys[lo] >> 32) == r0 + threadIdx.x;
  }
  __syncthreads();
  typename T::elem* table = reinterpret_cast<typename T::elem*>(a.table);
  const float zero[kPer<T>] = {};
  for (uint32_t e = threadIdx.x; e < n * cpr; e += NT) {
    const uint32_t r = e / cpr, c = (e - r * cpr) * kPer<T>;
    if (s_has[r]) continue;
    typename T::elem* p = table + (int64_t)(r0 + r) * a.table_row;
    if (vec && PAST)
      __builtin_nontemporal_store(Chunk<T>{}, reinterpret_cast<Chunk<T>*>(p + c));
    else
      put_chunk<T>(p, c, a.dim, vec, zero);
  }
}

// The zeros of the blocks from `before` on, to rows r0 .. end; tables of 2^24 rows and more go round
// (fill_blocks). (Two loops of stores, since two stores of one loop that differ in this alone become
// one plain store.)
template <class T, uint32_t NT>
__device__ __forceinline__ void fill_rows(const pots_embedding& a, const uint64_t* keys,
                                          uint32_t before, uint32_t r0, uint32_t end,
                                          uint32_t cpr, bool vec) {
  const uint32_t step = (gridDim.x - before) * kFill;
  for (uint32_t r = r0 + (blockIdx.x - before) * kFill; r < end; r += step) {
    if ((uint64_t)a.vocab * cpr * 16 > kCache)
      fill_rows_as<T, NT, true>(a, keys, r, end, cpr, vec);
    else
      fill_rows_as<T, NT, false>(a, keys, r, end, cpr, vec);
    if (r + step < end) __syncthreads();  // every lane is done with what the block looked up
  }
}

// Places 32 keys a block within their run, each of them in a lane of both halves of every wave:
// 32 shares of the run. The run's keys before the block's own count where they are not above
// (equal ids keep their order), the ones after it where they are below. The blocks after the
// first `order` write zeros to the rows below `end`.
template <class T>
__global__ __launch_bounds__(1024) void embed_order(pots_embedding a,
                                                    uint64_t* __restrict__ keys, uint32_t run,
                                                    uint32_t order, uint32_t end, uint32_t cpr,
                                                    bool vec) {
  constexpr uint32_t kOwn = 32, G = 16;  // keys of a block; keys compared per step
  __shared__ __attribute__((aligned(16))) uint32_t s_id[kOneRun];
  __shared__ uint32_t s_count[32][kOwn];
  if (blockIdx.x >= order) {
    fill_rows<T, 1024>(a, nullptr, order, 0, end, cpr, vec);
    return;
  }
  const uint32_t t = threadIdx.x, lane = t % kOwn, part = t / kOwn;
  const uint32_t own = blockIdx.x * kOwn, base = own / run * run, i = own + lane;
  const uint32_t n = min(run, a.tokens - base), n_pad = (n + G - 1) / G * G;
  for (uint32_t j = t; j < n_pad; j += 1024) {
    const int64_t id = j < n ? gload<int64_t>(a.ids + base + j) : -1;
    s_id[j] = id >= 0 && id < a.vocab ? (uint32_t)id : kNoRow;
  }
  __syncthreads();
  // (past the run's end a key compares as one that comes after all others)
  const uint32_t id = s_id[min(own - base + lane, n_pad - 1)], o0 = (own - base) / G * G;
  const uint32_t share = (n_pad / G + 31) / 32 * G;
  const uint32_t j0 = min(part * share, n_pad), j1 = min(j0 + share, n_pad);
  uint32_t count = 0;
  for (uint32_t j = j0; j < j1; j += G) {
    u32x4v o[G / 4];
#pragma unroll
    for (uint32_t x = 0; x < G / 4; x++) o[x] = reinterpret_cast<const u32x4v*>(s_id + j)[x];
    if (j < o0) {
#pragma unroll
      for (uint32_t x = 0; x < G; x++) count += o[x / 4][x % 4] <= id;
    } else if (j >= own - base + kOwn) {
#pragma unroll
      for (uint32_t x = 0; x < G; x++) count += o[x / 4][x % 4] < id;
    } else {
#pragma unroll
      for (uint32_t x = 0; x < G; x++)
        count += o[x / 4][x % 4] < id || (o[x / 4][x % 4] == id && base + j + x < i);
    }
  }
  s_count[part][lane] = count;
  __syncthreads();
  if (part != 0 || i >= a.tokens) return;
#pragma unroll
  for (uint32_t w = 1; w < 32; w++) count += s_count[w][lane];
  keys[base + count] = (uint64_t)id << 32 | i;
}

// Runs of `run` keys into runs of up to kMerge times as many.
__global__ __launch_bounds__(256) void embed_merge(const uint64_t* __restrict__ from,
                                                   uint64_t* __restrict__ to, uint32_t n,
                                                   uint64_t run) {
  const uint32_t i = blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const uint64_t key = from[i], group = i / (run * kMerge) * run * kMerge;
  uint64_t at = i % run;
  for (uint64_t r = group; r < n && r < group + run * kMerge; r += run) {
    if (r == i / run * run) continue;
    uint64_t lo = r, hi = r + run < n ? r + run : n;
    while (lo < hi) {
      const uint64_t mid = (lo + hi) / 2;
      if (from[mid] < key)
        lo = mid + 1;
      else
        hi = mid;
    }
    at += lo - r;
  }
  to[group + at] = key;
}

// Below `sums` waves: one adds up one piece of the sorted list for 64 chunks of columns. part:
// [piece][2][dim padded to chunks]: the sum of the row that an earlier piece began, and of the one
// that goes on. The blocks after those write zeros to rows from `r0` to `end` that no token has.
// FEW: up to kFew tokens, whose order each block finds in its LDS (one launch less, 5 us); the
// first leaves it in `keys` for embed_join.
template <class T, bool FEW, bool ADD, bool VEC>
__global__ __launch_bounds__(256) void embed_sum(pots_embedding a, uint64_t* __restrict__ list,
                                                 uint32_t piece, uint32_t groups, uint32_t sums,
                                                 uint32_t cpr, uint32_t r0, uint32_t end,
                                                 float* __restrict__ part) {
  constexpr uint32_t P = kPer<T>;
  const typename T::elem* rows = reinterpret_cast<const typename T::elem*>(a.rows);
  typename T::elem* table = reinterpret_cast<typename T::elem*>(a.table);
  const uint32_t blocks = (sums + 3) / 4;
  __shared__ uint64_t s_list[FEW ? kFew : 1];
  if constexpr (FEW) {
    __shared__ __attribute__((aligned(16))) uint32_t s_id[kFew];
    const uint32_t t = threadIdx.x;
    const int64_t own = t < a.tokens ? gload<int64_t>(a.ids + t) : -1;
    const uint32_t id = own >= 0 && own < a.vocab ? (uint32_t)own : kNoRow;
    s_id[t] = id;
    __syncthreads();
    uint32_t at = 0;
    for (uint32_t j = 0; j < a.tokens; j += 4) {  // (what lies past the last token comes after it)
      const u32x4v o = *reinterpret_cast<const u32x4v*>(s_id + j);
#pragma unroll
      for (uint32_t x = 0; x < 4; x++) at += o[x] < id || (o[x] == id && j + x < t);
    }
    if (t < a.tokens) {
      s_list[at] = (uint64_t)id << 32 | t;
      if (blockIdx.x == 0) list[at] = (uint64_t)id << 32 | t;
    }
    __syncthreads();
  }
  const uint64_t* const keys = FEW ? s_list : list;
  if (blockIdx.x >= blocks) {
    fill_rows<T, 256>(a, keys, blocks, r0, end, cpr, VEC);
    return;
  }
  const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (unit >= sums) return;
  const uint32_t b = unit / groups, ch = unit % groups * 64 + threadIdx.x % 64, c = ch * P;
  const uint32_t k0 = b * piece, k1 = min(k0 + piece, a.tokens);
  const bool on = ch < cpr;
  const uint32_t cl = on ? c : 0;  // the columns that a lane without any loads
  float sum[P] = {};
  // a row that an earlier piece began does not start here
  bool begun = k0 > 0 && (uint32_t)(keys[k0 - 1] >> 32) == (uint32_t)(keys[k0] >> 32);
  constexpr uint32_t U = kPiece;  // rows on their way at once
  for (uint32_t k = k0; k < k1; k += U) {
    Chunk<T> v[U], old[U];
    uint32_t id[U + 1], at[U];
#pragma unroll
    for (uint32_t u = 0; u <= U; u++) {
      const uint64_t key = k + u < a.tokens ? keys[k + u] : ~0ull;
      id[u] = key >> 32;
      if (u < U) at[u] = id[u] == kNoRow ? 0 : (uint32_t)key;
    }
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {  // (no branch between the loads: some are not used)
      v[u] = load_chunk<T>(rows + (int64_t)at[u] * a.rows_row, cl, a.dim, VEC);
      if (ADD) {
        const uint32_t row = id[u] == kNoRow ? 0 : id[u];
        old[u] = load_chunk<T>(table + (int64_t)row * a.table_row, cl, a.dim, VEC);
      }
    }
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
      if (k + u >= k1 || id[u] == kNoRow) continue;
#pragma unroll
      for (uint32_t j = 0; j < P; j++) sum[j] += T::get(v[u][j]);
      const bool ends = id[u + 1] != id[u], last = k + u + 1 == k1;
      if (!ends && !last) continue;
      if (on) {
        if (ends && !begun) {
          float y[P];
#pragma unroll
          for (uint32_t j = 0; j < P; j++)
            y[j] = ADD ? T::get(old[u][j]) + sum[j] * a.scale : sum[j] * a.scale;
          put_chunk<T>(table + (int64_t)id[u] * a.table_row, c, a.dim, VEC, y);
        } else {
          float* p = part + ((uint64_t)b * 2 + (begun ? 0 : 1)) * cpr * P + c;
#pragma unroll
          for (uint32_t j = 0; j < P; j++) p[j] = sum[j];
        }
      }
#pragma unroll
      for (uint32_t j = 0; j < P; j++) sum[j] = 0.f;
      begun = false;
    }
  }
}

// The rows that cross pieces, by the piece in which they begin, a wave for 64 chunks of
// columns; the blocks after the first `sums` waves' write zeros from `r0` on.
template <class T>
__global__ __launch_bounds__(256) void embed_join(pots_embedding a,
                                                  const uint64_t* __restrict__ keys,
                                                  uint32_t piece, uint32_t groups, uint32_t sums,
                                                  uint32_t cpr, uint32_t r0,
                                                  const float* __restrict__ part, bool vec) {
  constexpr uint32_t P = kPer<T>;
  const uint32_t blocks = (sums + 3) / 4;
  if (blockIdx.x >= blocks) {
    fill_rows<T, 256>(a, keys, blocks, r0, a.vocab, cpr, vec);
    return;
  }
  const uint32_t unit = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  if (unit >= sums) return;
  const uint32_t own = unit / groups, ch = unit % groups * 64 + threadIdx.x % 64, c = ch * P;
  const uint32_t k0 = own * piece, k1 = min(k0 + piece, a.tokens);
  if (k1 >= a.tokens || ch >= cpr) return;
  const uint32_t id = keys[k1 - 1] >> 32;
  if (id == kNoRow || (uint32_t)(keys[k1] >> 32) != id) return;       // ends here
  if ((uint32_t)(keys[k0] >> 32) == id && k0 > 0 && (uint32_t)(keys[k0 - 1] >> 32) == id)
    return;                                                           // began earlier
  float sum[P];
  const float* p = part + ((uint64_t)own * 2 + 1) * cpr * P + c;
#pragma unroll
  for (uint32_t j = 0; j < P; j++) sum[j] = p[j];
  constexpr uint32_t U = 8;  // pieces on their way at once
  for (uint64_t k = k1, b = own + 1;; k += U * piece, b += U) {
    bool in[U];
    float v[U][P];
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
      const uint64_t at = k + u * piece;
      in[u] = at < a.tokens && (uint32_t)(keys[at] >> 32) == id;
      const float* q = part + (at < a.tokens ? b + u : own) * 2 * cpr * P + c;
#pragma unroll
      for (uint32_t j = 0; j < P; j++) v[u][j] = q[j];
    }
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
#pragma unroll
      for (uint32_t j = 0; j < P; j++) sum[j] += in[u] ? v[u][j] : 0.f;
    if (!in[U - 1]) break;
  }
  typename T::elem* t = reinterpret_cast<typename T::elem*>(a.table) + (int64_t)id * a.table_row;
  float y[P] = {};
  if (a.add) get_chunk<T>(t, c, a.dim, vec, y);
#pragma unroll
  for (uint32_t j = 0; j < P; j++) y[j] = y[j] + sum[j] * a.scale;
  put_chunk<T>(t, c, a.dim, vec, y);
}

namespace {

bool bad(const pots_embedding* a) {
  return !a || a->dtype > POTS_OP_BF16 || a->dim == 0 || a->vocab == 0 || a->dim > 1u << 20 ||
         a->tokens > 1u << 24 || a->vocab > 1u << 30 || !isfinite(a->scale);
}

uint32_t per_chunk(const pots_embedding* a) { return a->dtype == POTS_OP_BF16 ? 8 : 4; }

bool chunked(const pots_embedding* a) {
  const uint32_t per = per_chunk(a);
  return a->dim % per == 0 && a->table_row % per == 0 && a->rows_row % per == 0 &&
         reinterpret_cast<uint64_t>(a->table) % 16 == 0 &&
         reinterpret_cast<uint64_t>(a->rows) % 16 == 0;
}

// Blocks that write zeros to so many rows; no more than a launch has room for beside its others
// (less than 2^32 threads).
uint32_t fill_blocks(uint32_t rows) {
  const uint32_t blocks = (rows + kFill - 1) / kFill;
  return blocks < 1u << 20 ? blocks : 1u << 20;
}

struct Cut {
  uint32_t cpr, order, run, piece, pieces;
  uint64_t keys, part, bytes;  // `keys` bytes of one list; two of them, then the sums
};

// Pieces: short ones so that few tokens still spread over the GPU, longer ones so that their
// sums stay a small part of the rows; four times as long where the zeros of a dense gradient
// (64 MiB or more) take longer than the sums beside them, for fewer rows to join after.
Cut cut(const pots_embedding* a) {
  Cut c;
  c.cpr = (a->dim + per_chunk(a) - 1) / per_chunk(a);
  c.order = (a->tokens + 31) / 32;
  c.run = a->tokens <= kOneRun ? kOneRun : kRun;
  c.piece = kPiece;
  if (!a->add && (uint64_t)a->vocab * c.cpr * 16 >= 64ull << 20) c.piece *= 4;
  while (c.piece < 2048 && a->tokens / c.piece > 1024) c.piece *= 2;
  c.pieces = (a->tokens + c.piece - 1) / c.piece;
  c.keys = align_up(8ull * a->tokens, 256);
  c.part = 2ull * c.pieces * c.cpr * per_chunk(a) * 4;
  c.bytes = 2 * c.keys + c.part;
  return c;
}

template <class T>
int forward(const pots_embedding* a, hipStream_t s) {
  const uint32_t cpr = (a->dim + kPer<T> - 1) / kPer<T>;
  const uint32_t most = (1u << 31) / cpr;  // tokens of a launch, which has less than 2^32 threads
  const bool vec = chunked(a);
  for (uint32_t t0 = 0; t0 < a->tokens; t0 += most) {
    pots_embedding part = *a;
    part.ids += t0;
    part.rows = reinterpret_cast<typename T::elem*>(a->rows) + (int64_t)t0 * a->rows_row;
    part.tokens = a->tokens - t0 < most ? a->tokens - t0 : most;
    const uint32_t nb = (uint32_t)(((uint64_t)part.tokens * cpr + 255) / 256);
    hipLaunchKernelGGL((embed_rows<T>), dim3(nb), dim3(256), 0, s, part, cpr, vec);
    POTS_HIP(hipGetLastError());
  }
  return POTS_E_OK;
}

template <class T>
auto sum_kernel(bool few, bool add, bool vec) {
  if (vec)
    return few ? (add ? embed_sum<T, true, true, true> : embed_sum<T, true, false, true>)
               : (add ? embed_sum<T, false, true, true> : embed_sum<T, false, false, true>);
  return few ? (add ? embed_sum<T, true, true, false> : embed_sum<T, true, false, false>)
             : (add ? embed_sum<T, false, true, false> : embed_sum<T, false, false, false>);
}

template <class T>
int backward(const pots_embedding* a, char* work, hipStream_t s) {
  const Cut c = cut(a);
  const bool vec = chunked(a);
  uint64_t* from = reinterpret_cast<uint64_t*>(work);
  uint64_t* to = reinterpret_cast<uint64_t*>(work + c.keys);
  float* part = reinterpret_cast<float*>(work + 2 * c.keys);
  // The zeros of a dense gradient: a share beside each of the three launches. Ordering and joining
  // are short chains of dependent steps that would leave the memory idle, about as long as a
  // twelfth of a large table takes to write.
  const bool few = a->tokens <= kFew;
  const uint32_t r1 = a->add || few ? 0 : a->vocab / 12;
  const uint32_t r2 = a->add ? 0 : c.pieces > 1 ? a->vocab - r1 : a->vocab;
  if (!few) {
    hipLaunchKernelGGL((embed_order<T>), dim3(c.order + fill_blocks(r1)), dim3(1024), 0, s, *a,
                       from, c.run, c.order, r1, c.cpr, vec);
    POTS_HIP(hipGetLastError());
  }
  for (uint64_t run = c.run; run < a->tokens; run *= kMerge) {
    hipLaunchKernelGGL(embed_merge, dim3((a->tokens + 255) / 256), dim3(256), 0, s, from, to,
                       a->tokens, run);
    POTS_HIP(hipGetLastError());
    uint64_t* t = from;
    from = to;
    to = t;
  }
  const uint32_t groups = (c.cpr + 63) / 64, sums = c.pieces * groups, blocks = (sums + 3) / 4;
  if (blocks + fill_blocks(r2 - r1)) {
    const auto kernel = sum_kernel<T>(few, a->add, vec);
    hipLaunchKernelGGL(kernel, dim3(blocks + fill_blocks(r2 - r1)), dim3(256), 0, s, *a, from,
                       c.piece, groups, sums, c.cpr, r1, r2, part);
    POTS_HIP(hipGetLastError());
  }
  if (c.pieces > 1) {
    hipLaunchKernelGGL((embed_join<T>), dim3(blocks + (a->add ? 0 : fill_blocks(a->vocab - r2))),
                       dim3(256), 0, s, *a, from, c.piece, groups, sums, c.cpr, r2, part, vec);
    POTS_HIP(hipGetLastError());
  }
  return POTS_E_OK;
}

}  // namespace

}  // namespace pots

using namespace pots;

extern "C" int pots_embedding_forward(const pots_embedding* a, void* stream) {
  if (bad(a)) return POTS_E_ARG;
  if (a->tokens == 0) return POTS_E_OK;
  if (!a->ids || !a->table || !a->rows) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return a->dtype == POTS_OP_BF16 ? forward<Bf16>(a, s) : forward<Fp32>(a, s);
}

extern "C" uint64_t pots_embedding_backward_work(const pots_embedding* a) {
  return bad(a) ? 0 : cut(a).bytes;
}

extern "C" int pots_embedding_backward(const pots_embedding* a, void* work, void* stream) {
  if (bad(a) || !a->table) return POTS_E_ARG;
  if (a->tokens && (!a->ids || !a->rows || !work)) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* w = static_cast<char*>(work);
  return a->dtype == POTS_OP_BF16 ? backward<Bf16>(a, w, s) : backward<Fp32>(a, w, s);
}
