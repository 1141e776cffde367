// Rows of a table by token, scaled, and the table's gradient by sorted tokens.
//
//   out_i = scale·table[id_i]        dtable_v (+)= scale · Σ_{i: id_i = v} dout_i
//
// Both are bound by memory. The gradient's sums are taken in the order of the positions, so no
// result depends on atomics: the tokens are sorted by (id, position), the sorted list is cut
// into equal pieces whatever the ids' frequencies, and each piece adds up its rows in registers.
// A row whose tokens lie within one piece is written right away; one that crosses pieces leaves
// fp32 sums that embed_join adds in order.
//
// Sorting: a block sorts 2048 keys (id above position, so all differ) in LDS; runs are then
// merged up to 32 at a time, where a key's place is its own index plus, for each other run,
// the number of smaller keys there. A dense gradient's zeros are written by other blocks of the
// sort's launch.
#include <math.h>

#include "common.h"
#include "gmem.h"
#include "tiles.h"

namespace pots {

constexpr uint32_t kRun = 2048;    // keys a block sorts
constexpr uint32_t kMerge = 32;    // runs a pass merges
constexpr uint32_t kNoRow = ~0u;   // the id of a token outside the table; sorts last

template <class T>
constexpr uint32_t kPer = 16 / sizeof(typename T::elem);  // values in a 16-byte chunk

// A chunk's values as floats, from column c of a row of d.
template <class T>
__device__ __forceinline__ void get_chunk(const typename T::elem* p, uint32_t c, uint32_t d,
                                          bool vec, float (&v)[kPer<T>]) {
  if (vec) {
    typedef typename T::elem chunk __attribute__((ext_vector_type(kPer<T>)));
    const chunk x = gload<chunk>(p + c);
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++) v[j] = T::get(x[j]);
  } else {
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++)
      v[j] = c + j < d ? T::get(gload<typename T::elem>(p + c + j)) : 0.f;
  }
}

template <class T>
__device__ __forceinline__ void put_chunk(typename T::elem* p, uint32_t c, uint32_t d, bool vec,
                                          const float (&v)[kPer<T>]) {
  if (vec) {
    typedef typename T::elem chunk __attribute__((ext_vector_type(kPer<T>)));
    chunk x;
#pragma unroll
    for (uint32_t j = 0; j < kPer<T>; j++) x[j] = T::put(v[j]);
    gstore<chunk>(p + c, x);
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

// Blocks below `runs` sort a run each; the others write zeros to the table.
template <class T>
__global__ __launch_bounds__(1024) void embed_sort(pots_embedding a, uint64_t* __restrict__ keys,
                                                   uint32_t runs, uint32_t cpr, bool vec) {
  __shared__ uint64_t s_key[kRun];
  if (blockIdx.x >= runs) {
    const uint64_t all = (uint64_t)a.vocab * cpr, step = (uint64_t)(gridDim.x - runs) * 1024;
    const float zero[kPer<T>] = {};
    for (uint64_t e = (uint64_t)(blockIdx.x - runs) * 1024 + threadIdx.x; e < all; e += step) {
      const uint32_t r = e / cpr, c = (e - (uint64_t)r * cpr) * kPer<T>;
      put_chunk<T>(reinterpret_cast<typename T::elem*>(a.table) + (int64_t)r * a.table_row, c,
                   a.dim, vec, zero);
    }
    return;
  }
  const uint32_t base = blockIdx.x * kRun, t = threadIdx.x;
#pragma unroll
  for (uint32_t x = 0; x < kRun; x += 1024) {
    const uint32_t i = base + x + t;
    uint64_t key = ~0ull;
    if (i < a.tokens) {
      const int64_t id = gload<int64_t>(a.ids + i);
      key = (uint64_t)(id >= 0 && id < a.vocab ? (uint32_t)id : kNoRow) << 32 | i;
    }
    s_key[x + t] = key;
  }
  for (uint32_t size = 2; size <= kRun; size *= 2)
    for (uint32_t gap = size / 2; gap > 0; gap /= 2) {
      __syncthreads();
      const uint32_t lo = t / gap * 2 * gap + t % gap, hi = lo + gap;
      const uint64_t x = s_key[lo], y = s_key[hi];
      if ((x > y) == ((lo & size) == 0)) {
        s_key[lo] = y;
        s_key[hi] = x;
      }
    }
  __syncthreads();
#pragma unroll
  for (uint32_t x = 0; x < kRun; x += 1024)
    if (base + x + t < a.tokens) keys[base + x + t] = s_key[x + t];
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

// Adds up one piece of the sorted list for 64 chunks of columns. part: [piece][2][dim padded to
// chunks]: the sum of the row that an earlier piece began, and of the one that goes on.
template <class T>
__global__ __launch_bounds__(64) void embed_sum(pots_embedding a,
                                                const uint64_t* __restrict__ keys,
                                                uint32_t piece, uint32_t cpr,
                                                float* __restrict__ part, bool vec) {
  constexpr uint32_t P = kPer<T>;
  const uint32_t ch = blockIdx.y * 64 + threadIdx.x, c = ch * P;
  const uint32_t k0 = blockIdx.x * piece, k1 = min(k0 + piece, a.tokens);
  const bool on = ch < cpr;
  const typename T::elem* rows = reinterpret_cast<const typename T::elem*>(a.rows);
  typename T::elem* table = reinterpret_cast<typename T::elem*>(a.table);
  float sum[P] = {};
  // a row that an earlier piece began does not start here
  bool begun = k0 > 0 && (uint32_t)(keys[k0 - 1] >> 32) == (uint32_t)(keys[k0] >> 32);
  constexpr uint32_t U = 8;
  for (uint32_t k = k0; k < k1; k += U) {
    float v[U][P];
    uint32_t id[U + 1];
#pragma unroll
    for (uint32_t u = 0; u <= U; u++) id[u] = k + u < a.tokens ? keys[k + u] >> 32 : kNoRow;
#pragma unroll
    for (uint32_t u = 0; u < U; u++)
      if (on && k + u < k1 && id[u] != kNoRow)
        get_chunk<T>(rows + (int64_t)(uint32_t)keys[k + u] * a.rows_row, c, a.dim, vec, v[u]);
#pragma unroll
    for (uint32_t u = 0; u < U; u++) {
      if (k + u >= k1 || id[u] == kNoRow) continue;
#pragma unroll
      for (uint32_t j = 0; j < P; j++) sum[j] += v[u][j];
      const bool ends = id[u + 1] != id[u], last = k + u + 1 == k1;
      if (!ends && !last) continue;
      if (on) {
        if (ends && !begun) {
          typename T::elem* p = table + (int64_t)id[u] * a.table_row;
          float y[P] = {};
          if (a.add) get_chunk<T>(p, c, a.dim, vec, y);
#pragma unroll
          for (uint32_t j = 0; j < P; j++) y[j] = y[j] + sum[j] * a.scale;
          put_chunk<T>(p, c, a.dim, vec, y);
        } else {
          float* p = part + ((uint64_t)blockIdx.x * 2 + (begun ? 0 : 1)) * cpr * P + c;
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

// The rows that cross pieces, by the piece in which they begin.
template <class T>
__global__ __launch_bounds__(64) void embed_join(pots_embedding a,
                                                 const uint64_t* __restrict__ keys,
                                                 uint32_t piece, uint32_t cpr,
                                                 const float* __restrict__ part, bool vec) {
  constexpr uint32_t P = kPer<T>;
  const uint32_t ch = blockIdx.y * 64 + threadIdx.x, c = ch * P;
  const uint32_t k0 = blockIdx.x * piece, k1 = min(k0 + piece, a.tokens);
  if (k1 >= a.tokens || ch >= cpr) return;
  const uint32_t id = keys[k1 - 1] >> 32;
  if (id == kNoRow || (uint32_t)(keys[k1] >> 32) != id) return;       // ends here
  if ((uint32_t)(keys[k0] >> 32) == id && k0 > 0 && (uint32_t)(keys[k0 - 1] >> 32) == id)
    return;                                                           // began earlier
  float sum[P];
  const float* p = part + ((uint64_t)blockIdx.x * 2 + 1) * cpr * P + c;
#pragma unroll
  for (uint32_t j = 0; j < P; j++) sum[j] = p[j];
  for (uint64_t k = k1, b = blockIdx.x + 1; k < a.tokens && (uint32_t)(keys[k] >> 32) == id;
       k += piece, b++) {
    const float* q = part + b * 2 * cpr * P + c;
#pragma unroll
    for (uint32_t j = 0; j < P; j++) sum[j] += q[j];
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

struct Cut {
  uint32_t cpr, runs, piece, pieces;
  uint64_t keys, part, bytes;  // `keys` bytes of one list; two of them, then the sums
};

// Pieces: short ones so that few tokens still spread over the GPU, longer ones so that their
// sums stay a small part of the rows.
Cut cut(const pots_embedding* a) {
  Cut c;
  c.cpr = (a->dim + per_chunk(a) - 1) / per_chunk(a);
  c.runs = (a->tokens + kRun - 1) / kRun;
  c.piece = 16;
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
  const uint64_t nb = ((uint64_t)a->tokens * cpr + 255) / 256;
  if (nb > 0x7FFFFFFFu) return POTS_E_ARG;
  hipLaunchKernelGGL((embed_rows<T>), dim3((uint32_t)nb), dim3(256), 0, s, *a, cpr, chunked(a));
  POTS_HIP(hipGetLastError());
  return POTS_E_OK;
}

template <class T>
int backward(const pots_embedding* a, char* work, hipStream_t s) {
  const Cut c = cut(a);
  const bool vec = chunked(a);
  uint64_t* from = reinterpret_cast<uint64_t*>(work);
  uint64_t* to = reinterpret_cast<uint64_t*>(work + c.keys);
  float* part = reinterpret_cast<float*>(work + 2 * c.keys);
  uint32_t fill = 0;
  if (!a->add) {
    const uint64_t nb = ((uint64_t)a->vocab * c.cpr + 1023) / 1024;
    fill = (uint32_t)(nb < 4096 ? nb : 4096);
  }
  if (c.runs + fill == 0) return POTS_E_OK;
  hipLaunchKernelGGL((embed_sort<T>), dim3(c.runs + fill), dim3(1024), 0, s, *a, from, c.runs,
                     c.cpr, vec);
  POTS_HIP(hipGetLastError());
  if (a->tokens == 0) return POTS_E_OK;
  for (uint64_t run = kRun; run < a->tokens; run *= kMerge) {
    hipLaunchKernelGGL(embed_merge, dim3((a->tokens + 255) / 256), dim3(256), 0, s, from, to,
                       a->tokens, run);
    POTS_HIP(hipGetLastError());
    uint64_t* t = from;
    from = to;
    to = t;
  }
  const dim3 grid(c.pieces, (c.cpr + 63) / 64);
  hipLaunchKernelGGL((embed_sum<T>), grid, dim3(64), 0, s, *a, from, c.piece, c.cpr, part, vec);
  POTS_HIP(hipGetLastError());
  if (c.pieces > 1) {
    hipLaunchKernelGGL((embed_join<T>), grid, dim3(64), 0, s, *a, from, c.piece, c.cpr, part,
                       vec);
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
