// The 2-norm of a whole model's gradient, and what a step does with it: the gradient scaled by the
// clip's factor, or the weights updated by it.
//
//   norm = √Σ g²,  f = min(1, max_norm / norm),  out = f·g  or  out = w − (η f)·g
//
// An infinite max_norm is no bound: f is 1 whatever the norm, so that a value that is not finite stays its
// own weight's affair.
//
// Bound by memory, and the gradient is read twice: the factor needs all of it first. The second pass
// goes backwards, so that what the first read last is still in the last cache. Squares are added in
// fp64, which no fp32 gradient leaves: 3.4e38² is 1e77, and the smallest one's square 2e-90.
//
// The tensors' addresses travel as kernel arguments, kNormed or kUpdated tensors a launch: a captured
// graph keeps them, and no copy to the device precedes the work. Tensors are cut into chunks; block b of
// g takes the chunks b, b + g, ... and leaves one sum, and the blocks of the second pass each add up all
// sums in the same order.
#include <math.h>

#include <algorithm>
#include <vector>

#include "common.h"
#include "gmem.h"
#include "tiles.h"
#include "values.h"

namespace pots {

// Values of a chunk: 16 KiB of the gradient, four or eight runs of four to each of 256 lanes, which are all
// on their way at once.
constexpr uint32_t kRuns32 = 4, kRuns16 = 8;
__host__ __device__ constexpr uint32_t chunk_values(uint32_t type) {
  return 1024 * (type == POTS_OP_BF16 ? kRuns16 : kRuns32);
}
// Tensors of a launch: below 4 KiB of arguments, or a third of that for few (each KiB of arguments
// takes the host half a microsecond).
constexpr uint32_t kNormed = 160, kUpdated = 96, kFewTensors = 32;
// Four to a compute unit: the update of 1.54e9 fp32 weights takes 4.30 ms, with eight 4.43.
constexpr uint32_t kBlocks = 1024;
// The last cache is left to the chunks that the second pass begins with, 192 MiB: what comes
// before them is read past it, and so is all that the second pass reads and writes if there is more
// than that (1.54e9 weights: 4.68 ms all through it, 4.30 so; a clip of 1.35e8 gradients 335 and 276
// us). A smaller gradient's results stay there for whoever reads them next.
constexpr uint64_t kKept = 12288;
constexpr uint32_t kMostTensors = 1u << 16;

template <uint32_t N>
struct alignas(16) Normed {
  static constexpr uint32_t kMost = N;
  const void* g[N];
  uint64_t count[N];
  uint32_t first[N];  // chunk
  uint8_t type[N];
  uint32_t tensors, chunks, kept;  // the chunks from `kept` on stay in the cache
};

template <uint32_t N>
struct alignas(16) Updated {
  static constexpr uint32_t kMost = N;
  const void *g[N], *w[N];
  void* out[N];
  uint64_t count[N];
  uint32_t first[N];
  uint8_t type[N], weight_type[N];
  uint32_t tensors, chunks, past;
};

__device__ __forceinline__ double sum_block(double v, double* s) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v += __shfl_xor(v, m);
  if (threadIdx.x % 64 == 0) s[threadIdx.x / 64] = v;
  __syncthreads();
  return s[0] + s[1] + s[2] + s[3];
}

// A launch's table, from its arguments to LDS: the look-ups in it are one after the other, and each from
// the arguments would wait for memory.
template <class TABLE>
__device__ __forceinline__ void table_to_lds(const TABLE& t, TABLE& to) {
  static_assert(sizeof(TABLE) % 16 == 0 && sizeof(TABLE) <= 4096, "a run of 16 bytes to each lane");
  const u32x4v* const from = reinterpret_cast<const u32x4v*>(&t);
  if (threadIdx.x < sizeof(TABLE) / 16)
    reinterpret_cast<u32x4v*>(&to)[threadIdx.x] = from[threadIdx.x];
  __syncthreads();
}

// The tensor that chunk c lies in, of those that start at the chunks first[0 .. n).
__device__ __forceinline__ uint32_t tensor_of(const uint32_t* first, uint32_t n, uint32_t c) {
  uint32_t lo = 0;
  while (n > 1) {
    const uint32_t half = n / 2;
    if (first[lo + half] <= c) lo += half;
    n -= half;
  }
  return lo;
}

// A lane's R runs of the chunk that starts at value `at` of a tensor of `count`.
template <class T, uint32_t R, bool PAST>
__device__ __forceinline__ void chunk_of(const void* p, uint64_t at, uint64_t count,
                                         float (&v)[R][4]) {
  const typename T::elem* q = reinterpret_cast<const typename T::elem*>(p) + at;
  Run<T, 4> x[R];
  if (count - at >= 1024 * R) {
#pragma unroll
    for (uint32_t i = 0; i < R; i++) {
      const typename T::elem* const r = q + 4 * threadIdx.x + 1024 * i;
      x[i] = PAST ? load_past<Run<T, 4>>(r) : load_any<Run<T, 4>>(r);
    }
  } else {
    load_runs<T, 4, R>(q, 4 * threadIdx.x, 1024, (uint32_t)(count - at), x);
  }
#pragma unroll
  for (uint32_t i = 0; i < R; i++)
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) v[i][j] = T::get(x[i][j]);
}

template <uint32_t R, bool PAST>
__device__ __forceinline__ void chunk_of(const void* p, uint32_t type, uint64_t at, uint64_t count,
                                         float (&v)[R][4]) {
  if (type == POTS_OP_BF16)
    chunk_of<Bf16, R, PAST>(p, at, count, v);
  else
    chunk_of<Fp32, R, PAST>(p, at, count, v);
}

template <class T, uint32_t R, bool PAST, class TABLE>
__device__ __forceinline__ void add_squares(const TABLE& t, uint32_t i, uint64_t at,
                                            double (&sum)[4]) {
  float v[R][4];
  chunk_of<T, R, PAST>(t.g[i], at, t.count[i], v);
#pragma unroll
  for (uint32_t r = 0; r < R; r++)
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) sum[j] = fma((double)v[r][j], (double)v[r][j], sum[j]);
}

template <class TABLE>
__global__ __launch_bounds__(256) void norm_sums(TABLE args, double* __restrict__ part) {
  __shared__ double s_sum[4];
  __shared__ TABLE t;
  table_to_lds(args, t);
  double sum[4] = {};
  uint32_t i = tensor_of(t.first, t.tensors, blockIdx.x);
  for (uint32_t c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    while (i + 1 < t.tensors && c >= t.first[i + 1]) i++;
    const uint64_t at = (uint64_t)(c - t.first[i]) * chunk_values(t.type[i]);
    if (t.type[i] == POTS_OP_BF16) {
      if (c < t.kept)
        add_squares<Bf16, kRuns16, true>(t, i, at, sum);
      else
        add_squares<Bf16, kRuns16, false>(t, i, at, sum);
    } else {
      if (c < t.kept)
        add_squares<Fp32, kRuns32, true>(t, i, at, sum);
      else
        add_squares<Fp32, kRuns32, false>(t, i, at, sum);
    }
  }
  const double all = sum_block((sum[0] + sum[1]) + (sum[2] + sum[3]), s_sum);
  if (threadIdx.x == 0) part[blockIdx.x] = all;
}

__device__ __forceinline__ double norm_of(const double* part, uint32_t parts, double* s) {
  double v = 0.;
  for (uint32_t i = threadIdx.x; i < parts; i += 1024) {
    double x[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++)
      x[j] = i + 256 * j < parts ? gload<double>(part + i + 256 * j) : 0.;
    v += (x[0] + x[1]) + (x[2] + x[3]);
  }
  return sqrt(sum_block(v, s));
}

__global__ __launch_bounds__(256) void norm_write(const double* __restrict__ part, uint32_t parts,
                                                  float* norm) {
  __shared__ double s_sum[4];
  const double n = norm_of(part, parts, s_sum);
  if (threadIdx.x == 0) *norm = (float)n;
}

template <bool STEP, uint32_t R, bool PAST, class TABLE>
__device__ __forceinline__ void update_chunk(const TABLE& t, uint32_t i, uint64_t at, float f) {
  const uint64_t count = t.count[i];
  float g[R][4], w[R][4];
  chunk_of<R, PAST>(t.g[i], t.type[i], at, count, g);
  if (STEP) chunk_of<R, PAST>(t.w[i], t.weight_type[i], at, count, w);
  const uint32_t left = count - at < 1024 * R ? (uint32_t)(count - at) : 1024 * R;
  const uint32_t type = STEP ? t.weight_type[i] : t.type[i];
#pragma unroll
  for (uint32_t r = 0; r < R; r++) {
    const uint32_t c = 4 * threadIdx.x + 1024 * r;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) g[r][j] = STEP ? fmaf(f, g[r][j], w[r][j]) : f * g[r][j];
    put_run<4, PAST>(t.out[i], type, (int64_t)at + c, left > c ? left - c : 0, g[r]);
  }
}

// STEP: w - eta·f·g, else f·g. The launch that writes the norm has its address.
template <bool STEP, class TABLE>
__global__ __launch_bounds__(256) void update(TABLE args, const double* __restrict__ part,
                                              uint32_t parts, float max_norm, float eta, float* norm) {
  __shared__ double s_sum[4];
  __shared__ TABLE t;
  table_to_lds(args, t);
  const double n = norm_of(part, parts, s_sum);
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)n;
  const double factor =
      n <= (double)max_norm || max_norm == INFINITY ? 1. : (double)max_norm / n;
  const float f = (float)(STEP ? -(double)eta * factor : factor);
  if (blockIdx.x >= t.chunks) return;
  const uint32_t last = (t.chunks - 1 - blockIdx.x) / gridDim.x * gridDim.x + blockIdx.x;
  uint32_t i = tensor_of(t.first, t.tensors, last);
  for (uint32_t k = 0; k <= last / gridDim.x; k++) {
    const uint32_t c = last - k * gridDim.x;
    while (c < t.first[i]) i--;
    const uint64_t at = (uint64_t)(c - t.first[i]) * chunk_values(t.type[i]);
    if (t.type[i] == POTS_OP_BF16) {
      if (t.past)
        update_chunk<STEP, kRuns16, true>(t, i, at, f);
      else
        update_chunk<STEP, kRuns16, false>(t, i, at, f);
    } else {
      if (t.past)
        update_chunk<STEP, kRuns32, true>(t, i, at, f);
      else
        update_chunk<STEP, kRuns32, false>(t, i, at, f);
    }
  }
}

namespace {

const pots_gradient* entries(const pots_gradients* a) {
  return reinterpret_cast<const pots_gradient*>(a + 1);
}

uint64_t chunks_of(const pots_gradient& e) {
  const uint32_t values = chunk_values(e.gradient_type);
  return (e.count + values - 1) / values;
}

uint64_t chunks_of(const pots_gradients* a) {
  uint64_t chunks = 0;
  for (uint32_t i = 0; i < a->tensors; i++) chunks += chunks_of(entries(a)[i]);
  return chunks;
}

bool bad(const pots_gradients* a, bool clips, bool steps) {
  if (!a || a->tensors == 0 || a->tensors > kMostTensors) return true;
  if (clips && !(a->max_norm > 0.f)) return true;
  if (steps && !isfinite(a->eta)) return true;
  for (uint32_t i = 0; i < a->tensors; i++) {
    const pots_gradient& e = entries(a)[i];
    if (e.gradient_type > POTS_OP_BF16 || (steps && e.weight_type > POTS_OP_BF16) ||
        e.count > 1ull << 42)
      return true;
  }
  return chunks_of(a) > 0x7fffffffu;
}

// The entries that hold something, `most` of them at a time: f(their indices, how many).
template <class F>
int each_launch(const pots_gradients* a, uint32_t most, F&& f) {
  std::vector<uint32_t> some;
  some.reserve(a->tensors);
  for (uint32_t i = 0; i < a->tensors; i++)
    if (entries(a)[i].count) some.push_back(i);
  for (size_t at = 0; at < some.size(); at += most) {
    const uint32_t n = (uint32_t)std::min<size_t>(most, some.size() - at);
    const int rc = f(some.data() + at, n);
    if (rc != POTS_E_OK) return rc;
  }
  return POTS_E_OK;
}

uint32_t blocks_of(uint64_t chunks) { return (uint32_t)std::min<uint64_t>(chunks, kBlocks); }

// The sums that the launches of each_launch leave, counted without a list, which could find no memory.
uint32_t parts_of(const pots_gradients* a) {
  uint32_t parts = 0, n = 0;
  uint64_t chunks = 0;
  for (uint32_t i = 0; i < a->tensors; i++) {
    if (!entries(a)[i].count) continue;
    chunks += chunks_of(entries(a)[i]);
    if (++n % kNormed == 0) {
      parts += blocks_of(chunks);
      chunks = 0;
    }
  }
  return parts + blocks_of(chunks);
}

template <class TABLE>
int sums_by(const pots_gradients* a, double* part, uint32_t* parts, hipStream_t s) {
  *parts = 0;
  uint64_t left = chunks_of(a);  // from the launch's first one to the list's last
  return each_launch(a, TABLE::kMost, [&](const uint32_t* some, uint32_t n) {
    TABLE t = {};
    for (uint32_t i = 0; i < n; i++) {
      const pots_gradient& e = entries(a)[some[i]];
      t.g[i] = e.gradient;
      t.count[i] = e.count;
      t.first[i] = t.chunks;
      t.type[i] = (uint8_t)e.gradient_type;
      t.chunks += (uint32_t)chunks_of(e);
    }
    t.tensors = n;
    t.kept = left > kKept ? (uint32_t)std::min<uint64_t>(left - kKept, t.chunks) : 0;
    left -= t.chunks;
    const uint32_t blocks = blocks_of(t.chunks);
    hipLaunchKernelGGL(norm_sums<TABLE>, dim3(blocks), dim3(256), 0, s, t, part + *parts);
    POTS_HIP(hipGetLastError());
    *parts += blocks;
    return POTS_E_OK;
  });
}

int sums(const pots_gradients* a, double* part, uint32_t* parts, hipStream_t s) {
  return a->tensors <= kFewTensors ? sums_by<Normed<kFewTensors>>(a, part, parts, s)
                                   : sums_by<Normed<kNormed>>(a, part, parts, s);
}

template <bool STEP, class TABLE>
int updates_by(const pots_gradients* a, const double* part, uint32_t parts, hipStream_t s) {
  std::vector<TABLE> launches;
  const bool past = chunks_of(a) > kKept;
  (void)each_launch(a, TABLE::kMost, [&](const uint32_t* some, uint32_t n) {
    launches.emplace_back();
    TABLE& t = launches.back();
    t.tensors = n;
    t.chunks = 0;
    t.past = past;
    for (uint32_t i = 0; i < n; i++) {
      const pots_gradient& e = entries(a)[some[i]];
      t.g[i] = e.gradient;
      t.w[i] = e.weight;
      t.out[i] = e.out;
      t.count[i] = e.count;
      t.first[i] = t.chunks;
      t.type[i] = (uint8_t)e.gradient_type;
      t.weight_type[i] = (uint8_t)e.weight_type;
      t.chunks += (uint32_t)chunks_of(e);
    }
    return POTS_E_OK;
  });
  if (launches.empty()) launches.emplace_back(TABLE{});  // the norm of nothing
  float* norm = a->norm;
  for (size_t i = launches.size(); i-- > 0;) {
    const uint32_t blocks = std::max(1u, blocks_of(launches[i].chunks));
    hipLaunchKernelGGL((update<STEP, TABLE>), dim3(blocks), dim3(256), 0, s, launches[i], part, parts,
                       a->max_norm, a->eta, norm);
    POTS_HIP(hipGetLastError());
    norm = nullptr;
  }
  return POTS_E_OK;
}

template <bool STEP>
int updates(const pots_gradients* a, const double* part, uint32_t parts, hipStream_t s) {
  return a->tensors <= kFewTensors ? updates_by<STEP, Updated<kFewTensors>>(a, part, parts, s)
                                   : updates_by<STEP, Updated<kUpdated>>(a, part, parts, s);
}

// Whether what is written lies apart from everything else: each out from the others, and from every
// input but its own entry's, which it may be exactly.
struct Range {
  uint64_t from, to;
  uint32_t entry, size;
};

bool overlaps(const pots_gradients* a, bool steps) {
  std::vector<Range> outs;
  const uint32_t sizes[] = {4, 2};
  for (uint32_t i = 0; i < a->tensors; i++) {
    const pots_gradient& e = entries(a)[i];
    const uint32_t size = sizes[steps ? e.weight_type : e.gradient_type];
    const uint64_t p = reinterpret_cast<uint64_t>(e.out);
    if (e.count) outs.push_back({p, p + e.count * size, i, size});
  }
  std::sort(outs.begin(), outs.end(), [](const Range& x, const Range& y) { return x.from < y.from; });
  for (size_t i = 1; i < outs.size(); i++)
    if (outs[i].from < outs[i - 1].to) return true;
  for (uint32_t i = 0; i < a->tensors; i++) {
    const pots_gradient& e = entries(a)[i];
    if (!e.count) continue;
    const void* const ins[] = {e.gradient, e.weight};
    const uint32_t types[] = {e.gradient_type, e.weight_type};
    for (uint32_t k = 0; k < (steps ? 2u : 1u); k++) {
      const uint64_t from = reinterpret_cast<uint64_t>(ins[k]);
      const uint64_t to = from + e.count * sizes[types[k]];
      auto o = std::upper_bound(outs.begin(), outs.end(), from,
                                [](uint64_t p, const Range& r) { return p < r.to; });
      for (; o != outs.end() && o->from < to; ++o)
        if (o->entry != i || o->from != from || o->size != sizes[types[k]]) return true;
    }
  }
  return false;
}

bool missing(const pots_gradients* a, bool writes, bool steps) {
  if (!a->norm) return true;
  for (uint32_t i = 0; i < a->tensors; i++) {
    const pots_gradient& e = entries(a)[i];
    if (e.count && (!e.gradient || (writes && !e.out) || (steps && !e.weight))) return true;
  }
  return false;
}

template <bool STEP>
int change(const pots_gradients* a, void* work, void* stream) {
  if (bad(a, true, STEP) || missing(a, true, STEP) || overlaps(a, STEP)) return POTS_E_ARG;
  if (parts_of(a) && !work) return POTS_E_ARG;
  hipStream_t s = static_cast<hipStream_t>(stream);
  double* const part = static_cast<double*>(work);
  uint32_t parts = 0;
  const int rc = sums(a, part, &parts, s);
  return rc != POTS_E_OK ? rc : updates<STEP>(a, part, parts, s);
}

}  // namespace

}  // namespace pots

using namespace pots;

// The lists that a call makes may find no memory; it says so in a text short enough to need none.
template <class F>
static int guarded(F&& f) noexcept {
  try {
    return f();
  } catch (...) {
    note_error("out of memory");
    return POTS_E_NOMEM;
  }
}

extern "C" uint64_t pots_gradient_norm_work(const pots_gradients* a) {
  return bad(a, false, false) ? 0 : 8ull * parts_of(a);
}

extern "C" int pots_gradient_norm(const pots_gradients* a, void* work, void* stream) {
  return guarded([&] {
    if (bad(a, false, false) || missing(a, false, false)) return POTS_E_ARG;
    if (parts_of(a) && !work) return POTS_E_ARG;
    hipStream_t s = static_cast<hipStream_t>(stream);
    double* const part = static_cast<double*>(work);
    uint32_t parts = 0;
    const int rc = sums(a, part, &parts, s);
    if (rc != POTS_E_OK) return rc;
    hipLaunchKernelGGL(norm_write, dim3(1), dim3(256), 0, s, part, parts, a->norm);
    POTS_HIP(hipGetLastError());
    return POTS_E_OK;
  });
}

extern "C" uint64_t pots_clip_gradients_work(const pots_gradients* a) {
  return pots_gradient_norm_work(a);
}

extern "C" int pots_clip_gradients(const pots_gradients* a, void* work, void* stream) {
  return guarded([&] { return change<false>(a, work, stream); });
}

extern "C" uint64_t pots_sgd_step_work(const pots_gradients* a) { return pots_gradient_norm_work(a); }

extern "C" int pots_sgd_step(const pots_gradients* a, void* work, void* stream) {
  return guarded([&] { return change<true>(a, work, stream); });
}
