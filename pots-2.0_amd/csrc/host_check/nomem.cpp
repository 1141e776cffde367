// The calls over lists of tensors where memory runs out, on the sanitized CPU build of
// libpots_mi355x's host code (host_model.cpp stands in for the HIP runtime). The first allocation of a call
// fails, then the second, and so on until the call succeeds. For each attempt a line: the call's name, its return
// code, the scratch that its *_work call asks for at the same time, and the error's text.
#include <stdint.h>
#include <stdio.h>
#include <stdlib.h>
#include <string.h>

#include <new>
#include <vector>

#include "../../../include/pots_mi355x.h"

extern "C" void host_model_set(int pinned, int launches);

static long g_left = -1;  // how many allocations succeed yet (-1: all)

static void* allocate(size_t bytes) {
  if (g_left == 0) return nullptr;
  if (g_left > 0) g_left--;
  return malloc(bytes ? bytes : 1);
}
void* operator new(size_t bytes) {
  void* const p = allocate(bytes);
  if (!p) throw std::bad_alloc();
  return p;
}
void* operator new(size_t bytes, const std::nothrow_t&) noexcept { return allocate(bytes); }
void operator delete(void* p) noexcept { free(p); }
void operator delete(void* p, size_t) noexcept { free(p); }
void operator delete(void* p, const std::nothrow_t&) noexcept { free(p); }

int main() {
  constexpr uint32_t kTensors = 200;
  char* const p = reinterpret_cast<char*>(1ull << 44);  // (nothing reads it)
  std::vector<char> block(sizeof(pots_gradients) + kTensors * sizeof(pots_gradient));
  pots_gradients a = {};
  a.norm = reinterpret_cast<float*>(p), a.max_norm = 1.f, a.eta = 0.1f, a.tensors = kTensors;
  memcpy(block.data(), &a, sizeof a);
  for (uint32_t i = 0; i < kTensors; i++) {
    pots_gradient e = {};
    e.count = 1000;
    e.gradient = p + (1 << 20) + 4000 * i, e.weight = p + (2 << 20) + 4000 * i;
    e.out = p + (3 << 20) + 4000 * i;
    memcpy(block.data() + sizeof a + i * sizeof e, &e, sizeof e);
  }
  const pots_gradients* const g = reinterpret_cast<const pots_gradients*>(block.data());
  const struct {
    const char* name;
    int (*run)(const pots_gradients*, void*, void*);
    uint64_t (*work)(const pots_gradients*);
  } calls[] = {{"gradient_norm", pots_gradient_norm, pots_gradient_norm_work},
               {"clip_gradients", pots_clip_gradients, pots_clip_gradients_work},
               {"sgd_step", pots_sgd_step, pots_sgd_step_work}};
  for (const auto& c : calls) {
    int rc = -1;
    for (int n = 0; rc != 0 && n < 100; n++) {
      host_model_set(1, 0);
      (void)c.run(g, p, nullptr);  // leaves an error of its own
      host_model_set(1, 1);
      g_left = n;
      const uint64_t work = c.work(g);
      g_left = n;
      rc = c.run(g, p, nullptr);
      g_left = -1;
      printf("%s %d %llu %s\n", c.name, rc, (unsigned long long)work, rc ? pots_last_error() : "");
    }
  }
  return 0;
}
