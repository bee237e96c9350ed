// The calls of one decode step on caller-owned device buffers (declared, with their argument blocks,
// in include/kurumi_hip.h): argument checks and launchers. Checks throw std::runtime_error and touch
// no device; launchers take checked arguments.
#pragma once
#include <hip/hip_runtime_api.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "../../../../include/kurumi_hip.h"

namespace ku::hipbk {

void rope_freqs(size_t rot_dim, double base, uint32_t scaling, double factor, double trained_len, double low,
                double high, double* out);
void check_rope(const KuHipRopeArgs& a);
void launch_rope(const KuHipRopeArgs& a, hipStream_t s);

void check_sdpa_prefix(const KuHipSdpaPrefixArgs& a);
size_t sdpa_prefix_scratch_bytes(const KuHipSdpaPrefixArgs& a);
void launch_sdpa_prefix(const KuHipSdpaPrefixArgs& a, void* scratch, hipStream_t s);

void check_logits_adjust(const KuHipLogitsArgs& a);
void launch_logits_adjust(const KuHipLogitsArgs& a, hipStream_t s);

// ---- what the checks share ----

inline void require(bool ok, const char* what) {
  if (!ok) throw std::runtime_error(what);
}

inline size_t float_width(uint32_t dtype, const char* what) {
  if (dtype == KU_F32) return 4;
  if (dtype == KU_BF16 || dtype == KU_F16) return 2;
  throw std::runtime_error(std::string(what) + " must be KU_F32, KU_BF16 or KU_F16");
}

inline bool aligned_to(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// One strided axis of a buffer.
struct Axis {
  size_t n;
  int64_t stride;
};

// Elements from the first to one past the last that an array of contiguous runs of `inner` spans
// along strided axes; refuses negative strides and what no address space holds.
inline int64_t span_of(int64_t inner, std::initializer_list<Axis> axes, const char* what) {
  __int128 last = 0;
  for (const Axis& x : axes) {
    if (x.stride < 0) throw std::runtime_error(std::string(what) + " has a negative stride");
    if (x.n == 0) return 0;
    last += (__int128)(x.n - 1) * x.stride;
    if (last > ((__int128)1 << 58)) throw std::runtime_error(std::string(what) + " spans more than an address space");
  }
  return (int64_t)last + inner;
}

// The same for an array that is written: no two of its runs may share an element.
inline int64_t written_span(int64_t inner, std::initializer_list<Axis> axes, const char* what) {
  const int64_t whole = span_of(inner, axes, what);
  int64_t reach = inner;  // of the axes taken so far, by growing stride
  uint32_t taken = 0;
  for (size_t k = 0; k < axes.size(); ++k) {
    const Axis* next = nullptr;
    size_t at = 0, i = 0;
    for (const Axis& x : axes) {
      if (!(taken >> i & 1) && (!next || x.stride < next->stride)) {
        next = &x;
        at = i;
      }
      ++i;
    }
    taken |= 1u << at;
    if (next->n <= 1) continue;
    if (next->stride < reach) throw std::runtime_error(std::string(what) + " has rows that overlap");
    reach += (int64_t)(next->n - 1) * next->stride;
  }
  return whole;
}

inline bool overlap(const void* p, int64_t np, const void* q, int64_t nq) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p), b = reinterpret_cast<uintptr_t>(q);
  return a < b + (uintptr_t)nq && b < a + (uintptr_t)np;
}

// work-groups of `threads` in one launch, whose threads are counted in 32 bits
inline int64_t max_blocks(int threads) { return 0xffffffffll / threads; }

// Launches a kernel of one block of arguments. What the launch itself returns decides: an error that an earlier call of
// the thread left behind is neither taken for this launch's nor cleared.
template <class Args>
void launch(void (*kernel)(Args), dim3 grid, int threads, size_t lds, hipStream_t s, const Args& args) {
  void* p[] = {const_cast<Args*>(&args)};
  const hipError_t e = hipLaunchKernel(reinterpret_cast<const void*>(kernel), grid, dim3((unsigned)threads), p, lds, s);
  if (e != hipSuccess) throw std::runtime_error(std::string("launch failed: ") + hipGetErrorString(e));
}

}  // namespace ku::hipbk
