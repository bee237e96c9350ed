// The calls of one decode step on caller-owned device buffers (declared, with their argument blocks,
// in include/kurumi_hip.h): argument checks and launchers. Checks throw std::runtime_error and touch
// no device; launchers take checked arguments.
#pragma once
#include <hip/hip_runtime_api.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
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

// A buffer as a call reads or writes it: contiguous runs of `inner` elements of `width` bytes along strided axes, which
// span less than 2^61 bytes (span_of).
struct Buffer {
  const void* p = nullptr;
  int64_t inner = 0;  // bytes
  int64_t span = 0;   // bytes from the first to one past the last; 0: nothing
  struct {
    int64_t last, stride;  // steps, bytes
  } axes[3];
  int used = 0;

  Buffer() = default;
  Buffer(const void* at, int64_t run, std::initializer_list<Axis> along, size_t width) : p(at), inner(run * (int64_t)width), span(inner) {
    for (const Axis& x : along) {
      if (x.n == 0) p = nullptr;
      if (x.n <= 1 || x.stride == 0) continue;
      axes[used++] = {(int64_t)x.n - 1, x.stride * (int64_t)width};
      span += axes[used - 1].last * axes[used - 1].stride;
    }
    if (!p) span = 0;
  }
};

// Whether two buffers have a byte in common. Their runs' places differ by a sum of strides times steps of the axes, in
// ranges: the steps are tried from the longest stride down, those that the shorter ones cannot make up for left
// out, which leaves few of them where an axis' steps go past the axes inside it. Layouts that leave too many to
// try count as sharing.
inline bool share(const Buffer& a, const Buffer& b) {
  const int64_t apart = (int64_t)(reinterpret_cast<uintptr_t>(b.p) - reinterpret_cast<uintptr_t>(a.p));
  if (a.span == 0 || b.span == 0 || apart >= a.span || -apart >= b.span) return false;
  struct Term {
    int64_t stride, lo, hi;  // bytes; steps
  } t[6];
  int n = 0;
  for (const Buffer* x : {&a, &b})
    for (int i = 0; i < x->used; ++i) {
      int k = 0;
      while (k < n && t[k].stride > x->axes[i].stride) ++k;
      if (k == n || t[k].stride != x->axes[i].stride) {
        for (int j = n++; j > k; --j) t[j] = t[j - 1];
        t[k] = {x->axes[i].stride, 0, 0};
      }
      if (x == &a) t[k].lo -= x->axes[i].last;
      else t[k].hi += x->axes[i].last;
    }
  int64_t lo[7] = {}, hi[7] = {};  // what the terms from k on can add
  for (int k = n; k-- > 0;) {
    lo[k] = lo[k + 1] + t[k].stride * t[k].lo;
    hi[k] = hi[k + 1] + t[k].stride * t[k].hi;
  }
  const auto floor_div = [](int64_t x, int64_t y) { return x / y - (x % y < 0); };
  int tries = 20000;
  auto meet = [&](auto& self, int k, int64_t at) -> bool {
    if (k == n) return at > -b.inner && at < a.inner;
    // steps from whose place the terms after this one can still bring the runs together
    const int64_t first = std::max(t[k].lo, floor_div(-b.inner - at - hi[k + 1], t[k].stride) + 1),
                  last = std::min(t[k].hi, -floor_div(-(a.inner - at - lo[k + 1]), t[k].stride) - 1);
    for (int64_t i = first; i <= last; ++i)
      if (--tries < 0 || self(self, k + 1, at + i * t[k].stride)) return true;
    return false;
  };
  return meet(meet, 0, apart);
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
