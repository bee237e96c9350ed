// What the kernels of the shared-prefix attention have in common: their arguments, where a key lies,
// and one query by itself.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.h"
#include "numeric.h"

namespace ku::hipbk {

constexpr int kSdpaMaxDim = 128;

struct SdpaDev {
  const void *q, *pk, *pv, *k, *v;
  void* o;
  float* lse;
  int64_t qb, qt, qh, ob, ot, oh;  // element strides
  int64_t prow, phead, row, head;
  const int32_t *lens, *pages;
  int64_t seq_rows, per_seq;
  int32_t batch, q_len, q_heads, kv_heads, dim, group;
  int32_t prefix, own_max, page_shift, npages;  // page_shift < 0: contiguous
  float scale;
};

// own keys of sequence b
__device__ __forceinline__ int sdpa_len(const SdpaDev& a, int b) {
  if (a.own_max == 0) return 0;
  const int n = a.lens[b];
  return n < 0 ? 0 : n > a.own_max ? a.own_max : n;
}
// row of own key j of sequence b, or -1 where its page is none of the cache's
__device__ __forceinline__ int64_t sdpa_row(const SdpaDev& a, int b, int j) {
  if (a.page_shift < 0) return b * a.seq_rows + j;
  const int32_t page = a.pages[b * a.per_seq + (j >> a.page_shift)];
  if (page < 0 || page >= a.npages) return -1;
  return ((int64_t)page << a.page_shift) + (j & ((1 << a.page_shift) - 1));
}

template <int DT>
struct SdpaElem {
  using T = uint16_t;
  static constexpr int V = 8;  // elements in 16 bytes
};
template <>
struct SdpaElem<GT_F32> {
  using T = float;
  static constexpr int V = 4;
};

// One query by one wave, from the definition: the maximum over the keys it sees, the sum of their
// probabilities, then the values by probabilities that add up to one, so that nothing overflows that the
// result does not. Only keys that it sees are read, and infinities and NaN come out as the definition has
// them: the tiled kernels leave queries to it whose sums are not finite. `lds`: kSdpaMaxDim floats of the wave.
template <int DT>
__device__ void sdpa_one(const SdpaDev& a, int b, int t, int h, float* lds) {
  using T = typename SdpaElem<DT>::T;
  constexpr int V = SdpaElem<DT>::V;
  const int lane = threadIdx.x & 63, kvh = h / a.group;
  const T* q = static_cast<const T*>(a.q) + b * a.qb + t * a.qt + h * a.qh;
  for (int d = lane; d < a.dim; d += 64) lds[d] = load_elem<DT, T, float>(q[d]);
  __builtin_amdgcn_wave_barrier();
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  int seen = sdpa_len(a, b) - (a.q_len - 1 - t);
  if (seen < 0) seen = 0;
  const int64_t n = (int64_t)a.prefix + seen;
  const T *pk = static_cast<const T*>(a.pk) + kvh * a.phead, *pv = static_cast<const T*>(a.pv) + kvh * a.phead;
  const T *ok = static_cast<const T*>(a.k) + kvh * a.head, *ov = static_cast<const T*>(a.v) + kvh * a.head;
  // offset of key j, or -1 where it is not there
  auto offset = [&](int64_t j) -> int64_t {
    if (j < a.prefix) return j * a.prow;
    const int64_t r = sdpa_row(a, b, (int)(j - a.prefix));
    return r < 0 ? -1 : r * a.row;
  };
  auto score = [&](int64_t j, int64_t off) {
    const T* key = (j < a.prefix ? pk : ok) + off;
    float s = 0.f;
    for (int d = 0; d < a.dim; d += V) {
      const uint4 w = *reinterpret_cast<const uint4*>(key + d);
      T e[V];
      __builtin_memcpy(e, &w, 16);
#pragma unroll
      for (int i = 0; i < V; ++i) s = fmaf(lds[d + i], load_elem<DT, T, float>(e[i]), s);
    }
    return s * a.scale;
  };
  float m = -INFINITY;
  bool nan = false, any = false;
  for (int64_t j = lane; j < n; j += 64) {
    const int64_t off = offset(j);
    if (off < 0) continue;
    const float s = score(j, off);
    any = true;
    nan |= s != s;
    m = fmaxf(m, s);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  any = __builtin_amdgcn_ballot_w64(any) != 0;
  nan = __builtin_amdgcn_ballot_w64(nan) != 0;
  float l = 0.f, acc[kSdpaMaxDim / 64] = {};
  for (int64_t j = lane; j < n; j += 64) {
    const int64_t off = offset(j);
    if (off >= 0) l += expf(score(j, off) - m);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) l += __shfl_xor(l, o, 64);
  const float inv = 1.f / l;
  for (int64_t j0 = 0; j0 < n; j0 += 64) {
    const int64_t j = j0 + lane, off = j < n ? offset(j) : -1;
    const float p = off < 0 ? 0.f : expf(score(j, off) - m) * inv;
    const int left = n - j0 < 64 ? (int)(n - j0) : 64;
    for (int i = 0; i < left; ++i) {
      const int64_t oi = ((int64_t)__builtin_amdgcn_readlane((int)(off >> 32), i) << 32) |
                         (uint32_t)__builtin_amdgcn_readlane((int)off, i);
      if (oi < 0) continue;
      const float pi = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(p), i));
      const T* val = (j0 + i < a.prefix ? pv : ov) + oi;
#pragma unroll
      for (int c = 0; c < kSdpaMaxDim / 64; ++c)
        if (lane + 64 * c < a.dim) acc[c] = fmaf(pi, load_elem<DT, T, float>(val[lane + 64 * c]), acc[c]);
    }
  }
  T* out = static_cast<T*>(a.o) + b * a.ob + t * a.ot + h * a.oh;
#pragma unroll
  for (int c = 0; c < kSdpaMaxDim / 64; ++c)
    if (lane + 64 * c < a.dim) out[lane + 64 * c] = store_elem<DT, T, float>(any ? acc[c] : 0.f);
  if (a.lse && lane == 0)
    a.lse[((int64_t)b * a.q_len + t) * a.q_heads + h] = nan ? NAN : isinf(m) ? m : m + logf(l);
}

}  // namespace ku::hipbk
