// Penalties, biases and a grammar's mask on logits (ku_hip_logits_adjust).
//
//   y = x;  seen: y = y > 0 ? y / rep : y * rep;  y -= freq n + (n > 0 ? pres : 0);
//   y += biases in list order;  y = -inf where the mask's bit is 0
// with n the times a token was generated in the row and seen whether it occurs in its tokens at all.
//
// A work-group takes a chunk of one row's vocabulary and counts, in LDS, the row's tokens that fall
// into it: whole numbers, so the order of the atomics does not matter. Bit 31 of a counter says that
// the token is in the prompt, the others count how often it was generated.
#include <hip/hip_runtime.h>

#include "decode.h"
#include "kernels.h"
#include "numeric.h"

namespace ku::hipbk {

namespace {

constexpr int kThreads = 256, kChunk = 4096;
constexpr uint32_t kInPrompt = 0x80000000u;

struct LogitsDev {
  const void* x;
  void* y;
  int64_t xs, ys, ts, ms, vocab;
  const int32_t *tokens, *lens, *prompt_lens;
  const float *repetition, *presence, *frequency;
  const int32_t* bias_ids;
  const float* bias_values;
  const int32_t* bias_offsets;
  const uint32_t* mask;
  const int32_t* mask_index;
  int32_t history, bias_count, mask_rows;
  uint32_t chunks;  // work-groups a row
};

__device__ __forceinline__ int32_t clamped(int32_t v, int32_t hi) { return v < 0 ? 0 : v > hi ? hi : v; }

template <int DT, class T, int OT, class O>
__global__ void __launch_bounds__(kThreads) logits_k(LogitsDev a) {
  __shared__ uint32_t count[kChunk];
  __shared__ float val[kChunk];
  const int64_t r = blockIdx.x / a.chunks, c0 = (int64_t)(blockIdx.x % a.chunks) * kChunk;
  const int n = (int)(a.vocab - c0 < kChunk ? a.vocab - c0 : kChunk), tid = threadIdx.x;
  for (int i = tid; i < n; i += kThreads) count[i] = 0;
  __syncthreads();
  if (a.tokens) {
    const int32_t len = a.lens ? clamped(a.lens[r], a.history) : a.history;
    const int32_t prompt = a.prompt_lens ? clamped(a.prompt_lens[r], len) : 0;
    const int32_t* tok = a.tokens + r * a.ts;
    for (int32_t i = tid; i < len; i += kThreads) {
      const int64_t at = (int64_t)tok[i] - c0;
      if (at < 0 || at >= n) continue;
      if (i < prompt)
        atomicOr(&count[at], kInPrompt);
      else
        atomicAdd(&count[at], 1u);
    }
  }
  __syncthreads();
  const float rep = a.repetition ? a.repetition[r] : 1.f, pres = a.presence ? a.presence[r] : 0.f,
              freq = a.frequency ? a.frequency[r] : 0.f;
  const T* x = static_cast<const T*>(a.x) + r * a.xs + c0;
  for (int i = tid; i < n; i += kThreads) {
    float v = load_elem<DT, T, float>(x[i]);
    const uint32_t c = count[i];
    if (c) {
      v = v > 0.f ? v / rep : v * rep;
      const uint32_t g = c & ~kInPrompt;
      if (g) v -= fmaf(freq, (float)g, pres);
    }
    val[i] = v;
  }
  if (a.bias_ids) {
    // an id's entries all go to the thread that holds its logit, in list order
    const int32_t e0 = clamped(a.bias_offsets[r], a.bias_count), e1 = clamped(a.bias_offsets[r + 1], a.bias_count);
    for (int32_t e = e0; e < e1; ++e) {
      const int64_t at = (int64_t)a.bias_ids[e] - c0;
      if (at >= 0 && at < n && at % kThreads == tid) val[at] += a.bias_values[e];
    }
  }
  const uint32_t* bits = nullptr;
  if (a.mask) {
    const int64_t m = a.mask_index ? a.mask_index[r] : r;
    if (m >= 0 && m < a.mask_rows) bits = a.mask + m * a.ms + c0 / 32;
  }
  O* y = static_cast<O*>(a.y) + r * a.ys + c0;
  for (int i = tid; i < n; i += kThreads) {
    float v = val[i];
    if (bits && !(bits[i >> 5] >> (i & 31) & 1)) v = -INFINITY;
    y[i] = store_elem<OT, O>(v);
  }
}

template <int DT, class T>
void launch_t(const LogitsDev& d, uint32_t out, int64_t rows, hipStream_t s) {
  const dim3 grid((unsigned)(d.chunks * rows));
  switch (out) {
    case KU_BF16: hipLaunchKernelGGL((logits_k<DT, T, GT_BF16, uint16_t>), grid, dim3(kThreads), 0, s, d); break;
    case KU_F16: hipLaunchKernelGGL((logits_k<DT, T, GT_F16, uint16_t>), grid, dim3(kThreads), 0, s, d); break;
    default: hipLaunchKernelGGL((logits_k<DT, T, GT_F32, float>), grid, dim3(kThreads), 0, s, d); break;
  }
}

}  // namespace

void check_logits_adjust(const KuHipLogitsArgs& a) {
  require(a.size == sizeof(KuHipLogitsArgs), "size is not sizeof(KuHipLogitsArgs)");
  const int64_t w = (int64_t)float_width(a.dtype, "dtype"), wo = (int64_t)float_width(a.out_dtype, "out_dtype");
  require(a.rows <= 0x7fffffff, "too many rows");
  require(a.vocab >= 1 && a.vocab <= 0x7fffffff, "vocab must be 1 to 2^31 - 1");
  require((__int128)((a.vocab + kChunk - 1) / kChunk) * a.rows <= 0x7fffffff, "too many rows of this vocab");
  require((a.logits && a.out) || a.rows == 0, "null logits or out");
  require(aligned_to(a.logits, (size_t)w) && aligned_to(a.out, (size_t)wo), "pointers must be aligned to their elements");
  const int64_t ni = span_of((int64_t)a.vocab, {{a.rows, a.logits_stride}}, "logits") * w;
  const int64_t no = written_span((int64_t)a.vocab, {{a.rows, a.out_stride}}, "out") * wo;
  if (a.rows && overlap(a.logits, ni, a.out, no))
    require(a.logits == a.out && a.dtype == a.out_dtype && (a.rows == 1 || a.logits_stride == a.out_stride),
            "out overlaps logits without being the same");
  require(a.history <= 0x7fffffff, "history is more than 2^31 - 1");
  if (a.tokens) span_of((int64_t)a.history, {{a.rows, a.tokens_stride}}, "tokens");
  require(a.tokens || !(a.lens || a.prompt_lens), "lens or prompt_lens without tokens");
  require((a.bias_ids != nullptr) == (a.bias_values != nullptr) && (a.bias_ids != nullptr) == (a.bias_offsets != nullptr),
          "bias_ids, bias_values and bias_offsets go together");
  require(a.bias_count <= 0x7fffffff, "bias_count is more than 2^31 - 1");
  require(a.mask || !a.mask_index, "mask_index without mask");
  if (a.mask) {
    require(a.mask_rows <= 0x7fffffff, "too many mask rows");
    require(a.mask_index || a.mask_rows >= a.rows, "fewer mask rows than rows, and no mask_index");
    span_of((int64_t)(a.vocab + 31) / 32, {{a.mask_rows, a.mask_stride}}, "mask");
  }
  for (const void* p : {(const void*)a.tokens, (const void*)a.lens, (const void*)a.prompt_lens, (const void*)a.repetition,
                        (const void*)a.presence, (const void*)a.frequency, (const void*)a.bias_ids,
                        (const void*)a.bias_values, (const void*)a.bias_offsets, (const void*)a.mask,
                        (const void*)a.mask_index})
    require(aligned_to(p, 4), "pointers must be aligned to their elements");
}

void launch_logits_adjust(const KuHipLogitsArgs& a, hipStream_t s) {
  if (a.rows == 0) return;
  LogitsDev d;
  d.x = a.logits;
  d.y = a.out;
  d.xs = a.logits_stride;
  d.ys = a.out_stride;
  d.ts = a.tokens_stride;
  d.ms = a.mask_stride;
  d.vocab = (int64_t)a.vocab;
  d.tokens = a.history ? a.tokens : nullptr;
  d.lens = a.lens;
  d.prompt_lens = a.prompt_lens;
  d.repetition = a.repetition;
  d.presence = a.presence;
  d.frequency = a.frequency;
  d.bias_ids = a.bias_count ? a.bias_ids : nullptr;
  d.bias_values = a.bias_values;
  d.bias_offsets = a.bias_offsets;
  d.mask = a.mask;
  d.mask_index = a.mask_index;
  d.history = (int32_t)a.history;
  d.bias_count = (int32_t)a.bias_count;
  d.mask_rows = (int32_t)a.mask_rows;
  d.chunks = (uint32_t)((d.vocab + kChunk - 1) / kChunk);
  switch (a.dtype) {
    case KU_BF16: launch_t<GT_BF16, uint16_t>(d, a.out_dtype, (int64_t)a.rows, s); break;
    case KU_F16: launch_t<GT_F16, uint16_t>(d, a.out_dtype, (int64_t)a.rows, s); break;
    default: launch_t<GT_F32, float>(d, a.out_dtype, (int64_t)a.rows, s); break;
  }
  check_launch();
}

}  // namespace ku::hipbk
