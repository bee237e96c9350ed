// Penalties, biases and a grammar's mask on logits (ku_hip_logits_adjust).
//
//   y = x;  seen: y = y > 0 ? y / rep : y * rep;  y -= freq n + (n > 0 ? pres : 0);
//   y += biases in list order;  y = -inf where the mask's bit is 0
// with n the times a token was generated in the row and seen whether it occurs in its tokens at all.
//
// A work-group takes a chunk of one row's vocabulary and counts, in LDS, the row's tokens that fall
// into it: whole numbers, so the order of the atomics does not matter. Nothing the size of the
// vocabulary is kept or cleared in memory; every logit is read once and written once, and the row's
// tokens and biases are read again by each of its chunks: neighbouring chunks run on different XCDs, so
// that each of these fetches a row's tokens into its own L2.
#include <hip/hip_runtime.h>

#include "decode.h"
#include "kernels.h"
#include "numeric.h"

namespace ku::hipbk {

namespace {

constexpr int kThreads = 512;
constexpr int kLarge = 16, kSmall = 4;  // logits a thread: chunks of 8192 or 2048
// A counter: how often the token was generated, and whether it is in the prompt and has biases.
constexpr uint32_t kInPrompt = 0x80000000u, kBiased = 0x40000000u, kCount = kBiased - 1;

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

// N elements at element alignment: rows of an odd vocabulary start anywhere.
template <class T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
  T e[N];
};

template <int DT, class T, int OT, class O, int PER>
__global__ void __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(8))) logits_k(LogitsDev a) {
  // what the wider side moves 16 bytes at a time: consecutive lanes then write consecutive pieces
  constexpr int WIDE = 16 / (int)(sizeof(T) > sizeof(O) ? sizeof(T) : sizeof(O)), V = WIDE < PER ? WIDE : PER, N = PER / V;
  constexpr int CHUNK = kThreads * PER, IDS = PER == kLarge ? 4 : 8;  // vectors of four token ids in flight
  __shared__ __attribute__((aligned(16))) uint32_t count[CHUNK];
  __shared__ int repeats;
  const int64_t r = blockIdx.x / a.chunks, c0 = (int64_t)(blockIdx.x % a.chunks) * CHUNK;
  const int n = (int)(a.vocab - c0 < CHUNK ? a.vocab - c0 : CHUNK), tid = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + r * a.xs + c0;
  O* y = static_cast<O*>(a.y) + r * a.ys + c0;

  // the logits are on their way while the tokens are counted
  Vec<T, V> in[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = (j * kThreads + tid) * V;
    if (i + V <= n) {
      in[j] = *reinterpret_cast<const Vec<T, V>*>(x + i);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i + e < n) in[j].e[e] = x[i + e];
    }
  }
  int32_t len = 0, prompt = 0;
  uint32_t e0 = 0, e1 = 0;  // below 2^31, so a place a round further is below 2^32
  if (a.tokens) {
    len = a.lens ? clamped(a.lens[r], a.history) : a.history;
    prompt = a.prompt_lens ? clamped(a.prompt_lens[r], len) : 0;
  }
  if (a.bias_ids) {
    e0 = clamped(a.bias_offsets[r], a.bias_count);
    e1 = clamped(a.bias_offsets[r + 1], a.bias_count);
  }
  const float rep = a.repetition ? a.repetition[r] : 1.f, pres = a.presence ? a.presence[r] : 0.f,
              freq = a.frequency ? a.frequency[r] : 0.f;
  const uint8_t* bits = nullptr;
  if (a.mask) {
    const int64_t m = a.mask_index ? a.mask_index[r] : r;
    if (m >= 0 && m < a.mask_rows) bits = reinterpret_cast<const uint8_t*>(a.mask + m * a.ms) + c0 / 8;
  }
  uint32_t allowed[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = (j * kThreads + tid) * V;
    allowed[j] = bits && i < n ? bits[i / 8] >> (i & 7) : 0xffu;
  }
  const bool counts = len > 0 || e1 > e0;
  // a thread's first bias, loaded beside the tokens
  int32_t bias_id = -1;
  float bias_value = 0.f;
  if (e0 + tid < e1) {
    bias_id = a.bias_ids[e0 + tid];
    bias_value = a.bias_values[e0 + tid];
  }
  // The place of token v in the chunk, or one past it. 32 bits are enough: c0 + n < 2^31, so a negative v
  // less c0 wraps to 2^31 - c0 or more, which is past n.
  auto place = [&](int32_t v) {
    const uint32_t at = (uint32_t)v - (uint32_t)c0;
    return at < (uint32_t)n ? (int)at : CHUNK;
  };
  if (counts) {
#pragma unroll
    for (int i = 0; i < PER / 4; ++i) reinterpret_cast<uint4*>(count)[i * kThreads + tid] = make_uint4(0, 0, 0, 0);
    if (tid == 0) repeats = 0;
    __syncthreads();
    const int32_t* tok = a.tokens + r * a.ts;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    for (int32_t i0 = 0; i0 < len; i0 += 4 * IDS * kThreads) {
      // IDS vectors of a wave, without those past the row's tokens: a group's instructions are as many
      // whether it holds a token or not
      const int32_t w0 = i0 + 256 * wave;
      Vec<int32_t, 4> id[IDS];
#pragma unroll
      for (int j = 0; j < IDS; ++j) {
        if (w0 + 4 * j * kThreads >= len) break;
        const int32_t i = i0 + 4 * (j * kThreads + tid);
        if (i + 4 <= len) {
          id[j] = *reinterpret_cast<const Vec<int32_t, 4>*>(tok + i);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) id[j].e[e] = i + e < len ? tok[i + e] : -1;
        }
      }
#pragma unroll
      for (int j = 0; j < IDS; ++j) {
        if (w0 + 4 * j * kThreads >= len) break;
        const int32_t i = i0 + 4 * (j * kThreads + tid);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = place(id[j].e[e]);
          if (at == CHUNK) continue;
          if (i + e < prompt)
            atomicOr(&count[at], kInPrompt);
          else
            atomicAdd(&count[at], 1u);
        }
      }
    }
    for (uint32_t e = e0 + tid; e < e1; e += kThreads) {
      const int at = place(e == e0 + tid ? bias_id : a.bias_ids[e]);
      if (at != CHUNK && (atomicOr(&count[at], kBiased) & kBiased)) repeats = 1;
    }
    __syncthreads();
  }
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int i = (j * kThreads + tid) * V;
    if (i >= n) break;
    Vec<O, V> out;
    float plain[V];
    uint32_t biased = 0;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      float v = load_elem<DT, T, float>(in[j].e[e]);
      if (counts) {
        // Without a branch: of a wave's 64 places one is touched more often than not. A division, not a product with
        // the reciprocal, which rounds once more and is infinite for penalties under 2^-128: 57 us for 55 on 256 rows
        // of 131072.
        const uint32_t c = count[i + e], g = c & kCount;
        const float take = fmaf(freq, (float)g, pres), by = v > 0.f ? v / rep : v * rep;
        v = c & ~kBiased ? by : v;
        v -= g ? take : 0.f;
        plain[e] = v;
        biased |= c;
      }
      if (!(allowed[j] >> e & 1)) v = -INFINITY;
      out.e[e] = store_elem<OT, O>(v);
    }
    if (biased & kBiased)  // for the bias, below
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (count[i + e] & kBiased) count[i + e] = __float_as_uint(plain[e]);
    if (i + V <= n) {
      *reinterpret_cast<Vec<O, V>*>(y + i) = out;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i + e < n) y[i + e] = out.e[e];
    }
  }
  if (e1 <= e0) return;
  // The few biased logits are written again, by the threads that read their biases. An id comes once as a
  // rule; where one comes again, each thread adds those of its places (at % kThreads) in list order first.
  __syncthreads();
  const bool again = repeats;
  if (again) {
    for (uint32_t e = e0; e < e1; ++e) {
      const int at = place(a.bias_ids[e]);
      if (at != CHUNK && at % kThreads == tid) count[at] = __float_as_uint(__uint_as_float(count[at]) + a.bias_values[e]);
    }
    __syncthreads();
  }
  for (uint32_t e = e0 + tid; e < e1; e += kThreads) {
    const int at = place(e == e0 + tid ? bias_id : a.bias_ids[e]);
    if (at == CHUNK || (bits && !(bits[at / 8] >> (at & 7) & 1))) continue;
    const float v = __uint_as_float(count[at]);
    y[at] = store_elem<OT, O>(again ? v : v + (e == e0 + tid ? bias_value : a.bias_values[e]));
  }
}

// Large chunks read a row's tokens fewer times, small ones spread few rows over the chip; they meet where
// there is a large one for every CU. us, large / small: 50257 logits, bf16 to f32, 1000 tokens: 16 rows
// 7.0 / 5.4, 32 rows (224 chunks) 7.4 / 7.0, 64 rows 9.8 / 10.6, 128 rows 14.4 / 17.1; 32000 logits, f16,
// 32768 tokens: 16 rows 10.7 / 9.2, 32 rows 12.0 / 12.2; 4 rows of 50257 f32 6.7 / 4.6; 256 rows of 131072,
// 4000 tokens: 56.5 / 88. Of large ones, 12 or 24 logits a thread or 256 threads: the same within 2 us.
bool large_chunks(int64_t vocab, int64_t rows) {
  return (vocab + kThreads * kLarge - 1) / (kThreads * kLarge) * rows >= (int64_t)cu_count();
}

template <int DT, class T, int OT, class O>
void launch_o(LogitsDev& d, int64_t rows, hipStream_t s) {
  const bool large = large_chunks(d.vocab, rows);
  const int64_t chunk = kThreads * (large ? kLarge : kSmall);
  d.chunks = (uint32_t)((d.vocab + chunk - 1) / chunk);
  const dim3 grid((unsigned)(d.chunks * rows));
  if (large)
    launch(logits_k<DT, T, OT, O, kLarge>, grid, kThreads, 0, s, d);
  else
    launch(logits_k<DT, T, OT, O, kSmall>, grid, kThreads, 0, s, d);
}
template <int DT, class T>
void launch_t(LogitsDev& d, uint32_t out, int64_t rows, hipStream_t s) {
  switch (out) {
    case KU_BF16: launch_o<DT, T, GT_BF16, uint16_t>(d, rows, s); break;
    case KU_F16: launch_o<DT, T, GT_F16, uint16_t>(d, rows, s); break;
    default: launch_o<DT, T, GT_F32, float>(d, rows, s); break;
  }
}

}  // namespace

void check_logits_adjust(const KuHipLogitsArgs& a) {
  require(a.size == sizeof(KuHipLogitsArgs), "size is not sizeof(KuHipLogitsArgs)");
  const int64_t w = (int64_t)float_width(a.dtype, "dtype"), wo = (int64_t)float_width(a.out_dtype, "out_dtype");
  require(a.rows <= 0x7fffffff, "too many rows");
  require(a.vocab >= 1 && a.vocab <= 0x7fffffff, "vocab must be 1 to 2^31 - 1");
  // so many rows take large chunks
  require((__int128)((a.vocab + kThreads * kLarge - 1) / (kThreads * kLarge)) * a.rows <= max_blocks(kThreads), "too many rows of this vocab");
  require((a.logits && a.out) || a.rows == 0, "null logits or out");
  require(aligned_to(a.logits, (size_t)w) && aligned_to(a.out, (size_t)wo), "pointers must be aligned to their elements");
  span_of((int64_t)a.vocab, {{a.rows, a.logits_stride}}, "logits");
  written_span((int64_t)a.vocab, {{a.rows, a.out_stride}}, "out");
  const Buffer out(a.out, (int64_t)a.vocab, {{a.rows, a.out_stride}}, wo);
  if (share(out, Buffer(a.logits, (int64_t)a.vocab, {{a.rows, a.logits_stride}}, w)))
    require(a.logits == a.out && a.dtype == a.out_dtype && (a.rows == 1 || a.logits_stride == a.out_stride),
            "out overlaps logits without being the same");
  require(a.history <= kCount, "history is more than 2^30 - 1");
  if (a.tokens) span_of((int64_t)a.history, {{a.rows, a.tokens_stride}}, "tokens");
  // an array of no elements may be null beside others that are there
  require(a.tokens || a.history == 0 || !(a.lens || a.prompt_lens), "lens or prompt_lens without tokens");
  require(a.bias_count == 0 || ((a.bias_ids != nullptr) == (a.bias_values != nullptr) && (a.bias_ids != nullptr) == (a.bias_offsets != nullptr)),
          "bias_ids, bias_values and bias_offsets go together");
  require(a.bias_count <= 0x7fffffff, "bias_count is more than 2^31 - 1");
  require(a.mask || a.mask_rows == 0 || !a.mask_index, "mask_index without mask");
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
  const auto flat = [](const void* p, size_t n) { return Buffer(p, (int64_t)n, {}, 4); };
  for (const Buffer& x :
       {Buffer(a.tokens, (int64_t)a.history, {{a.rows, a.tokens_stride}}, 4), flat(a.lens, a.rows), flat(a.prompt_lens, a.rows),
        flat(a.repetition, a.rows), flat(a.presence, a.rows), flat(a.frequency, a.rows), flat(a.bias_ids, a.bias_count),
        flat(a.bias_values, a.bias_count), flat(a.bias_count ? a.bias_offsets : nullptr, a.rows + 1),
        Buffer(a.mask, (int64_t)(a.vocab + 31) / 32, {{a.mask_rows, a.mask_stride}}, 4), flat(a.mask ? a.mask_index : nullptr, a.rows)})
    require(!share(out, x), "out overlaps an array that is read");
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
  switch (a.dtype) {
    case KU_BF16: launch_t<GT_BF16, uint16_t>(d, a.out_dtype, (int64_t)a.rows, s); break;
    case KU_F16: launch_t<GT_F16, uint16_t>(d, a.out_dtype, (int64_t)a.rows, s); break;
    default: launch_t<GT_F32, float>(d, a.out_dtype, (int64_t)a.rows, s); break;
  }
}

}  // namespace ku::hipbk
