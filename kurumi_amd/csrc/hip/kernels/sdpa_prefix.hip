// Attention of a batch that shares its first keys (ku_hip_sdpa_prefix).
//
//   out[b, t, h] = sum_j softmax_j(scale q[b, t, h] . K_j) V_j
// over the shared prefix and the keys of sequence b that query t sees.
//
// The queries that read one kv head are the rows of a matrix product with its keys. Over the prefix
// the rows of every sequence go through together ("pooled"): a key is read once for each tile of them,
// which is what makes it a matrix product and not a vector one. A sequence's own keys meet its own rows
// only. Where one sequence fills whole tiles of rows by itself (many queries), its tiles walk the prefix
// and then its own keys in one pass ("joint").
//
// Tiles are computed transposed, so that one lane owns one query:
//   S^T[key][q] = K[key][:] . Q[q][:],   O^T[d][q] += V^T[d][key] . P^T[key][q]
// with 32 x 32 MFMA tiles. Lane l of an accumulator holds query l % 32 and rows 8 (v / 4) + 4 (l / 32)
// + v % 4, so maximum, sum and rescale are a lane's own scalars, and the probabilities lie in registers
// as the second product's operand. K and V go to LDS by DMA.
//
// The keys of a tile are cut into splits until the chip is full; each split leaves its maximum, sums and
// unnormalised output in f32 in the scratch and a second kernel joins them in split order. A tile with
// one split writes its output itself.
//
// Only rows that some query sees are ever loaded (places past the end repeat the last one), so what lies
// behind them cannot matter. A query whose sums are not finite, or that saw nothing, is done again from
// the definition by sdpa_one: an infinity or NaN in a value that another query of the tile sees comes out right that way
// (64 queries of 32 heads on 8192 keys with one such value: 6 ms). Keys whose page is none are masked in their tiles.
//
// What bounds it, 32 heads over 8 of 128 features, with lse, us of both kernels:
//   1 query each of 32 sequences, 65536 shared keys, f16 (303 MB): 81, 3.7 TB/s; the loop alone runs at the
//     rate of a copy (5 TB/s), the rest is a unit's start, its partial result and the join
//   64 sequences of up to 1024 own keys in pages of 16 beside 8192 shared ones, bf16 (171 MB): 50, 3.4 TB/s;
//     the own keys, which few work-groups read with little in flight at the end
//   256 queries each of 8 sequences, 16 heads over 4 of 64, 4096 shared keys, bf16 (37 GFLOP): 65, 0.6 PFLOP/s;
//     the vector units: over 64 features a score's exponential and sums take as long as its two products
// The second sum, for lse, takes 2 to 3 us of each.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "decode.h"
#include "lds_dma.h"
#include "pair16.h"
#include "sdpa_prefix.h"

namespace ku::hipbk {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((__vector_size__(4 * sizeof(short))));
#define KU_LDS __attribute__((address_space(3)))

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// The running maximum moves only when a block exceeds it by more than this (in powers of two), so most
// blocks leave O alone; probabilities reach 2^8 at most before they are normalised.
constexpr float RESCALE = 8.f;
// Probabilities of f16 keys are formed 2^7 times as large (at most 2^15, with RESCALE): those below 2^-21 of the
// largest, not 2^-14, are rounded to a step of one size, 2^-32 of the largest being half of it. Without it 65536 keys
// far below one would leave up to 2^-9 of their values' size. All sums carry the factor; lse takes it out.
template <int DT>
constexpr float SHIFT = DT == GT_F16 ? 7.f : 0.f;
template <int DT>
__device__ __forceinline__ float lse_of(float m, float sum) {
  return (m + __builtin_amdgcn_logf(sum * (DT == GT_F16 ? 0.0078125f : 1.f))) * LN2;
}

// Division by a number known at the launch: a product, and one correction.
struct Div {
  uint32_t d = 1, m = 0xffffffffu;
  Div() = default;
  explicit Div(int64_t by) : d((uint32_t)std::max<int64_t>(by, 1)), m((uint32_t)std::min<uint64_t>(((uint64_t)1 << 32) / d, 0xffffffffu)) {}
  __device__ __forceinline__ int split(int n, int& rest) const {
    uint32_t q = __umulhi((uint32_t)n, m), r = (uint32_t)n - q * d;
    if (r >= d) {
      ++q;
      r -= d;
    }
    rest = (int)r;
    return (int)q;
  }
};

// How a call is cut into work-groups.
struct SdpaPlan {
  bool joint = false;
  // [0] the prefix with the rows of all sequences (joint: prefix and own keys of a sequence's rows);
  // [1] a sequence's own keys with its rows
  struct Part {
    bool shared = false;  // four waves of 32 rows over the same blocks of keys; else 32 rows, the blocks dealt to the waves
    int tiles = 0, splits = 0;   // row tiles a kv head (and sequence), splits of their keys
    int units = 0;               // work-groups: tiles times splits of all of them
    Div by_tiles, by_splits;
  } part[2];
  int slots = 0;        // partial results a row
  bool sorted = false;  // the own keys' units by their sequences' lengths
  Div by_kv, by_group, by_seq, by_q_len, by_heads;  // kv heads; q heads of one; a sequence's rows; its queries; q heads
};

struct SdpaArgs {
  SdpaDev a;
  SdpaPlan p;
  float* po;   // [rows][slots][D]
  float4* ml;  // [rows][slots]: maximum in powers of two, sum, sum of the probabilities before rounding
};

template <int DT>
__device__ __forceinline__ void mfma_step(const u32x4& a, const u32x4& b, f32x16& c) {
  static_assert(DT != GT_F32, "16-bit elements");
  if constexpr (DT == GT_BF16)
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// the value of the other half of the wave
__device__ __forceinline__ float other_half(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? sw[0] : sw[1]);
}

// Rows of keys lie in LDS as D features, of which the products take the first DR (heads of 65 to 96
// features as 96 of 128: a quarter of the products less).
template <int DT, int D, int DR>
struct Tile {
  static constexpr int ES = DT == GT_F32 ? 4 : 2;
  static constexpr int RB = D * ES;          // bytes of a row in LDS
  static constexpr int CPR = RB / 16;        // 16-byte chunks of a row
  static constexpr int KT = 32 * RB;         // bytes of 32 keys
  static constexpr int DS = DR * ES / 32;    // chunk pairs: steps of S^T
  static constexpr int DTL = DR / 32;        // 32-row tiles of O^T
  static constexpr int SB = DT == GT_F32 ? 1 : 2;  // 32-key tiles of a shared block
  // shared: K and V, two buffers each; solo: K and V of every wave
  static constexpr int LDS = std::max(4 * SB * KT, 4 * 2 * KT);
  // rows r at one chunk: 16 of them on 16 bank groups of the 256-byte window
  static __device__ __forceinline__ int kswz(int r) {
    if constexpr (RB >= 256) return r & 15;
    else return (r / (256 / RB)) % (16 / (256 / RB));
  }
  static __device__ __forceinline__ int vswz(int r) {
    if constexpr (DT == GT_F32) return RB >= 256 ? ((r >> 2) & 1) * 8 : 0;
    else if constexpr (RB >= 256) return 4 * (r & 3);
    else return 4 * ((r / (256 / RB)) % (4 / (256 / RB)));
  }
};

// One wave's 32 rows of a tile: Q fragments, running maximum, sum and O.
//
// Probabilities of 16-bit keys are rounded to 16 bits for the second product, and the output is divided by the sum
// of the rounded ones: where many round the same way, a mean with unrounded ones below would be off by that rounding.
// lse is of the unrounded sum, which is formed where it is asked for (LSE). Heads of up to 32 features hold a
// probability as two 16-bit values with a product each, its rounding and the rounding of what that left, to 2^-17 of
// itself in bf16 and 2^-22 in f16, and one unrounded sum: there the second product is a small part of a block.
// Larger heads hold one value, off by half a step (the output's own rounding is another): with two, 64 sequences on
// 8192 keys of 128 features would take 60 us for 50, 32 on 65536 100 for 80, 8 x 256 queries on 4096 of 64 78 for 67
// (kernel times, with lse).
template <int DT, int D, int DR, bool LSE>
struct Rows {
  using T = Tile<DT, D, DR>;
  static constexpr bool TWO = DT != GT_F32 && D == 32;        // two values a probability
  static constexpr bool WHOLE = LSE && DT != GT_F32 && !TWO;  // two sums
  u32x4 q[T::DS];
  f32x16 o[T::DTL];
  float m, l;  // m in powers of two, already times scale
  float w;     // WHOLE: the sum before rounding
  int limit;   // own keys that this lane's query sees

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = w = 0.f;
#pragma unroll
    for (int t = 0; t < T::DTL; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) o[t][v] = 0.f;
  }
  // `row`: this lane's query, or null past the last
  __device__ __forceinline__ void load_q(const void* row, int dim) {
    const int h = (threadIdx.x & 63) >> 5, chunks = dim * T::ES / 16;
#pragma unroll
    for (int s = 0; s < T::DS; ++s) {
      const int c = 2 * s + h;
      q[s] = u32x4{0, 0, 0, 0};
      if (row && c < chunks) q[s] = *reinterpret_cast<const u32x4*>(static_cast<const char*>(row) + c * 16);
    }
  }
  // Scores of 32 keys. In f32 the products go into four sums: the error of a chain of d of them grows with
  // its length, and a fourth of it halves the scores' error, which is most of the output's where keys are few.
  __device__ __forceinline__ f32x16 scores(const KU_LDS unsigned char* K) const {
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    constexpr int SUMS = DT == GT_F32 ? 4 : 1;
    f32x16 s[SUMS] = {};
    u32x4 k[3];  // fragments two steps ahead
    auto read = [&](int i) { return *(const KU_LDS u32x4*)(K + r * T::RB + (((2 * i + h) ^ T::kswz(r)) << 4)); };
    k[0] = read(0);
    if (T::DS > 1) k[1] = read(1);
#pragma unroll
    for (int i = 0; i < T::DS; ++i) {
      if (i + 2 < T::DS) k[(i + 2) % 3] = read(i + 2);
      if constexpr (DT == GT_F32) {
        const f32x4 x = __builtin_bit_cast(f32x4, k[i % 3]), y = __builtin_bit_cast(f32x4, q[i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) s[j] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], s[j], 0, 0, 0);
      } else {
        mfma_step<DT>(k[i % 3], q[i], s[0]);
      }
    }
    if constexpr (DT == GT_F32)
#pragma unroll
      for (int v = 0; v < 16; ++v) s[0][v] = (s[0][v] + s[1][v]) + (s[2][v] + s[3][v]);
    return s[0];
  }
  // Sums of a block's probabilities of 16 bits, in two chains.
  struct Sums {
    float l[2] = {0.f, 0.f}, w[2] = {0.f, 0.f};
    // two probabilities as the product takes them, `lo` what their rounding left
    __device__ __forceinline__ uint32_t add(int i, float p0, float p1, uint32_t& lo) {
      const uint32_t pp = pack2<DT>(p0, p1);
      if constexpr (TWO) {
        lo = pack2<DT>(p0 - lower<DT>(pp), p1 - upper<DT>(pp));
        l[i] += p0 + p1;
      } else {
        l[i] = sum2<DT>(pp, l[i]);
        if constexpr (WHOLE) w[i] += p0 + p1;
      }
      return pp;
    }
  };
  __device__ __forceinline__ void join(const Sums& r) {
    l += r.l[0] + r.l[1];
    if constexpr (WHOLE) w += r.w[0] + r.w[1];
  }
  // what a score in powers of two is brought to the exponent of a probability by; of nothing seen so far every score is -inf
  __device__ __forceinline__ float exponent() const { return m == -INFINITY ? 0.f : SHIFT<DT> - m; }
  // keys from `left` on are not seen (left counts from the tile's first key)
  static __device__ __forceinline__ void mask(f32x16& s, int left) {
    const int lim = left - 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int v = 0; v < 16; ++v)
      if ((v >> 2) * 8 + (v & 3) >= lim) s[v] = -INFINITY;
  }
  // keys whose bit is not set are not there
  static __device__ __forceinline__ void mask_absent(f32x16& s, uint32_t present) {
    const uint32_t mine = present >> (4 * ((threadIdx.x & 63) >> 5));
#pragma unroll
    for (int v = 0; v < 16; ++v)
      if (!(mine >> ((v >> 2) * 8 + (v & 3)) & 1)) s[v] = -INFINITY;
  }
  // the new maximum over NT tiles of scores, O and l brought to it
  template <int NT>
  __device__ __forceinline__ void rescale(const f32x16 (&s)[NT], float c) {
    float bm = s[0][0];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int v = 0; v < 16; ++v) bm = fmaxf(bm, s[t][v]);
    bm = fmaxf(bm, other_half(bm)) * c;
    const bool need = bm > m + RESCALE || (bm > m && m == -INFINITY);
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
      const float mn = need ? bm : m, corr = need ? __builtin_amdgcn_exp2f(m - mn) : 1.f;
      m = mn;
      l *= corr;
      if constexpr (WHOLE) w *= corr;
#pragma unroll
      for (int t = 0; t < T::DTL; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] *= corr;
    }
  }
  // O^T += V^T P^T over 32 keys of 16-bit values, the fragments of V read a step of 16 keys ahead.
  // V^T fragments by transposing reads: in each 16-lane group input lane 4 k' + j points at key row k',
  // dims 4 j.. + 3, and output lane i receives keys 0..3 of dim i; two of them fetch the keys that the
  // probability registers hold, 16 s + 4 h + 0..3 and those + 8.
  // `lo`: the second values of the probabilities, where there are two.
  template <int STEPS>
  __device__ __forceinline__ void product(const u32x4 (&p)[STEPS], const u32x4 (&lo)[STEPS], const KU_LDS unsigned char* V) {
    const int lane = threadIdx.x & 63, h = lane >> 5, g = lane >> 4, c16 = lane & 15;
    auto read = [&](int st, u32x4 (&f)[T::DTL]) {
#pragma unroll
      for (int t = 0; t < T::DTL; ++t) {
        const int d = t * 32 + (g & 1) * 16 + (c16 & 3) * 4;
        u32x2 half[2];
#pragma unroll
        for (int r2 = 0; r2 < 2; ++r2) {
          const int kr = 16 * st + 8 * r2 + 4 * h + (c16 >> 2);
          const KU_LDS unsigned char* a = V + kr * T::RB + (((d >> 3) ^ T::vswz(kr)) << 4) + (d & 7) * 2;
          half[r2] = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((KU_LDS s16x4*)a));
        }
        f[t] = u32x4{half[0][0], half[0][1], half[1][0], half[1][1]};
      }
    };
    u32x4 f[2][T::DTL];
    read(0, f[0]);
#pragma unroll
    for (int st = 0; st < STEPS; ++st) {
      if (st + 1 < STEPS) read(st + 1, f[(st + 1) & 1]);
#pragma unroll
      for (int t = 0; t < T::DTL; ++t) {
        mfma_step<DT>(f[st & 1][t], p[st], o[t]);
        if constexpr (TWO) mfma_step<DT>(f[st & 1][t], lo[st], o[t]);
      }
    }
  }
  // O^T += V^T P^T over 32 keys, with the probabilities' sums.
  __device__ __forceinline__ void weigh(const f32x16& s, float c, const KU_LDS unsigned char* V) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const float em = exponent();
    if constexpr (DT == GT_F32) {
      // 32 keys in a sum of their own, which then joins O: a chain of every key's products would have an
      // error that grows with the keys
      const int r = lane & 31;
      float p[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        p[v] = __builtin_amdgcn_exp2f(fmaf(s[v], c, em));
        l += p[v];
      }
#pragma unroll
      for (int t = 0; t < T::DTL; ++t) {
        f32x16 sum = {};
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int key = (v >> 2) * 8 + (v & 3) + 4 * h, d = 32 * t + r;
          const float x = *(const KU_LDS float*)(V + key * T::RB + (((d >> 2) ^ T::vswz(key)) << 4) + (d & 3) * 4);
          sum = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p[v], sum, 0, 0, 0);
        }
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] += sum[v];
      }
    } else {
      u32x4 p[2], lo[2];
      Sums r;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * i], c, em));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], c, em));
        uint32_t rest = 0;
        p[i >> 2][i & 3] = r.add(i & 1, p0, p1, rest);
        lo[i >> 2][i & 3] = rest;
      }
      join(r);
      product(p, lo, V);
    }
  }
};

// A run of keys of one kv head, prefix or own, and the DMA of tiles of it.
template <int DT, int D, int DR>
struct Keys {
  using T = Tile<DT, D, DR>;
  static constexpr int RPD = 1024 / T::RB;  // rows of one DMA instruction
  const char *k, *v;     // row 0 of the head
  int64_t stride;        // bytes a row
  int n;                 // keys that there are
  const int32_t* table;  // pages, or null
  int shift, npages;
  bool flat;             // rows one after another, 64 of them within 2 GiB: the DMA takes buffer offsets
  int held = -1;         // pages held .. held + 63 of the table lie in `page`, one a lane: the loop over
  int page = 0;          // the blocks then loads nothing that the compiler would wait for
  bool none = false;     // a page that is none lay among those held so far

  __device__ __forceinline__ bool there(int pg) const { return pg >= 0 && pg < npages; }
  // The pages of the keys from j0 on, one a lane.
  __device__ __forceinline__ void hold(int j0) {
    const int last = (n - 1) >> shift;
    held = j0 >> shift;
    page = table[held + (threadIdx.x & 63) < last ? held + (threadIdx.x & 63) : last];
    none |= __builtin_amdgcn_ballot_w64(!there(page)) != 0;
  }
  // bit i: key j0 + i of 32 has a page
  __device__ __forceinline__ uint32_t present(int j0) const {
    const int j = j0 + (threadIdx.x & 31);
    return (uint32_t)__builtin_amdgcn_ballot_w64(there(table[(j < n ? j : n - 1) >> shift]));
  }
  // Byte offsets of the rows that this wave's share (of WAVES) of KEYS keys from j0 on reads.
  template <int KEYS, int WAVES>
  __device__ __forceinline__ void rows(int j0, int wave, int64_t (&off)[KEYS / RPD / WAVES]) {
    constexpr int N = KEYS / RPD / WAVES;
    static_assert(N * RPD * WAVES == KEYS, "whole DMA instructions");
    if (flat) return;
    const int lane = threadIdx.x & 63, r = lane / T::CPR;
    if (table) {
      const int p0 = j0 >> shift, p1 = (j0 + KEYS - 1 < n ? j0 + KEYS - 1 : n - 1) >> shift;
      // V is a block behind K: its pages too, where a wave has the lanes
      if (held < 0 || p0 < held || p1 >= held + 64) hold(j0 >= KEYS && p1 < ((j0 - KEYS) >> shift) + 64 ? j0 - KEYS : j0);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        int j = j0 + (i * WAVES + wave) * RPD + r;
        j = j < n ? j : n - 1;
        int pg = __builtin_amdgcn_ds_bpermute(((j >> shift) - held) << 2, page), at = j & ((1 << shift) - 1);
        if (none) {
          // keys of a page that is none are masked; their values, which meet a probability of 0, are those of a
          // key that there is: the first of a page held
          const uint64_t some = __builtin_amdgcn_ballot_w64(there(page));
          const int spare = some ? __builtin_amdgcn_readlane(page, __builtin_ctzll(some)) : 0;
          if (!there(pg)) {
            pg = spare;
            at = 0;
          }
        }
        off[i] = (((int64_t)pg << shift) + at) * stride;
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = j0 + (i * WAVES + wave) * RPD + r;
        off[i] = (int64_t)(j < n ? j : n - 1) * stride;
      }
    }
  }
  // This wave's share (of WAVES) of the DMA of KEYS keys of K or V from j0 on into tiles at dst; `off` from
  // rows(), where the keys are not flat. Features past head_dim repeat its last 16 bytes: they meet zeros
  // of Q, or are not stored. Flat rows past the last key read as zeros, others repeat it.
  template <bool V, int KEYS, int WAVES>
  __device__ __forceinline__ void load(int j0, const int64_t (&off)[KEYS / RPD / WAVES], KU_LDS unsigned char* dst, int wave, int dim) const {
    constexpr int N = KEYS / RPD / WAVES;
    const int lane = threadIdx.x & 63, last = dim * T::ES / 16 - 1;
    if (flat) {
      const int left = n - j0 < KEYS ? n - j0 : KEYS;
      const uint64_t at = reinterpret_cast<uint64_t>((V ? v : k) + (int64_t)j0 * stride);
      const uint64_t base = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(at >> 32)) << 32 |
                            (uint32_t)__builtin_amdgcn_readfirstlane((int)at);
      const auto R = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(base), (short)0,
                                                       __builtin_amdgcn_readfirstlane(left * (int)stride), 0x00020000);
      // the wave's first destination, opaque to the optimiser: hoisted, the M0 values of all the DMAs
      // would stay live in SGPRs across the loop and spill
      KU_LDS unsigned char* wd = dst + wave * 1024;
      asm volatile("" : "+s"(wd));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int r = (i * WAVES + wave) * RPD + lane / T::CPR;
        int c = (lane % T::CPR) ^ (V ? T::vswz(r) : T::kswz(r));
        c = c < last ? c : last;
        lds_dma16(R, (uint32_t)(r * (int)stride + c * 16), 0, (KU_LDS void*)(wd + i * WAVES * 1024));
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int blk = i * WAVES + wave, r = blk * RPD + lane / T::CPR;
        int c = (lane % T::CPR) ^ (V ? T::vswz(r) : T::kswz(r));
        c = c < last ? c : last;
        lds_dma16_g((V ? v : k) + off[i] + c * 16, (KU_LDS void*)(dst + blk * 1024));
      }
    }
  }
};

// the prefix, or sequence b's own `n` keys
template <int DT, int D, int DR>
__device__ __forceinline__ Keys<DT, D, DR> keys_of(const SdpaDev& a, bool own, int b, int n, int kvh) {
  using E = typename SdpaElem<DT>::T;
  Keys<DT, D, DR> S;
  const bool paged = own && a.page_shift >= 0;
  const int64_t base = kvh * (own ? a.head : a.phead) + (own && !paged ? b * a.seq_rows * a.row : 0);
  S.k = reinterpret_cast<const char*>(static_cast<const E*>(own ? a.k : a.pk) + base);
  S.v = reinterpret_cast<const char*>(static_cast<const E*>(own ? a.v : a.pv) + base);
  S.stride = (own ? a.row : a.prow) * (int)sizeof(E);
  S.n = own ? n : a.prefix;
  S.table = paged ? a.pages + b * a.per_seq : nullptr;
  S.shift = paged ? a.page_shift : 0;
  S.npages = a.npages;
  S.flat = !paged && S.stride >= a.dim * (int)sizeof(E) && S.stride < (1 << 25);  // rows apart, 64 of them within 2 GiB
  return S;
}

// blocks [first, last) of n that split i takes
__device__ __forceinline__ void split_range(const Div& splits, int n, int i, int& first, int& last) {
  int rest;
  const int each = splits.split(n, rest);
  first = i * each + std::min(i, rest);
  last = first + each + (i < rest);
}

// The unit that work-group i takes: of part `second`, number `unit`; false where it has none.
//
// Work-groups go to the eight XCDs in turn, and within one to its CUs in turn. Each XCD gets a run of
// every part's units (neighbouring units read the same keys, and then from one L2), and takes 32 of one
// part and 32 of the other by turns, so that a CU holds one of the prefix, which keeps its matrix cores
// busy, beside one of the sequences' own keys, which keeps its memory busy.
__device__ __forceinline__ bool unit_of(const SdpaPlan& p, int i, bool& second, int& unit) {
  const int x = i & 7, n0 = p.part[0].units, n1 = p.part[1].units;
  int j = i >> 3;
  const int c0 = (n0 + 7) >> 3, c1 = (n1 + 7) >> 3;
  // chunks of 32 alternate while both parts have whole ones, then what is left of either
  const int turns = std::min(c0, c1) / 32;
  if (j < turns * 64) {
    second = (j >> 5) & 1;
    j = (j >> 6) * 32 + (j & 31);
  } else {
    j -= turns * 32;
    second = j >= c0;
    if (second) j -= c0 - turns * 32;
  }
  const int n = second ? n1 : n0, q = n >> 3, r = n & 7;
  if (j >= q + (x < r)) return false;
  unit = x * q + (x < r ? x : r) + j;
  return true;
}

// The sequence of a batch of up to 64 that unit position i of the own keys takes: the longest first, so that
// the last work-groups to start are the shortest, and by turns over the XCDs, each of which has a run of
// positions. 64 sequences of 16 to 1024 keys beside 8192 shared ones: 44.4 us, 48.4 in their own order; 32
// sequences 27.4 and 27.6.
__device__ __forceinline__ int longest_first(const SdpaDev& a, int i, int& len) {
  const int lane = threadIdx.x & 63, n = a.batch;
  const int g = n & 7 ? (n & 3 ? (n & 1 ? 1 : 2) : 4) : 8, period = n / g;
  const int want = i * 8 % n + i / period;
  // ties by number: lengths and lanes in one key
  const int key = lane < n ? (sdpa_len(a, lane) << 6 | (63 - lane)) : -1;
  int rank = 0;
#pragma unroll
  for (int j = 0; j < 64; ++j) rank += __builtin_amdgcn_readlane(key, j) > key;
  const int b = __builtin_ctzll(__builtin_amdgcn_ballot_w64(lane < n && rank == want));
  len = __builtin_amdgcn_readlane(key, b) >> 6;
  return b;
}

// where a query's row lies
struct RowAt {
  int b, t, h;
  // row r of a kv head: of all sequences' rows, or of sequence `seq`
  __device__ __forceinline__ RowAt(const SdpaPlan& p, bool pooled, int seq, int kvh, int r) : b(seq) {
    if (pooled) b = p.by_seq.split(r, r);
    t = p.by_group.split(r, h);
    h += kvh * (int)p.by_group.d;
  }
  // its (b, t, h) index, and back
  __device__ __forceinline__ int64_t index(const SdpaDev& a) const { return ((int64_t)b * a.q_len + t) * a.q_heads + h; }
  __device__ __forceinline__ RowAt(const SdpaPlan& p, int row) { b = p.by_q_len.split(p.by_heads.split(row, h), t); }
};

// four consecutive features from d on of a query's output, normalised
template <int DT>
__device__ __forceinline__ void write_out(const SdpaDev& a, const RowAt& at, int d, f32x4 x) {
  using E = typename SdpaElem<DT>::T;
  if (d >= a.dim) return;
  E* out = static_cast<E*>(a.o) + at.b * a.ob + at.t * a.ot + at.h * a.oh + d;
  if constexpr (DT == GT_F32)
    *reinterpret_cast<f32x4*>(out) = x;
  else
    *reinterpret_cast<u32x2*>(out) = u32x2{pack2<DT>(x[0], x[1]), pack2<DT>(x[2], x[3])};
}

// not finite: 0 * x is not 0
__device__ __forceinline__ bool bad_sum(float x) { return !(x * 0.f == 0.f); }

// Every cache line of the arguments at once: read as they are needed, each line's first read waits for
// memory by itself.
template <class Args>
__device__ __forceinline__ void touch_arguments() {
  const auto* p = (const uint32_t __attribute__((address_space(4)))*)__builtin_amdgcn_kernarg_segment_ptr();
  uint32_t x[(sizeof(Args) + 63) / 64];
#pragma unroll
  for (size_t i = 0; i < sizeof(x) / 4; ++i) x[i] = p[i * 16];
#pragma unroll
  for (size_t i = 0; i < sizeof(x) / 4; ++i) asm volatile("" ::"s"(x[i]));
}

// LDS of a work-group beside the tiles of keys.
struct SdpaShared {
  float4 ml[4][32];
  uint32_t redo;
};

// One unit: a tile of rows against a split of its keys. SHARED: four waves of 32 rows share blocks of
// keys; else the waves deal the blocks of one tile of 32 rows among them.
template <int DT, int D, int DR, bool LSE, bool SHARED>
__device__ __forceinline__ void run_unit(const SdpaArgs& g, bool second, int id, unsigned char* lds_raw, SdpaShared& sh) {
  using T = Tile<DT, D, DR>;
  using E = typename SdpaElem<DT>::T;
  constexpr int ROWS = SHARED ? 128 : 32;
  KU_LDS unsigned char* lds = (KU_LDS unsigned char*)lds_raw;
  const SdpaDev& a = g.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const float c = a.scale * LOG2E;
  const SdpaPlan::Part& part = g.p.part[second];
  const bool joint = SHARED && g.p.joint, pooled = !joint && !second;

  // the work-group's (sequence,) kv head, row tile and split of the keys
  int tile, kvh, split;
  id = part.by_tiles.split(id, tile);
  id = g.p.by_kv.split(id, kvh);  // heads before splits: their rows lie next to each other
  int b = part.by_splits.split(id, split);
  int own_len = 0;
  if (second && g.p.sorted)
    b = longest_first(a, b, own_len);
  else if (!pooled)
    own_len = __builtin_amdgcn_readfirstlane(sdpa_len(a, b));
  const int per_seq = a.q_len * a.group, nrows = pooled ? a.batch * per_seq : per_seq;
  const int row0 = tile * ROWS + (SHARED ? wave * 32 : 0);  // of this wave
  // the tile's blocks: those of the prefix, then those of the sequence's own keys that its last row sees
  constexpr int bk = SHARED ? 32 * T::SB : 32;
  int own_n = 0;
  if (own_len) {
    const int last_row = std::min((tile + 1) * ROWS, nrows) - 1;
    int rest;
    own_n = std::max(0, own_len - (a.q_len - 1 - g.p.by_group.split(last_row, rest)));
  }
  const int np = second ? 0 : (a.prefix + bk - 1) / bk, no = (own_n + bk - 1) / bk;
  int split_first, split_last;
  split_range(part.by_splits, np + no, split, split_first, split_last);
  Rows<DT, D, DR, LSE> R;
  R.clear();
  R.limit = 0;
  if (threadIdx.x == 0) sh.redo = 0;
  __syncthreads();
  // a few rows' own pages are asked for before Q: their loads return in order, and the first DMA needs them
  Keys<DT, D, DR> ahead;
  if constexpr (!SHARED) {
    ahead = keys_of<DT, D, DR>(a, second, b, own_len, kvh);
    if (ahead.table && split_first + wave < split_last) ahead.hold((split_first + wave) * 32);
  }
  {
    const E* q = nullptr;
    if (row0 + (lane & 31) < nrows) {
      const RowAt at(g.p, pooled, b, kvh, row0 + (lane & 31));
      q = static_cast<const E*>(a.q) + at.b * a.qb + at.t * a.qt + at.h * a.qh;
      R.limit = own_len - (a.q_len - 1 - at.t);
    }
    R.load_q(q, a.dim);
  }

  // one run of keys after another: a joint tile's prefix and own keys, or the part's only ones
#pragma clang loop unroll(disable)
  for (int seg = second; seg <= (int)(second || joint); ++seg) {
    const int first = seg ? std::max(split_first, np) - np : split_first, last = seg ? split_last - np : std::min(split_last, np);
    if (first >= last) continue;
    Keys<DT, D, DR> S = SHARED ? keys_of<DT, D, DR>(a, seg, b, own_len, kvh) : ahead;
    const int all = seg ? 0 : a.prefix;  // keys that every query sees
    if constexpr (SHARED) {
      // Four waves of 32 rows over blocks of BK keys, two buffers for K and two for V.
      constexpr int BK = 32 * T::SB, TB = T::SB * T::KT, N = BK / Keys<DT, D, DR>::RPD / 4;
      const bool active = row0 < nrows;  // a wave past the last row only fetches
      auto kbuf = [&](int i) { return lds + i * TB; };
      auto vbuf = [&](int i) { return lds + (2 + i) * TB; };
      auto fetch = [&](int blk, auto is_v, KU_LDS unsigned char* dst) {
        int64_t off[N];
        S.template rows<BK, 4>(blk * BK, wave, off);
        S.template load<decltype(is_v)::value, BK, 4>(blk * BK, off, dst, wave, a.dim);
      };
      constexpr std::false_type IsK{};
      constexpr std::true_type IsV{};
      // keys that are not there or not seen
      auto mask = [&](f32x16 (&s)[T::SB], int blk) {
        if (blk * BK + BK > all) {
#pragma unroll
          for (int t = 0; t < T::SB; ++t) R.mask(s[t], (seg ? R.limit : all) - blk * BK - 32 * t);
          if (S.none)
#pragma unroll
            for (int t = 0; t < T::SB; ++t) R.mask_absent(s[t], S.present(blk * BK + 32 * t));
        }
      };
      if constexpr (DT == GT_F32) {
        // a step of f32 products takes longer than a read of LDS or the softmax: nothing to interleave
        fetch(first, IsK, kbuf(0));
        fetch(first, IsV, vbuf(0));
        for (int blk = first; blk < last; ++blk) {
          const int par = (blk - first) & 1;
          vm_wait<0>();
          __syncthreads();
          if (blk + 1 < last) {
            fetch(blk + 1, IsK, kbuf(par ^ 1));
            fetch(blk + 1, IsV, vbuf(par ^ 1));
          }
          if (!active) continue;
          f32x16 s[T::SB];
#pragma unroll
          for (int t = 0; t < T::SB; ++t) s[t] = R.scores(kbuf(par) + t * T::KT);
          mask(s, blk);
          R.rescale(s, c);
#pragma unroll
          for (int t = 0; t < T::SB; ++t) R.weigh(s[t], c, vbuf(par) + t * T::KT);
        }
        __syncthreads();  // the next run's first block goes where this one's last may lie
      } else {
        // K runs one block ahead of V: the products of block blk + 1's scores, which are independent of
        // block blk's softmax, are issued between its exponentials, each fragment of K read two products
        // ahead (a scheduling barrier after each group keeps them so). Two blocks a trip, so that the
        // parity of the buffers is a constant.
        constexpr int NM = 2 * T::DS;  // products of a block's scores, among 16 exponential pairs
        static_assert(T::SB == 2 && NM <= 16);
        auto step = [&](int blk, f32x16 (&sc)[2], f32x16 (&sn)[2], auto par) __attribute__((always_inline)) {
          constexpr int PAR = decltype(par)::value;
          if (blk + 2 < last) fetch(blk + 2, IsK, kbuf(PAR));
          if (blk + 1 < last) fetch(blk + 1, IsV, vbuf(PAR ^ 1));
          if (active) {
            mask(sc, blk);
            R.rescale(sc, c);
            const float em = R.exponent();
            u32x4 p[4], lo[4];
            typename Rows<DT, D, DR, LSE>::Sums rs;
            const int r = lane & 31;
            const KU_LDS unsigned char* LK = kbuf(PAR ^ 1);
            auto kread = [&](int m) {
              return *(const KU_LDS u32x4*)(LK + ((m & 1) * 32 + r) * T::RB + (((2 * (m >> 1) + h) ^ T::kswz(r)) << 4));
            };
            u32x4 kf[3];
            kf[0] = kread(0);
            kf[1] = kread(1);
            __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int m = 0; m < NM; ++m) {
              if (m + 2 < NM) kf[(m + 2) % 3] = kread(m + 2);
#pragma unroll
              for (int i = 16 * m / NM; i < 16 * (m + 1) / NM; ++i) {
                const int te = i >> 3, v2 = i & 7;
                const float p0 = __builtin_amdgcn_exp2f(fmaf(sc[te][2 * v2], c, em));
                const float p1 = __builtin_amdgcn_exp2f(fmaf(sc[te][2 * v2 + 1], c, em));
                uint32_t rest = 0;
                p[2 * te + (v2 >> 2)][v2 & 3] = rs.add(v2 & 1, p0, p1, rest);
                lo[2 * te + (v2 >> 2)][v2 & 3] = rest;
              }
              if (m < 2) sn[m & 1] = f32x16{};
              mfma_step<DT>(kf[m % 3], R.q[m >> 1], sn[m & 1]);
              __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_s_setprio(0);
            R.join(rs);
            R.product(p, lo, vbuf(PAR));
          }
          vm_wait<0>();
          __syncthreads();
        };
        fetch(first, IsK, kbuf(0));
        fetch(first, IsV, vbuf(0));
        if (first + 1 < last) fetch(first + 1, IsK, kbuf(1));
        vm_wait<0>();
        __syncthreads();
        f32x16 sa[2], sb[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) sa[t] = R.scores(kbuf(0) + t * T::KT);
        __syncthreads();  // every wave has read K's first buffer
        for (int blk = first; blk < last; blk += 2) {
          step(blk, sa, sb, std::integral_constant<int, 0>{});
          if (blk + 1 < last) step(blk + 1, sb, sa, std::integral_constant<int, 1>{});
        }
      }
    } else {
      // The waves take blocks of 32 keys in turn, each by itself: K of its next block is fetched once this
      // one's scores are done, V once its products are, so either is on its way while the other is used.
      constexpr int N = 32 / Keys<DT, D, DR>::RPD;
      KU_LDS unsigned char *K = lds + wave * 2 * T::KT, *V = K + T::KT;
      int64_t off[N];
      auto fetch_k = [&](int blk) {
        S.template rows<32, 1>(blk * 32, 0, off);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the last block's K has been read
        S.template load<false, 32, 1>(blk * 32, off, K, 0, a.dim);
      };
      auto fetch_v = [&](int blk) {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        S.template load<true, 32, 1>(blk * 32, off, V, 0, a.dim);
      };
      int blk = first + wave;
      if (blk < last) {
        fetch_k(blk);
        fetch_v(blk);
      }
      for (; blk < last; blk += 4) {
        const bool more = blk + 4 < last;
        vm_wait<N>();  // K is there, V on its way
        asm volatile("" ::: "memory");
        f32x16 s[1];
        s[0] = R.scores(K);
        if (more) fetch_k(blk + 4);
        if (blk * 32 + 32 > all) {
          R.mask(s[0], (seg ? R.limit : all) - blk * 32);
          if (S.none) R.mask_absent(s[0], S.present(blk * 32));
        }
        R.rescale(s, c);
        if (more)
          vm_wait<N>();
        else
          vm_wait<0>();
        asm volatile("" ::: "memory");
        R.weigh(s[0], c, V);
        if (more) fetch_v(blk + 4);
      }
    }
  }

  {
  // ---- the results ----
  // The arguments read afresh: kept across the loop, what only this part uses cost it its registers.
  const SdpaArgs* afresh = static_cast<const SdpaArgs*>((const void*)__builtin_amdgcn_kernarg_segment_ptr());
  asm volatile("" : "+s"(afresh));
  const SdpaArgs& g = *afresh;
  const SdpaDev& a = g.a;
  auto at_row = [&](int r) { return RowAt(g.p, pooled, b, kvh, r); };
  const bool there = row0 + (lane & 31) < nrows;
  const int slots = g.p.slots, slot = second ? g.p.part[0].splits + split : split;
  R.l += other_half(R.l);
  R.w = Rows<DT, D, DR, LSE>::WHOLE ? R.w + other_half(R.w) : R.l;
  uint32_t redo = 0;  // rows of this wave that are done again
  __syncthreads();
  if constexpr (SHARED) {
    const RowAt at = at_row(there ? row0 + (lane & 31) : 0);
    const int64_t row = at.index(a);
    if (slots > 1) {
      if (there) {
        float* o = g.po + (row * slots + slot) * D;
#pragma unroll
        for (int t = 0; t < T::DTL; ++t)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            *reinterpret_cast<f32x4*>(o + 32 * t + 8 * v + 4 * h) =
                f32x4{R.o[t][4 * v], R.o[t][4 * v + 1], R.o[t][4 * v + 2], R.o[t][4 * v + 3]};
        if (h == 0) g.ml[row * slots + slot] = make_float4(R.m, R.l, R.w, 0.f);
      }
    } else {
      float z = R.l * 0.f;
#pragma unroll
      for (int t = 0; t < T::DTL; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) z = fmaf(R.o[t][v], 0.f, z);
      z += other_half(z);
      const bool bad = there && (!(z == 0.f) || R.l == 0.f);
      if (there && !bad) {
        const float inv = 1.f / R.l;
#pragma unroll
        for (int t = 0; t < T::DTL; ++t)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            write_out<DT>(a, at, 32 * t + 8 * v + 4 * h,
                          f32x4{R.o[t][4 * v] * inv, R.o[t][4 * v + 1] * inv, R.o[t][4 * v + 2] * inv, R.o[t][4 * v + 3] * inv});
        if (a.lse && h == 0) a.lse[row] = lse_of<DT>(R.m, R.w);
      }
      redo = (uint32_t)__builtin_amdgcn_ballot_w64(bad && h == 0);
    }
  } else {
    // the waves' results of the same 32 rows are brought to one maximum and added through LDS
    if (h == 0) sh.ml[wave][lane] = make_float4(R.m, R.l, R.w, 0.f);
    __syncthreads();
    float m = -INFINITY, l = 0.f, whole = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, sh.ml[w][lane & 31].x);
    const float from = m == -INFINITY ? 0.f : m;  // nothing seen
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float4 x = sh.ml[w][lane & 31];
      const float e = __builtin_amdgcn_exp2f(x.x - from);
      l = fmaf(e, x.y, l);
      whole = fmaf(e, x.z, whole);
    }
    const float mine = __builtin_amdgcn_exp2f(R.m - from);
    constexpr int CH = D / 4;  // 16-byte chunks of a row, swizzled by the row
    if (there) {
      KU_LDS unsigned char* o = lds + wave * 32 * D * 4 + (lane & 31) * D * 4;
#pragma unroll
      for (int t = 0; t < T::DTL; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          *(KU_LDS f32x4*)(o + (((8 * t + 2 * v + h) ^ (lane & (CH - 1) & 31)) << 4)) =
              f32x4{R.o[t][4 * v] * mine, R.o[t][4 * v + 1] * mine, R.o[t][4 * v + 2] * mine, R.o[t][4 * v + 3] * mine};
    }
    __syncthreads();
    if (wave == 0 && h == 0) sh.ml[0][lane] = make_float4(m, l, whole, 0.f);
    __syncthreads();
    const int rows = std::min(32, nrows - row0);
    for (int i = threadIdx.x; i < rows * (DR / 4); i += 256) {
      const int r = i / (DR / 4), ch = i % (DR / 4);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) o += *(const KU_LDS f32x4*)(lds + w * 32 * D * 4 + r * D * 4 + ((ch ^ (r & (CH - 1) & 31)) << 4));
      const float4 x = sh.ml[0][r];
      const RowAt where = at_row(row0 + r);
      const int64_t at = where.index(a);
      if (slots > 1) {
        *reinterpret_cast<f32x4*>(g.po + (at * slots + slot) * D + ch * 4) = o;
        if (ch == 0) g.ml[at * slots + slot] = x;
      } else {
        if (bad_sum(x.y) || x.y == 0.f || bad_sum(o[0]) || bad_sum(o[1]) || bad_sum(o[2]) || bad_sum(o[3])) atomicOr(&sh.redo, 1u << r);
        const float inv = 1.f / x.y;
        write_out<DT>(a, where, ch * 4, o * inv);
        if (ch == 0 && a.lse) a.lse[at] = lse_of<DT>(x.x, x.z);
      }
    }
    if (slots == 1) {
      __syncthreads();  // also orders the outputs written so far before those written again
      redo = __builtin_amdgcn_readfirstlane(sh.redo) & (0x11111111u << wave);
    }
  }
  while (redo) {
    const int i = __builtin_ctz(redo);
    redo &= redo - 1;
    const RowAt at = at_row(row0 + i);
    sdpa_one<DT>(a, at.b, at.t, at.h, reinterpret_cast<float*>(lds_raw + wave * 32 * D * 4));
  }
  }
}

template <int DT, int D, int DR, bool LSE>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) sdpa_tiles_k(SdpaArgs g) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[Tile<DT, D, DR>::LDS];
  __shared__ SdpaShared sh;
  touch_arguments<SdpaArgs>();
  bool second;
  int unit;
  if (!unit_of(g.p, blockIdx.x, second, unit)) return;
  if (g.p.part[second].shared)
    run_unit<DT, D, DR, LSE, true>(g, second, unit, lds, sh);
  else
    run_unit<DT, D, DR, LSE, false>(g, second, unit, lds, sh);
}

// Joins the partial results of rows, eight slots a lane at a time: with SIDE slots of a row side by side
// in a wave, or several rows beside each other. One round of loads where that covers the slots.
template <int DT, int D, int SIDE>
__global__ void __launch_bounds__(256) sdpa_join_k(SdpaArgs g) {
  constexpr int L = D / 4, ROWS = 64 / (L * SIDE), U = 8;  // lanes a slot's output takes, rows of a wave
  __shared__ float lds[4][kSdpaMaxDim];
  const SdpaDev& a = g.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), ch = lane % L, sub = lane / L % SIDE;
  const int rows = a.batch * a.q_len * a.q_heads, row0 = ((int)blockIdx.x * 4 + wave) * ROWS, row = row0 + lane / (L * SIDE);
  const bool there = row < rows;
  const int n = there ? g.p.slots : 0;
  const float4* ml = g.ml + (int64_t)row * g.p.slots;
  const f32x4* po = reinterpret_cast<const f32x4*>(g.po + (int64_t)row * g.p.slots * D) + ch;
  float m = -INFINITY, l = 0.f, whole = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int i0 = 0; i0 < g.p.slots; i0 += U * SIDE) {
    f32x4 x[U];
    float4 y[U];
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const int i = i0 + j * SIDE + sub;
      x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      y[j] = make_float4(-INFINITY, 0.f, 0.f, 0.f);
      if (i < n) {
        if (ch * 4 < a.dim) x[j] = po[i * L];
        y[j] = ml[i];
      }
    }
    float top = m;
#pragma unroll
    for (int j = 0; j < U; ++j) top = fmaxf(top, y[j].x);
#pragma unroll
    for (int o = L; o < L * SIDE; o <<= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    const float from = top == -INFINITY ? 0.f : top, old = __builtin_amdgcn_exp2f(m - from);
    m = top;
    l *= old;
    whole *= old;
    acc *= old;
#pragma unroll
    for (int j = 0; j < U; ++j) {
      const float w = __builtin_amdgcn_exp2f(y[j].x - from);  // 0 for a slot that saw nothing
      l = fmaf(w, y[j].y, l);
      whole = fmaf(w, y[j].z, whole);
      acc += x[j] * w;
    }
  }
  // the slots side by side are added in one order in every lane
#pragma unroll
  for (int o = L; o < L * SIDE; o <<= 1) {
    l += __shfl_xor(l, o, 64);
    whole += __shfl_xor(whole, o, 64);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] += __shfl_xor(acc[k], o, 64);
  }
  const RowAt at(g.p, there ? row : 0);
  // a row's lanes that are not finite: the whole row is done again
  const uint64_t bad = __builtin_amdgcn_ballot_w64(
      there && (l == 0.f || bad_sum(l) || bad_sum(acc[0]) || bad_sum(acc[1]) || bad_sum(acc[2]) || bad_sum(acc[3])));
  constexpr uint64_t LANES = L * SIDE == 64 ? ~0ull : (1ull << (L * SIDE % 64)) - 1;
  if (there && (bad >> (lane / (L * SIDE) * (L * SIDE)) & LANES) == 0) {
    if (sub == 0) write_out<DT>(a, at, ch * 4, acc * (1.f / l));
    if (a.lse && ch == 0 && sub == 0) a.lse[row] = lse_of<DT>(m, whole);
  }
  if (bad)
    for (int i = 0; i < ROWS; ++i)
      if (bad >> (i * L * SIDE) & LANES) {
        const RowAt again(g.p, row0 + i);
        sdpa_one<DT>(a, again.b, again.t, again.h, lds[wave]);
      }
}

SdpaDev device_args(const KuHipSdpaPrefixArgs& a) {
  SdpaDev d;
  d.q = a.q;
  d.pk = a.prefix_k;
  d.pv = a.prefix_v;
  d.k = a.own_k;
  d.v = a.own_v;
  d.o = a.out;
  d.lse = a.lse;
  d.qb = a.q_batch_stride;
  d.qt = a.q_token_stride;
  d.qh = a.q_head_stride;
  d.ob = a.out_batch_stride;
  d.ot = a.out_token_stride;
  d.oh = a.out_head_stride;
  d.prow = a.prefix_row_stride;
  d.phead = a.prefix_head_stride;
  d.row = a.own_row_stride;
  d.head = a.own_head_stride;
  d.lens = a.own_lens;
  d.pages = a.pages;
  d.seq_rows = (int64_t)a.own_seq_rows;
  d.per_seq = (int64_t)a.pages_per_seq;
  d.batch = (int32_t)a.batch;
  d.q_len = (int32_t)a.q_len;
  d.q_heads = (int32_t)a.q_heads;
  d.kv_heads = (int32_t)a.kv_heads;
  d.dim = (int32_t)a.head_dim;
  d.group = (int32_t)(a.q_heads / a.kv_heads);
  d.prefix = (int32_t)a.prefix_len;
  d.own_max = (int32_t)a.own_max;
  d.page_shift = a.pages ? __builtin_ctzll(a.page_size) : -1;
  d.npages = a.pages ? (int32_t)(a.own_rows / a.page_size) : 0;
  d.scale = a.scale;
  return d;
}

SdpaPlan make_plan(const KuHipSdpaPrefixArgs& a) {
  SdpaPlan p;
  const int64_t group = (int64_t)(a.q_heads / a.kv_heads), per_seq = (int64_t)a.q_len * group, kv = (int64_t)a.kv_heads,
                nb = (int64_t)a.batch, cu = cu_count();
  // One sequence's rows walk the prefix by themselves where they fill tiles of 128 to four fifths; else
  // the sequences' rows share tiles over it.
  p.joint = (per_seq + 127) / 128 * 128 * 4 <= per_seq * 5;
  auto cut = [&](SdpaPlan::Part& part, int64_t rows, int64_t items, int64_t keys, int64_t want, bool halves = false) {
    if (keys == 0 || items == 0 || rows == 0) return;
    // Tiles of 128 rows read a key once where four tiles of 32 read it four times (from L2, and with every
    // wave's own DMA); tiles of 32 spread few rows' keys over all four waves. us of both kernels, 128 / 32
    // rows, bf16, 32 heads over 8 of 128, 8192 shared keys: 48 rows 20.5 / 17.4, 96 rows 23.2 / 21.0, 128 rows
    // 25.0 / 22.1; 65536 keys: 64 rows 69.0 / 68.4, 128 rows 75.0 / 106: what short prefixes lose is less than
    // what long ones would.
    part.shared = rows > 64;
    part.tiles = (int)((rows + (part.shared ? 127 : 31)) / (part.shared ? 128 : 32));
    const int64_t bk = part.shared ? (a.dtype == KU_F32 ? 32 : 64) : 128, blocks = (keys + bk - 1) / bk;
    const int64_t least = halves && items * part.tiles <= cu ? 2 : 1;
    part.splits = (int)std::max<int64_t>(1, std::min<int64_t>({std::max(want / (items * part.tiles), least), blocks, 256}));
    part.units = (int)(items * part.tiles * part.splits);
    part.by_tiles = Div(part.tiles);
    part.by_splits = Div(part.splits);
  };
  if (p.joint) {
    // two a CU, so that one's products meet the other's exponentials: 256 queries each of 4 sequences on 4096
    // shared keys, 16 heads over 4 of 128, 63 us and 71 with one; of one sequence 33 and 32; of 8 sequences,
    // heads of 64, 65 and 82
    cut(p.part[0], per_seq, nb * kv, (int64_t)(a.prefix_len + a.own_max), 2 * cu);
  } else {
    // A unit costs about 4 us before its first product and 3 to write its partial result, so more of them
    // than CUs lose: the prefix alone 29 us with one a CU, 37 with two and 36 with one for two CUs (256 rows,
    // 8192 keys), 76 / 85 / 107 (128 rows, 65536 keys). Beside own keys of half its length or more it leaves
    // every other CU to them: 49 us, and 55 with one a CU (64 sequences of up to 1024 own keys), 33 and 38
    // (32 sequences). own_max stands for the lengths, which the host does not know: with up to 16 own keys
    // and an own_max of 16 / 4096 8 sequences take 16.1 / 16.4, 16 16.4 / 19.8, 32 24.3 / 25.6, 64 28.6 / 36.1.
    const bool beside = nb * (int64_t)a.own_max * 2 >= (int64_t)a.prefix_len;
    cut(p.part[0], nb * per_seq, kv, (int64_t)a.prefix_len, beside ? cu / 2 : cu);
    // Own keys: a unit a CU, but halves where each sequence would be one unit and every CU had at most one,
    // unless the prefix outlasts them. us of the tiles with cu / 2 and cu units wanted, bf16, 8192 shared and up to
    // 1024 own keys: 4 sequences 12.7 / 13.0, 8 15.2 / 15.2, 16 18.2 / 18.4; up to 8192 own keys: 4 sequences 36.4 /
    // 27.4, one 15.0 / 15.2. Wholes, halves and quarters: 32 sequences 28.8 / 27.5 / 31.5, 64 sequences (which
    // stay whole) 44.3 / 48.4 / 57.9.
    cut(p.part[1], per_seq, nb * kv, (int64_t)a.own_max, cu, beside);
  }
  p.slots = p.part[0].splits + p.part[1].splits;
  // keys fit 25 bits beside a lane's number; one round of work-groups needs no order
  p.sorted = a.batch > 1 && a.batch <= 64 && a.own_max < (1u << 25) && p.part[1].units > cu;
  p.by_kv = Div(kv);
  p.by_group = Div(group);
  p.by_seq = Div(per_seq);
  p.by_q_len = Div((int64_t)a.q_len);
  p.by_heads = Div((int64_t)a.q_heads);
  return p;
}

int padded_dim(size_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

int64_t tile_groups(const SdpaPlan& p) {
  return 8 * (((int64_t)p.part[0].units + 7) / 8 + ((int64_t)p.part[1].units + 7) / 8);
}
// Few slots: several rows a wave (32768 rows of 64, two slots: 7.4 us, and 14 with a wave a row).
int64_t join_groups(int64_t rows, int slots, int d) {
  const int64_t each = 4 * (slots <= 8 ? 256 / d : 1);
  return slots == 1 ? 0 : (rows + each - 1) / each;
}

template <int DT, int D, int DR>
void launch_d(const SdpaArgs& g, hipStream_t s) {
  const unsigned groups = (unsigned)tile_groups(g.p);
  if (groups && g.a.lse)
    launch(sdpa_tiles_k<DT, D, DR, Rows<DT, D, DR, true>::WHOLE>, dim3(groups), 256, 0, s, g);
  else if (groups)
    launch(sdpa_tiles_k<DT, D, DR, false>, dim3(groups), 256, 0, s, g);
  const unsigned joins = (unsigned)join_groups((int64_t)g.a.batch * g.a.q_len * g.a.q_heads, g.p.slots, D);
  if (joins == 0) return;
  if (g.p.slots <= 8)
    launch(sdpa_join_k<DT, D, 1>, dim3(joins), 256, 0, s, g);
  else
    launch(sdpa_join_k<DT, D, 256 / D>, dim3(joins), 256, 0, s, g);
}
template <int DT>
void launch_t(const SdpaArgs& g, int d, hipStream_t s) {
  switch (d) {
    case 32: launch_d<DT, 32, 32>(g, s); break;
    case 64: launch_d<DT, 64, 64>(g, s); break;
    default: g.a.dim <= 96 ? launch_d<DT, 128, 96>(g, s) : launch_d<DT, 128, 128>(g, s); break;
  }
}

}  // namespace

void check_sdpa_prefix(const KuHipSdpaPrefixArgs& a) {
  require(a.size == sizeof(KuHipSdpaPrefixArgs), "size is not sizeof(KuHipSdpaPrefixArgs)");
  const int64_t w = (int64_t)float_width(a.dtype, "dtype"), v = 16 / w, d = (int64_t)a.head_dim;
  require(std::isfinite(a.scale) && a.scale > 0, "scale must be positive and finite");
  require(a.head_dim >= 1 && a.head_dim <= kSdpaMaxDim && d % v == 0,
          "head_dim must be a multiple of 16 bytes, up to 128 elements");
  require(a.q_len >= 1 && a.q_heads >= 1 && a.kv_heads >= 1, "q_len, q_heads and kv_heads must be positive");
  require(a.q_heads % a.kv_heads == 0, "q_heads must be a multiple of kv_heads");
  const size_t most = 0x7fffffff;
  require(a.batch <= most && a.q_len <= most && a.q_heads <= most &&
              (__int128)a.batch * a.q_len * a.q_heads <= (__int128)1 << 30,
          "more than 2^30 queries");
  require(a.prefix_len <= most - 256 && a.own_max <= most - 256 && a.q_len <= most - 256, "more than 2^31 - 257 keys");
  auto strides16 = [&](std::initializer_list<int64_t> s) {
    for (int64_t x : s) require(x % v == 0, "strides must be multiples of 16 bytes");
  };
  auto pointers16 = [&](std::initializer_list<const void*> ps) {
    for (const void* p : ps) {
      require(p != nullptr, "null device pointer");
      require(aligned_to(p, 16), "pointers must be 16-byte aligned");
    }
  };
  require(aligned_to(a.lse, 4) && aligned_to(a.own_lens, 4) && aligned_to(a.pages, 4),
          "lse, own_lens and pages must be 4-byte aligned");
  require(aligned_to(a.scratch, 16), "scratch must be 16-byte aligned");
  strides16({a.q_batch_stride, a.q_token_stride, a.q_head_stride, a.out_batch_stride, a.out_token_stride,
             a.out_head_stride});
  const std::initializer_list<Axis> q_axes = {{a.batch, a.q_batch_stride}, {a.q_len, a.q_token_stride}, {a.q_heads, a.q_head_stride}},
                                    out_axes = {{a.batch, a.out_batch_stride}, {a.q_len, a.out_token_stride}, {a.q_heads, a.out_head_stride}};
  span_of(d, q_axes, "q");
  written_span(d, out_axes, "out");
  const Buffer q(a.q, d, q_axes, w), out(a.out, d, out_axes, w);
  if (a.batch) {
    pointers16({a.q, a.out});
    require(!share(q, out), "out overlaps q");
  }
  if (a.prefix_len) {
    pointers16({a.prefix_k, a.prefix_v});
    strides16({a.prefix_row_stride, a.prefix_head_stride});
    span_of(d, {{a.prefix_len, a.prefix_row_stride}, {a.kv_heads, a.prefix_head_stride}}, "prefix_k");
  }
  if (a.own_max && a.batch) {
    pointers16({a.own_k, a.own_v});
    require(a.own_lens, "own_max without own_lens");
    strides16({a.own_row_stride, a.own_head_stride});
    require(a.own_rows <= ((size_t)1 << 40), "too many own_rows");
    span_of(d, {{a.own_rows, a.own_row_stride}, {a.kv_heads, a.own_head_stride}}, "own_k");
    if (a.pages) {
      require(a.page_size && (a.page_size & (a.page_size - 1)) == 0 && a.page_size <= ((size_t)1 << 30),
              "page_size must be a power of two");
      require(a.pages_per_seq <= most && (__int128)a.pages_per_seq * a.page_size >= (__int128)a.own_max,
              "pages_per_seq pages do not hold own_max keys");
      require(a.own_rows / a.page_size >= 1 && a.own_rows / a.page_size <= most, "own_rows holds no page, or too many");
    } else {
      require(a.batch == 1 || a.own_seq_rows >= a.own_max, "own_seq_rows is less than own_max");
      require(a.own_seq_rows <= ((size_t)1 << 40) &&
                  (__int128)(a.batch - 1) * a.own_seq_rows + a.own_max <= (__int128)a.own_rows,
              "own_rows does not hold own_max keys of every sequence");
    }
  }
  if (a.batch) {
    const SdpaPlan p = make_plan(a);
    require(tile_groups(p) <= max_blocks(256) && join_groups(a.batch * a.q_len * a.q_heads, p.slots, padded_dim(a.head_dim)) <= max_blocks(256),
            "more queries than one launch takes");
    // what is written shares nothing with what is read, nor with each other
    const auto flat = [](const void* p, size_t n, size_t bytes) { return Buffer(p, (int64_t)n, {}, bytes); };
    const size_t own = a.own_max ? 1 : 0, prefix = a.prefix_len ? 1 : 0;
    const auto keys = [&](const void* p, size_t there, size_t rows, int64_t row, int64_t head) {
      return Buffer(there ? p : nullptr, d, {{rows, row}, {a.kv_heads, head}}, w);
    };
    const __int128 table = (__int128)a.batch * (__int128)a.pages_per_seq;
    const Buffer read[] = {q,
                           keys(a.prefix_k, prefix, a.prefix_len, a.prefix_row_stride, a.prefix_head_stride),
                           keys(a.prefix_v, prefix, a.prefix_len, a.prefix_row_stride, a.prefix_head_stride),
                           keys(a.own_k, own, a.own_rows, a.own_row_stride, a.own_head_stride),
                           keys(a.own_v, own, a.own_rows, a.own_row_stride, a.own_head_stride),
                           flat(own ? a.own_lens : nullptr, a.batch, 4),
                           flat(own ? a.pages : nullptr, (size_t)std::min<__int128>(table, (__int128)1 << 58), 4)};
    const Buffer written[] = {out, flat(a.lse, a.batch * a.q_len * a.q_heads, 4), flat(a.scratch, a.scratch ? sdpa_prefix_scratch_bytes(a) : 0, 1)};
    for (const Buffer& y : written) {
      for (const Buffer& x : read) require(!share(y, x), "out, lse or scratch overlaps an input");
      for (const Buffer& x : written) require(&x >= &y || !share(y, x), "two of out, lse and scratch overlap");
    }
  }
}

size_t sdpa_prefix_scratch_bytes(const KuHipSdpaPrefixArgs& a) {
  const SdpaPlan p = make_plan(a);
  if (a.batch == 0 || p.slots <= 1) return 0;
  return a.batch * a.q_len * a.q_heads * (size_t)p.slots * (padded_dim(a.head_dim) * sizeof(float) + sizeof(float4));
}

void launch_sdpa_prefix(const KuHipSdpaPrefixArgs& a, void* scratch, hipStream_t s) {
  if (a.batch == 0) return;
  SdpaArgs g;
  g.a = device_args(a);
  g.p = make_plan(a);
  const int d = padded_dim(a.head_dim);
  g.po = static_cast<float*>(scratch);
  g.ml = reinterpret_cast<float4*>(g.po + a.batch * a.q_len * a.q_heads * (size_t)g.p.slots * d);
  switch (a.dtype) {
    case KU_BF16: launch_t<GT_BF16>(g, d, s); break;
    case KU_F16: launch_t<GT_F16>(g, d, s); break;
    default: launch_t<GT_F32>(g, d, s); break;
  }
}

}  // namespace ku::hipbk
