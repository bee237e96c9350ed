// Attention of a batch that shares its first keys (ku_hip_sdpa_prefix).
//
//   out[b, t, h] = sum_j softmax_j(scale q[b, t, h] . K_j) V_j
// over the shared prefix and the keys of sequence b that query t sees.
//
// The queries that read one kv head are the rows of a matrix product with its keys. Over the prefix
// the rows of every sequence go through together ("pooled"): a key is read once for the whole batch,
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
// The keys of a tile are cut into splits until the chip is full; each split leaves its maximum, sum and
// unnormalised output in f32 in the scratch and a second kernel joins them in split order. A tile with
// one split writes its output itself.
//
// Only rows that some query sees are ever loaded (places past the end repeat the last one), so what lies
// behind them cannot matter. A query whose sums are not finite, or that saw nothing, is done again from
// the definition by sdpa_one: an infinity or NaN in a value that another query of the tile sees, and a
// page that is none, come out right that way.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "decode.h"
#include "lds_dma.h"
#include "sdpa_prefix.h"

namespace ku::hipbk {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef short s16x4 __attribute__((__vector_size__(4 * sizeof(short))));
#define KU_LDS __attribute__((address_space(3)))

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;
// The running maximum moves only when a block exceeds it by more than this (in powers of two), so most
// blocks leave O alone; probabilities reach 2^8 at most before they are normalised.
constexpr float RESCALE = 8.f;

// How a call is cut into work-groups.
struct SdpaPlan {
  bool joint = false;
  // [0] the prefix with the rows of all sequences (joint: prefix and own keys of a sequence's rows);
  // [1] a sequence's own keys with its rows
  struct Part {
    bool shared = false;  // four waves of 32 rows over the same blocks of keys; else 32 rows, the blocks dealt to the waves
    int tiles = 0, splits = 0;   // row tiles a kv head (and sequence), splits of their keys
    int units = 0;               // work-groups: tiles times splits of all of them
  } part[2];
  int slots = 0;  // partial results a row
};

struct SdpaArgs {
  SdpaDev a;
  SdpaPlan p;
  float* po;   // [rows][slots][D]
  float2* ml;  // [rows][slots]: maximum in powers of two, sum
};

template <int DT>
__device__ __forceinline__ void mfma_step(const u32x4& a, const u32x4& b, f32x16& c) {
  if constexpr (DT == GT_BF16) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else if constexpr (DT == GT_F16) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  } else {
    const f32x4 x = __builtin_bit_cast(f32x4, a), y = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
  }
}

template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const f32x2 v = {lo, hi};
  if constexpr (DT == GT_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}
template <int DT>
__device__ __forceinline__ float sum2(uint32_t pair, float c) {
  if constexpr (DT == GT_BF16) {
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, pair), one, c, false);
  } else {
    const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, pair), one, c, false);
  }
}
// the value of the other half of the wave
__device__ __forceinline__ float other_half(float x) {
  const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32) ? sw[0] : sw[1]);
}

template <int DT, int D>
struct Tile {
  static constexpr int ES = DT == GT_F32 ? 4 : 2;
  static constexpr int RB = D * ES;          // bytes of a row in LDS
  static constexpr int CPR = RB / 16;        // 16-byte chunks of a row
  static constexpr int KT = 32 * RB;         // bytes of 32 keys
  static constexpr int DS = CPR / 2;         // chunk pairs: steps of S^T
  static constexpr int DTL = D / 32;         // 32-row tiles of O^T
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
template <int DT, int D>
struct Rows {
  using T = Tile<DT, D>;
  u32x4 q[T::DS];
  f32x16 o[T::DTL];
  float m, l;  // m in powers of two, already times scale
  int limit;   // own keys that this lane's query sees

  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
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
  // scores of 32 keys
  __device__ __forceinline__ f32x16 scores(const KU_LDS unsigned char* K) const {
    const int lane = threadIdx.x & 63, r = lane & 31, h = lane >> 5;
    f32x16 s = {};
#pragma unroll
    for (int i = 0; i < T::DS; ++i) {
      const u32x4 k = *(const KU_LDS u32x4*)(K + r * T::RB + (((2 * i + h) ^ T::kswz(r)) << 4));
      mfma_step<DT>(k, q[i], s);
    }
    return s;
  }
  // keys from `left` on are not seen (left counts from the tile's first key)
  static __device__ __forceinline__ void mask(f32x16& s, int left) {
    const int lim = left - 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int v = 0; v < 16; ++v)
      if ((v >> 2) * 8 + (v & 3) >= lim) s[v] = -INFINITY;
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
#pragma unroll
      for (int t = 0; t < T::DTL; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[t][v] *= corr;
    }
  }
  // O^T += V^T P^T over 32 keys; the sum adds the probabilities that the product uses
  __device__ __forceinline__ void weigh(const f32x16& s, float c, const KU_LDS unsigned char* V) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    const float em = m == -INFINITY ? 0.f : -m;  // nothing seen so far: every score is -inf
    if constexpr (DT == GT_F32) {
      const int r = lane & 31;
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        const float p = __builtin_amdgcn_exp2f(fmaf(s[v], c, em));
        l += p;
        const int key = (v >> 2) * 8 + (v & 3) + 4 * h;
#pragma unroll
        for (int t = 0; t < T::DTL; ++t) {
          const int d = 32 * t + r;
          const float x = *(const KU_LDS float*)(V + key * T::RB + (((d >> 2) ^ T::vswz(key)) << 4) + (d & 3) * 4);
          o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(x, p, o[t], 0, 0, 0);
        }
      }
    } else {
      u32x4 p[2];
      float rs[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float p0 = __builtin_amdgcn_exp2f(fmaf(s[2 * i], c, em));
        const float p1 = __builtin_amdgcn_exp2f(fmaf(s[2 * i + 1], c, em));
        const uint32_t pp = pack2<DT>(p0, p1);
        rs[i & 1] = sum2<DT>(pp, rs[i & 1]);
        p[i >> 2][i & 3] = pp;
      }
      l += rs[0] + rs[1];
      // V^T fragments by transposing reads: in each 16-lane group input lane 4 k' + j points at key
      // row k', dims 4 j.. + 3, and output lane i receives keys 0..3 of dim i; two of them fetch the
      // keys that the probability registers hold, 16 s + 4 h + 0..3 and those + 8
      const int g = lane >> 4, c16 = lane & 15;
#pragma unroll
      for (int st = 0; st < 2; ++st)
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
          mfma_step<DT>(u32x4{half[0][0], half[0][1], half[1][0], half[1][1]}, p[st], o[t]);
        }
    }
  }
};

// A run of keys of one kv head, prefix or own, and the DMA of tiles of it.
template <int DT, int D>
struct Keys {
  using T = Tile<DT, D>;
  static constexpr int RPD = 1024 / T::RB;  // rows of one DMA instruction
  const char *k, *v;     // row 0 of the head
  int64_t stride;        // bytes a row
  int n;                 // keys that there are
  const int32_t* table;  // pages, or null
  int shift, npages;
  int held = -1;         // pages held .. held + 63 of the table lie in `page`, one a lane: the loop over
  int page = 0;          // the blocks then loads nothing that the compiler would wait for
  bool none = false;     // a page that is none was met

  // Byte offsets of the rows that this wave's share (of WAVES) of KEYS keys from j0 on reads.
  template <int KEYS, int WAVES>
  __device__ __forceinline__ void rows(int j0, int wave, int64_t (&off)[KEYS / RPD / WAVES]) {
    constexpr int N = KEYS / RPD / WAVES;
    static_assert(N * RPD * WAVES == KEYS, "whole DMA instructions");
    const int lane = threadIdx.x & 63, r = lane / T::CPR;
    if (table) {
      const int p0 = j0 >> shift, p1 = (j0 + KEYS - 1 < n ? j0 + KEYS - 1 : n - 1) >> shift;
      if (held < 0 || p1 >= held + 64) {
        held = p0;
        const int last = (n - 1) >> shift;
        page = table[p0 + lane < last ? p0 + lane : last];
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        int j = j0 + (i * WAVES + wave) * RPD + r;
        j = j < n ? j : n - 1;
        int pg = __builtin_amdgcn_ds_bpermute(((j >> shift) - held) << 2, page);
        if (pg < 0 || pg >= npages) {
          none = true;
          pg = 0;
        }
        off[i] = (((int64_t)pg << shift) + (j & ((1 << shift) - 1))) * stride;
      }
    } else if (j0 + KEYS <= n) {
      const int64_t mine = r * stride;
#pragma unroll
      for (int i = 0; i < N; ++i) off[i] = mine + (int64_t)(j0 + (i * WAVES + wave) * RPD) * stride;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int j = j0 + (i * WAVES + wave) * RPD + r;
        off[i] = (int64_t)(j < n ? j : n - 1) * stride;
      }
    }
  }
  // the DMA of those rows of K or V into tiles at dst
  template <bool V, int N, int WAVES>
  __device__ __forceinline__ void load(const int64_t (&off)[N], KU_LDS unsigned char* dst, int wave, int dim) const {
    const int lane = threadIdx.x & 63, last = dim * T::ES / 16 - 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int blk = i * WAVES + wave, r = blk * RPD + lane / T::CPR;
      int c = (lane % T::CPR) ^ (V ? T::vswz(r) : T::kswz(r));
      c = c < last ? c : last;  // features past head_dim meet zeros of Q, or are not stored
      lds_dma16_g((V ? v : k) + off[i] + c * 16, (KU_LDS void*)(dst + blk * 1024));
    }
  }
};

template <int DT, int D>
__device__ __forceinline__ Keys<DT, D> prefix_keys(const SdpaDev& a, int kvh) {
  using E = typename SdpaElem<DT>::T;
  return {reinterpret_cast<const char*>(static_cast<const E*>(a.pk) + kvh * a.phead),
          reinterpret_cast<const char*>(static_cast<const E*>(a.pv) + kvh * a.phead), a.prow * (int)sizeof(E), a.prefix, nullptr, 0, 0};
}
template <int DT, int D>
__device__ __forceinline__ Keys<DT, D> own_keys(const SdpaDev& a, int b, int kvh) {
  using E = typename SdpaElem<DT>::T;
  const int64_t base = kvh * a.head + (a.page_shift < 0 ? b * a.seq_rows * a.row : 0);
  return {reinterpret_cast<const char*>(static_cast<const E*>(a.k) + base), reinterpret_cast<const char*>(static_cast<const E*>(a.v) + base),
          a.row * (int)sizeof(E), sdpa_len(a, b), a.page_shift < 0 ? nullptr : a.pages + b * a.per_seq,
          a.page_shift < 0 ? 0 : a.page_shift, a.npages};
}

// blocks [first, last) of n that split i of s takes
__device__ __forceinline__ void split_range(int n, int i, int s, int& first, int& last) {
  first = (int)((int64_t)n * i / s);
  last = (int)((int64_t)n * (i + 1) / s);
}

// Item i of n in an order that gives each XCD (work-groups go to them in turn) a run of items: the row
// tiles of one split of keys, which come one after another, then read it from one L2.
__device__ __forceinline__ int xcd_order(int i, int n) {
  const int x = i & 7, q = n >> 3, r = n & 7;
  return x * q + (x < r ? x : r) + (i >> 3);
}

// where a query's row lies
struct RowAt {
  int b, t, h;
  __device__ __forceinline__ RowAt(const SdpaDev& a, int64_t row) {
    const int64_t tok = row / a.q_heads;
    b = (int)(tok / a.q_len), t = (int)(tok % a.q_len), h = (int)(row % a.q_heads);
  }
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

template <int DT, int D>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) sdpa_tiles_k(SdpaArgs g) {
  using T = Tile<DT, D>;
  using E = typename SdpaElem<DT>::T;
  __shared__ __attribute__((aligned(1024))) unsigned char lds_raw[T::LDS];
  __shared__ float2 wave_ml[4][32];
  __shared__ uint32_t redo_rows, met_none;
  KU_LDS unsigned char* lds = (KU_LDS unsigned char*)lds_raw;
  const SdpaDev& a = g.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = lane >> 5;
  const float c = a.scale * LOG2E;
  int id = blockIdx.x;
  const bool second = id >= g.p.part[0].units;
  const SdpaPlan::Part& part = g.p.part[second];
  id = second ? xcd_order(id - g.p.part[0].units, part.units) : xcd_order(id, part.units);
  const bool pooled = !g.p.joint && !second, shared = part.shared;

  // the work-group's (sequence,) kv head, row tile and split of the keys
  const int tile = id % part.tiles;
  id /= part.tiles;
  const int split = id % part.splits;
  id /= part.splits;
  const int kvh = id % a.kv_heads, b = id / a.kv_heads;
  const int per_seq = a.q_len * a.group, nrows = pooled ? a.batch * per_seq : per_seq;
  const int row0 = tile * (shared ? 128 : 32) + (shared ? wave * 32 : 0);  // of this wave
  const int own_len = pooled ? 0 : sdpa_len(a, b);
  // (b, t, h) index of row r of the tile's kv head (and sequence)
  auto row_of = [&](int r) {
    const int seq = pooled ? r / per_seq : b, in = pooled ? r % per_seq : r;
    return ((int64_t)seq * a.q_len + in / a.group) * a.q_heads + kvh * a.group + in % a.group;
  };
  Rows<DT, D> R;
  int64_t row = -1;
  const E* qrow = nullptr;
  R.limit = 0;
  if (row0 + (lane & 31) < nrows) {
    row = row_of(row0 + (lane & 31));
    const RowAt at(a, row);
    qrow = static_cast<const E*>(a.q) + at.b * a.qb + at.t * a.qt + at.h * a.qh;
    R.limit = own_len - (a.q_len - 1 - at.t);
  }
  R.load_q(qrow, a.dim);
  R.clear();
  if (threadIdx.x == 0) redo_rows = met_none = 0;
  __syncthreads();

  // the tile's blocks: those of the prefix, then those of the sequence's own keys that its last row sees
  const int bk = shared ? 32 * T::SB : 32;
  int own_n = 0;
  if (own_len) {
    const int last_row = std::min((tile + 1) * (shared ? 128 : 32), nrows) - 1;
    own_n = std::max(0, own_len - (a.q_len - 1 - last_row / a.group));
  }
  const int np = second ? 0 : (a.prefix + bk - 1) / bk, no = (own_n + bk - 1) / bk;
  int first, last;
  split_range(np + no, split, part.splits, first, last);
  Keys<DT, D> P = prefix_keys<DT, D>(a, kvh), O = own_keys<DT, D>(a, b, kvh);
  O.n = own_len;

  if (shared) {
    // Four waves of 32 rows over blocks of BK keys; the next block's DMA runs under this one's products.
    constexpr int BK = 32 * T::SB, TB = T::SB * T::KT, N = BK / Keys<DT, D>::RPD / 4;
    auto kbuf = [&](int i) { return lds + i * TB; };
    auto vbuf = [&](int i) { return lds + (2 + i) * TB; };
    auto fetch = [&](int blk) {
      int64_t off[N];
      if (blk < np) {
        P.template rows<BK, 4>(blk * BK, wave, off);
        P.template load<false, N, 4>(off, kbuf(blk & 1), wave, a.dim);
        P.template load<true, N, 4>(off, vbuf(blk & 1), wave, a.dim);
      } else {
        O.template rows<BK, 4>((blk - np) * BK, wave, off);
        O.template load<false, N, 4>(off, kbuf(blk & 1), wave, a.dim);
        O.template load<true, N, 4>(off, vbuf(blk & 1), wave, a.dim);
      }
    };
    if (first < last) fetch(first);
    for (int blk = first; blk < last; ++blk) {
      vm_wait<0>();
      __syncthreads();
      if (blk + 1 < last) fetch(blk + 1);
      const bool pre = blk < np;
      const int j0 = (pre ? blk : blk - np) * BK;
      f32x16 s[T::SB];
#pragma unroll
      for (int t = 0; t < T::SB; ++t) s[t] = R.scores(kbuf(blk & 1) + t * T::KT);
      const int lim = pre ? a.prefix : R.limit;
      if (!pre || j0 + BK > a.prefix)
#pragma unroll
        for (int t = 0; t < T::SB; ++t) R.mask(s[t], lim - j0 - 32 * t);
      R.rescale(s, c);
#pragma unroll
      for (int t = 0; t < T::SB; ++t) R.weigh(s[t], c, vbuf(blk & 1) + t * T::KT);
    }
  } else {
    // The waves take blocks of 32 keys in turn, each by itself: K of its next block is fetched once this
    // one's scores are done, V once its products are, so either is on its way while the other is used.
    constexpr int N = 32 / Keys<DT, D>::RPD;
    KU_LDS unsigned char *K = lds + wave * 2 * T::KT, *V = K + T::KT;
    int64_t off[N];
    auto rows = [&](int blk) {
      if (blk < np)
        P.template rows<32, 1>(blk * 32, 0, off);
      else
        O.template rows<32, 1>((blk - np) * 32, 0, off);
    };
    auto fetch_k = [&](int blk) { blk < np ? P.template load<false, N, 1>(off, K, 0, a.dim) : O.template load<false, N, 1>(off, K, 0, a.dim); };
    auto fetch_v = [&](int blk) { blk < np ? P.template load<true, N, 1>(off, V, 0, a.dim) : O.template load<true, N, 1>(off, V, 0, a.dim); };
    int blk = first + wave;
    if (blk < last) {
      rows(blk);
      fetch_k(blk);
      fetch_v(blk);
    }
    for (; blk < last; blk += 4) {
      const bool pre = blk < np, more = blk + 4 < last;
      const int j0 = (pre ? blk : blk - np) * 32;
      vm_wait<N>();  // K is there, V on its way
      asm volatile("" ::: "memory");
      f32x16 s[1];
      s[0] = R.scores(K);
      if (more) {
        rows(blk + 4);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // K has been read
        fetch_k(blk + 4);
      }
      const int lim = pre ? a.prefix : R.limit;
      if (!pre || j0 + 32 > a.prefix) R.mask(s[0], lim - j0);
      R.rescale(s, c);
      if (more)
        vm_wait<N>();
      else
        vm_wait<0>();
      asm volatile("" ::: "memory");
      R.weigh(s[0], c, V);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if (more) fetch_v(blk + 4);
    }
  }

  // ---- the results ----
  const int slots = g.p.slots, slot = second ? g.p.part[0].splits + split : split;
  R.l += other_half(R.l);
  if (__builtin_amdgcn_ballot_w64(O.none) != 0 && lane == 0) atomicOr(&met_none, 1u);
  uint32_t redo = 0;  // rows of this wave that are done again
  __syncthreads();
  if (met_none) R.l = NAN;
  if (shared) {
    if (slots > 1) {
      if (row >= 0) {
        float* o = g.po + (row * slots + slot) * D;
#pragma unroll
        for (int t = 0; t < T::DTL; ++t)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            *reinterpret_cast<f32x4*>(o + 32 * t + 8 * v + 4 * h) =
                f32x4{R.o[t][4 * v], R.o[t][4 * v + 1], R.o[t][4 * v + 2], R.o[t][4 * v + 3]};
        if (h == 0) g.ml[row * slots + slot] = make_float2(R.m, R.l);
      }
    } else {
      float z = R.l * 0.f;
#pragma unroll
      for (int t = 0; t < T::DTL; ++t)
#pragma unroll
        for (int v = 0; v < 16; ++v) z = fmaf(R.o[t][v], 0.f, z);
      z += other_half(z);
      const bool bad = row >= 0 && (!(z == 0.f) || R.l == 0.f);
      if (row >= 0 && !bad) {
        const RowAt at(a, row);
        const float inv = 1.f / R.l;
#pragma unroll
        for (int t = 0; t < T::DTL; ++t)
#pragma unroll
          for (int v = 0; v < 4; ++v)
            write_out<DT>(a, at, 32 * t + 8 * v + 4 * h,
                          f32x4{R.o[t][4 * v] * inv, R.o[t][4 * v + 1] * inv, R.o[t][4 * v + 2] * inv, R.o[t][4 * v + 3] * inv});
        if (a.lse && h == 0) a.lse[row] = (R.m + __builtin_amdgcn_logf(R.l)) * LN2;
      }
      redo = (uint32_t)__builtin_amdgcn_ballot_w64(bad && h == 0);
    }
  } else {
    // the waves' results of the same 32 rows are brought to one maximum and added through LDS
    if (h == 0) wave_ml[wave][lane] = make_float2(R.m, R.l);
    __syncthreads();
    float m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, wave_ml[w][lane & 31].x);
    const float from = m == -INFINITY ? 0.f : m;  // nothing seen
#pragma unroll
    for (int w = 0; w < 4; ++w) l = fmaf(__builtin_amdgcn_exp2f(wave_ml[w][lane & 31].x - from), wave_ml[w][lane & 31].y, l);
    const float mine = __builtin_amdgcn_exp2f(R.m - from);
    if (met_none) l = NAN;
    constexpr int CH = D / 4;  // 16-byte chunks of a row, swizzled by the row
    if (row >= 0) {
      KU_LDS unsigned char* o = lds + wave * 32 * D * 4 + (lane & 31) * D * 4;
#pragma unroll
      for (int t = 0; t < T::DTL; ++t)
#pragma unroll
        for (int v = 0; v < 4; ++v)
          *(KU_LDS f32x4*)(o + (((8 * t + 2 * v + h) ^ (lane & (CH - 1) & 31)) << 4)) =
              f32x4{R.o[t][4 * v] * mine, R.o[t][4 * v + 1] * mine, R.o[t][4 * v + 2] * mine, R.o[t][4 * v + 3] * mine};
    }
    __syncthreads();
    if (wave == 0 && h == 0) wave_ml[0][lane] = make_float2(m, l);
    __syncthreads();
    const int rows = std::min(32, nrows - row0);
    for (int i = threadIdx.x; i < rows * CH; i += 256) {
      const int r = i / CH, ch = i % CH;
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) o += *(const KU_LDS f32x4*)(lds + w * 32 * D * 4 + r * D * 4 + ((ch ^ (r & (CH - 1) & 31)) << 4));
      const float2 x = wave_ml[0][r];
      const int64_t at = row_of(row0 + r);
      if (slots > 1) {
        *reinterpret_cast<f32x4*>(g.po + (at * slots + slot) * D + ch * 4) = o;
        if (ch == 0) g.ml[at * slots + slot] = x;
      } else {
        if (bad_sum(x.y) || x.y == 0.f || bad_sum(o[0]) || bad_sum(o[1]) || bad_sum(o[2]) || bad_sum(o[3])) atomicOr(&redo_rows, 1u << r);
        const float inv = 1.f / x.y;
        write_out<DT>(a, RowAt(a, at), ch * 4, o * inv);
        if (ch == 0 && a.lse) a.lse[at] = (x.x + __builtin_amdgcn_logf(x.y)) * LN2;
      }
    }
    if (slots == 1) {
      __syncthreads();  // also orders the outputs written so far before those written again
      redo = __builtin_amdgcn_readfirstlane(redo_rows) & (0x11111111u << wave);
    }
  }
  while (redo) {
    const int i = __builtin_ctz(redo);
    redo &= redo - 1;
    const RowAt at(a, row_of(row0 + i));
    sdpa_one<DT>(a, at.b, at.t, at.h, reinterpret_cast<float*>(lds_raw + wave * 2 * T::KT));
  }
}

// Joins the partial results of a row, one wave a row: the slots' weights in the lanes, then eight slots'
// outputs at a time.
template <int DT, int D>
__global__ void __launch_bounds__(256) sdpa_join_k(SdpaArgs g) {
  __shared__ float lds[4][kSdpaMaxDim];
  const SdpaDev& a = g.a;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t row = (int64_t)blockIdx.x * 4 + wave;
  if (row >= (int64_t)a.batch * a.q_len * a.q_heads) return;
  const int n = g.p.slots;
  const float2* ml = g.ml + row * n;
  constexpr int L = D / 4, S = 64 / L;  // lanes a slot's output takes, slots side by side
  const int ch = lane % L, sub = lane / L;
  float m = -INFINITY;
  for (int i = lane; i < n; i += 64) m = fmaxf(m, ml[i].x);
#pragma unroll
  for (int o = 32; o; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  const float from = m == -INFINITY ? 0.f : m;
  float l = 0.f;
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  const f32x4* po = reinterpret_cast<const f32x4*>(g.po + row * n * D) + ch;
  for (int i0 = 0; i0 < n; i0 += 8 * S) {
    f32x4 x[8];
    float2 y[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int i = i0 + j * S + sub;
      x[j] = f32x4{0.f, 0.f, 0.f, 0.f};
      y[j] = make_float2(-INFINITY, 0.f);
      if (i < n) {
        x[j] = po[(int64_t)i * L];
        y[j] = ml[i];
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float w = __builtin_amdgcn_exp2f(y[j].x - from);  // 0 for a slot that saw nothing
      l = fmaf(w, y[j].y, l);
      acc += x[j] * w;
    }
  }
  // the slots side by side are added in one order in every lane
#pragma unroll
  for (int o = L; o < 64; o <<= 1) {
    l += __shfl_xor(l, o, 64);
#pragma unroll
    for (int k = 0; k < 4; ++k) acc[k] += __shfl_xor(acc[k], o, 64);
  }
  const RowAt at(a, row);
  if (__builtin_amdgcn_ballot_w64(bad_sum(l) || bad_sum(acc[0]) || bad_sum(acc[1]) || bad_sum(acc[2]) || bad_sum(acc[3])) != 0 || l == 0.f) {
    sdpa_one<DT>(a, at.b, at.t, at.h, lds[wave]);
    return;
  }
  if (sub == 0) write_out<DT>(a, at, ch * 4, acc * (1.f / l));
  if (a.lse && lane == 0) a.lse[row] = (m + __builtin_amdgcn_logf(l)) * LN2;
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

// Whether one sequence's rows fill tiles of 128 well enough to walk the prefix by themselves; where they
// do not, the sequences' rows share tiles over the prefix.
SdpaPlan make_plan(const KuHipSdpaPrefixArgs& a) {
  SdpaPlan p;
  const int64_t per_seq = (int64_t)(a.q_len * (a.q_heads / a.kv_heads)), kv = (int64_t)a.kv_heads, nb = (int64_t)a.batch;
  const bool f32 = a.dtype == KU_F32;
  const int64_t bk_shared = f32 ? 32 : 64;
  const int64_t full = (per_seq + 127) / 128 * 128;
  p.joint = full * 4 <= per_seq * 5;
  auto cut = [&](SdpaPlan::Part& part, int64_t rows, int64_t items, int64_t keys) {
    if (keys == 0 || items == 0 || rows == 0) return;
    part.shared = rows > 32;
    part.tiles = (int)((rows + (part.shared ? 127 : 31)) / (part.shared ? 128 : 32));
    const int64_t blocks = (keys + (part.shared ? bk_shared : 128) - 1) / (part.shared ? bk_shared : 128);
    const int64_t want = 2 * (int64_t)cu_count();
    part.splits = (int)std::max<int64_t>(1, std::min<int64_t>({want / (items * part.tiles), (blocks + 1) / 2, 256}));
    part.units = (int)(items * part.tiles * part.splits);
  };
  if (p.joint) {
    cut(p.part[0], per_seq, nb * kv, (int64_t)(a.prefix_len + a.own_max));
  } else {
    cut(p.part[0], nb * per_seq, kv, (int64_t)a.prefix_len);
    cut(p.part[1], per_seq, nb * kv, (int64_t)a.own_max);
  }
  p.slots = p.part[0].splits + p.part[1].splits;
  return p;
}

int padded_dim(size_t d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }

template <int DT, int D>
void launch_d(const SdpaArgs& g, hipStream_t s) {
  const unsigned groups = (unsigned)(g.p.part[0].units + g.p.part[1].units);
  if (groups) hipLaunchKernelGGL((sdpa_tiles_k<DT, D>), dim3(groups), dim3(256), 0, s, g);
  const int64_t rows = (int64_t)g.a.batch * g.a.q_len * g.a.q_heads;
  if (g.p.slots != 1) hipLaunchKernelGGL((sdpa_join_k<DT, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, s, g);
}
template <int DT>
void launch_t(const SdpaArgs& g, int d, hipStream_t s) {
  switch (d) {
    case 32: launch_d<DT, 32>(g, s); break;
    case 64: launch_d<DT, 64>(g, s); break;
    default: launch_d<DT, 128>(g, s); break;
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
              (__int128)a.batch * a.q_len * a.q_heads <= (__int128)most,
          "more than 2^31 - 1 queries");
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
  const int64_t nq = span_of(d, {{a.batch, a.q_batch_stride}, {a.q_len, a.q_token_stride}, {a.q_heads, a.q_head_stride}}, "q");
  const int64_t no = written_span(
      d, {{a.batch, a.out_batch_stride}, {a.q_len, a.out_token_stride}, {a.q_heads, a.out_head_stride}}, "out");
  if (a.batch) {
    pointers16({a.q, a.out});
    require(!overlap(a.q, nq * w, a.out, no * w), "out overlaps q");
  }
  if (a.prefix_len) {
    pointers16({a.prefix_k, a.prefix_v});
    strides16({a.prefix_row_stride, a.prefix_head_stride});
    span_of(d, {{a.prefix_len, a.prefix_row_stride}, {a.kv_heads, a.prefix_head_stride}}, "prefix_k");
  }
  if (a.own_max) {
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
    } else if (a.batch) {
      require(a.batch == 1 || a.own_seq_rows >= a.own_max, "own_seq_rows is less than own_max");
      require(a.own_seq_rows <= ((size_t)1 << 40) &&
                  (__int128)(a.batch - 1) * a.own_seq_rows + a.own_max <= (__int128)a.own_rows,
              "own_rows does not hold own_max keys of every sequence");
    }
  }
}

size_t sdpa_prefix_scratch_bytes(const KuHipSdpaPrefixArgs& a) {
  const SdpaPlan p = make_plan(a);
  if (a.batch == 0 || p.slots <= 1) return 0;
  return a.batch * a.q_len * a.q_heads * (size_t)p.slots * (padded_dim(a.head_dim) * sizeof(float) + sizeof(float2));
}

void launch_sdpa_prefix(const KuHipSdpaPrefixArgs& a, void* scratch, hipStream_t s) {
  if (a.batch == 0) return;
  SdpaArgs g;
  g.a = device_args(a);
  g.p = make_plan(a);
  const int d = padded_dim(a.head_dim);
  g.po = static_cast<float*>(scratch);
  g.ml = reinterpret_cast<float2*>(g.po + a.batch * a.q_len * a.q_heads * (size_t)g.p.slots * d);
  switch (a.dtype) {
    case KU_BF16: launch_t<GT_BF16>(g, d, s); break;
    case KU_F16: launch_t<GT_F16>(g, d, s); break;
    default: launch_t<GT_F32>(g, d, s); break;
  }
  check_launch();
}

}  // namespace ku::hipbk
