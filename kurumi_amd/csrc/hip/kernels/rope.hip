// Rotary positions with the store into a key / value cache (ku_hip_rope).
//
// Pair i of a head of token t turns by a = position_t * f_i:
//   y_lo = s (x_lo cos a - x_hi sin a),  y_hi = s (x_hi cos a + x_lo sin a)
// with (lo, hi) = (i, i + rot/2) or (2i, 2i + 1); the features from rot on, and v, are copied.
//
// The angle is formed in f64 as a number of turns, position * (f_i / 2 pi), of which only the
// fraction is kept: in f32 a position of 10^5 would leave the fastest pair 2^-8 of a turn. The
// fraction, up to half a turn, is then rounded to f32, by 2^-26 of a turn at most: 2^-23.3 of a radian,
// by which sine and cosine are off (absolutely: of a sine near 0 it can be any part), beside their own two
// steps at most.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>

#include "decode.h"
#include "kernels.h"
#include "numeric.h"

namespace ku::hipbk {

namespace {

constexpr size_t kMaxPairs = 128;

struct RopeSide {
  const void* in = nullptr;
  void* out = nullptr;
  int64_t in_token = 0, in_head = 0, out_row = 0, out_head = 0;
};

struct RopeDev {
  RopeSide q, k, v;
  const int32_t* positions;
  const int32_t* rows;
  int64_t tokens, out_rows;
  uint32_t dim, rot;
  uint32_t turned, copied, v_units;    // units of a q or k head: turned ones, then copied ones; of a v head
  uint32_t q_units, qk_units, units;   // units a token: up to the last q head, k head, v head
  uint32_t block_tokens, block_units;  // what a work-group takes
  float scale;
  double turns[kMaxPairs];  // f_i / 2 pi, negated for the inverse
};

constexpr int kThreads = 256;

template <int N>
struct Bits;
template <> struct Bits<2> { using T = uint16_t; };
template <> struct Bits<4> { using T = uint32_t; };
template <> struct Bits<8> { using T = uint2; };
template <> struct Bits<16> { using T = uint4; };

// A unit is two vectors of V elements of one head: the low and the high features of V pairs (half
// layout: i and i + rot / 2; interleaved: next to each other), or up to two vectors that are copied.
// A work-group takes block_tokens tokens; it forms their angles once, in LDS, for all heads: a sine and
// cosine of a 64-bit angle for each unit of each head would take longer than moving the unit.
// Bound by memory: 8192 tokens of 48 heads of 128, bf16, with the store (201 MB in and out), 40.2 us, 5.0 TB/s,
// where a copy of 1 GiB reaches 5.06; 16 tokens 3.6 us, a launch.
template <int DT, class T, int V, bool HALF>
__global__ void __launch_bounds__(kThreads) rope_k(RopeDev a) {
  using W = typename Bits<V * (int)sizeof(T)>::T;
  extern __shared__ float2 table[];  // [block_tokens][rot / 2]: cosine, sine, times scale
  const int64_t t0 = (int64_t)blockIdx.x * a.block_tokens;
  const uint32_t nt = (uint32_t)(a.tokens - t0 < a.block_tokens ? a.tokens - t0 : a.block_tokens);
  const uint32_t first = blockIdx.y * a.block_units;
  const uint32_t per_token = a.units - first < a.block_units ? a.units - first : a.block_units;
  const uint32_t total = nt * per_token, half = a.rot / 2;

  struct Unit {
    W x[2];
    T* y;           // null: nothing to store
    uint32_t hi;    // element offset of the second vector; 0: there is none
    uint32_t pair;  // table entry of the first pair, or ~0 for a copy
  };
  auto load = [&](uint32_t u) {
    Unit r{};
    const uint32_t t = u / per_token;
    uint32_t i = u - t * per_token + first, head, unit, lo;
    const bool is_q = i < a.q_units, is_v = i >= a.qk_units;
    const RopeSide& sd = is_q ? a.q : is_v ? a.v : a.k;
    i -= is_q ? 0 : is_v ? a.qk_units : a.q_units;
    const uint32_t each = is_v ? a.v_units : a.turned + a.copied;
    head = i / each;
    unit = i - head * each;
    int64_t row = t0 + t;
    if (!is_q && a.rows) row = a.rows[t0 + t];
    if (!is_q && (row < 0 || row >= a.out_rows)) return r;
    if (!is_v && unit < a.turned) {
      r.pair = t * half + unit * V;
      lo = HALF ? unit * V : 2 * unit * V;
      r.hi = HALF ? half : V;
    } else {
      r.pair = ~0u;
      lo = is_v ? 2 * unit * V : a.rot + 2 * (unit - a.turned) * V;
      if (lo >= a.dim) return r;  // a head of an odd number of copied vectors next to turned ones
      r.hi = lo + V < a.dim ? V : 0;
    }
    const T* x = static_cast<const T*>(sd.in) + (t0 + t) * sd.in_token + head * sd.in_head + lo;
    r.y = static_cast<T*>(sd.out) + row * sd.out_row + head * sd.out_head + lo;
    r.x[0] = *reinterpret_cast<const W*>(x);
    if (r.hi) r.x[1] = *reinterpret_cast<const W*>(x + r.hi);
    return r;
  };
  auto store = [&](Unit& r) {
    if (!r.y) return;
    if (r.pair != ~0u) {
      T e[2][V];
      __builtin_memcpy(e, r.x, sizeof(e));
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float2 cs = table[r.pair + i];
        // half layout: pair i of the unit is (e[0][i], e[1][i]); interleaved: elements 2 i, 2 i + 1 of both
        T& lo = HALF ? e[0][i] : e[(2 * i) / V][(2 * i) % V];
        T& hi = HALF ? e[1][i] : e[(2 * i + 1) / V][(2 * i + 1) % V];
        const float xl = load_elem<DT, T, float>(lo), xh = load_elem<DT, T, float>(hi);
        lo = store_elem<DT, T>(fmaf(xl, cs.x, -xh * cs.y));
        hi = store_elem<DT, T>(fmaf(xh, cs.x, xl * cs.y));
      }
      __builtin_memcpy(r.x, e, sizeof(e));
    }
    *reinterpret_cast<W*>(r.y) = r.x[0];
    if (r.hi) *reinterpret_cast<W*>(r.y + r.hi) = r.x[1];
  };

  uint32_t u = threadIdx.x;
  Unit unit{};
  if (u < total) unit = load(u);
  // the first loads are on their way
  for (uint32_t i = threadIdx.x; i < nt * half; i += kThreads) {
    const uint32_t t = i / half;
    const double turns = (double)a.positions[t0 + t] * a.turns[i - t * half];
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    table[i] = make_float2(cs * a.scale, sn * a.scale);
  }
  __syncthreads();
  while (u < total) {
    store(unit);
    u += kThreads;
    if (u < total) unit = load(u);
  }
}

// How a call runs: V elements at a time, the kernel's arguments and its launch.
struct RopePlan {
  RopeDev d;
  int v = 1;
  dim3 grid;
  size_t lds = 0;
};

RopePlan make_plan(const KuHipRopeArgs& a) {
  RopePlan p;
  RopeDev& d = p.d;
  d.q = {a.q, a.q_out, a.q_token_stride, a.q_head_stride, a.q_out_token_stride, a.q_out_head_stride};
  d.k = {a.k, a.k_out, a.k_token_stride, a.k_head_stride, a.k_out_row_stride, a.k_out_head_stride};
  d.v = {a.v, a.v_out, a.v_token_stride, a.v_head_stride, a.v_out_row_stride, a.v_out_head_stride};
  d.positions = a.positions;
  d.rows = a.rows;
  d.tokens = (int64_t)a.tokens;
  d.out_rows = (int64_t)a.out_rows;
  d.dim = (uint32_t)a.head_dim;
  d.rot = a.q || a.k ? (uint32_t)a.rot_dim : 0;
  d.scale = a.scale;
  for (uint32_t i = 0; i < d.rot / 2; ++i) d.turns[i] = (a.inverse ? -a.freqs[i] : a.freqs[i]) / 6.283185307179586476925;
  const uint32_t qh = a.q ? (uint32_t)a.q_heads : 0, kh = a.k ? (uint32_t)a.kv_heads : 0, vh = a.v ? (uint32_t)a.kv_heads : 0;
  // as many bytes at a time, up to 16, as everything is made of
  const size_t width = a.dtype == KU_F32 ? 4 : 2;
  auto made_of = [&](int64_t v) {
    bool ok = d.dim % v == 0 && (d.rot / 2) % v == 0;
    for (const RopeSide* x : {&d.q, &d.k, &d.v})
      if (x->in)
        ok = ok && aligned_to(x->in, v * width) && aligned_to(x->out, v * width) && x->in_token % v == 0 && x->in_head % v == 0 &&
             x->out_row % v == 0 && x->out_head % v == 0;
    return ok;
  };
  p.v = 16 / (int)width;
  while (p.v > 1 && !made_of(p.v)) p.v /= 2;
  auto units = [&](uint32_t features) { return (features + 2 * p.v - 1) / (2 * p.v); };
  d.turned = d.rot / 2 / p.v;
  d.copied = units(d.dim - d.rot);
  d.v_units = units(d.dim);
  d.q_units = qh * (d.turned + d.copied);
  d.qk_units = d.q_units + kh * (d.turned + d.copied);
  d.units = d.qk_units + vh * d.v_units;
  // Work-groups of about two units a thread where that leaves enough of them (8192 tokens of 48 heads of
  // 128, bf16: 41.8 us; 47 with eight a thread, 56 with four of those in flight), of one where it does not:
  // a few tokens are spread over their heads.
  const int64_t all = d.tokens * (int64_t)d.units, want = all / (2 * kThreads) >= 4 * (int64_t)cu_count() ? 2 * kThreads : kThreads;
  d.block_tokens = (uint32_t)std::max<int64_t>(1, std::min<int64_t>({want / d.units, d.tokens, 64}));
  d.block_units = d.block_tokens > 1 ? d.units : (uint32_t)std::min<int64_t>(d.units, std::max<int64_t>(want, (d.units + 65534) / 65535));
  p.grid = dim3((unsigned)((d.tokens + d.block_tokens - 1) / d.block_tokens), (d.units + d.block_units - 1) / d.block_units);
  p.lds = d.block_tokens * (d.rot / 2) * sizeof(float2);
  return p;
}

template <int DT, class T, int V>
void launch_v(const RopePlan& p, bool half, hipStream_t s) {
  if (half)
    launch(rope_k<DT, T, V, true>, p.grid, kThreads, p.lds, s, p.d);
  else
    launch(rope_k<DT, T, V, false>, p.grid, kThreads, p.lds, s, p.d);
}
template <int DT, class T>
void launch_t(const RopePlan& p, bool half, hipStream_t s) {
  switch (p.v) {
    case 8:
      if constexpr (sizeof(T) == 2) launch_v<DT, T, 8>(p, half, s);
      break;
    case 4: launch_v<DT, T, 4>(p, half, s); break;
    case 2: launch_v<DT, T, 2>(p, half, s); break;
    default: launch_v<DT, T, 1>(p, half, s); break;
  }
}

}  // namespace

void rope_freqs(size_t rot_dim, double base, uint32_t scaling, double factor, double trained_len, double low,
                double high, double* out) {
  require(rot_dim % 2 == 0, "rot_dim must be even");
  require(out || rot_dim == 0, "null output pointer");
  require(base > 0 && std::isfinite(base), "base must be positive and finite");
  require(scaling <= KU_ROPE_BY_PARTS, "unknown scaling");
  if (scaling != KU_ROPE_UNSCALED) require(factor > 0 && std::isfinite(factor), "factor must be positive and finite");
  if (scaling == KU_ROPE_BY_PARTS) {
    require(trained_len > 0 && std::isfinite(trained_len), "trained_len must be positive and finite");
    require(std::isfinite(low) && std::isfinite(high) && low < high, "low must be less than high");
  }
  const double r = (double)rot_dim, two_pi = 6.283185307179586476925;
  if (scaling == KU_ROPE_BASE && rot_dim > 2) base *= std::pow(factor, r / (r - 2));
  for (size_t i = 0; i < rot_dim / 2; ++i) {
    double f = std::pow(base, -2.0 * (double)i / r);
    if (scaling == KU_ROPE_LINEAR) f /= factor;
    if (scaling == KU_ROPE_BY_PARTS) {
      const double keep = std::fmin(1.0, std::fmax(0.0, (trained_len * f / two_pi - low) / (high - low)));
      f = f * keep + f / factor * (1.0 - keep);
    }
    out[i] = f;
  }
}

void check_rope(const KuHipRopeArgs& a) {
  require(a.size == sizeof(KuHipRopeArgs), "size is not sizeof(KuHipRopeArgs)");
  const int64_t w = (int64_t)float_width(a.dtype, "dtype"), d = (int64_t)a.head_dim;
  require(a.layout <= KU_ROPE_INTERLEAVED, "unknown layout");
  require(a.head_dim >= 1 && a.head_dim <= 65536, "head_dim must be 1 to 65536");
  require(a.rot_dim % 2 == 0 && a.rot_dim <= a.head_dim && a.rot_dim <= 2 * kMaxPairs,
          "rot_dim must be even and at most head_dim and 256");
  require(std::isfinite(a.scale), "scale must be finite");
  require(a.tokens <= 0x7fffffff, "too many tokens");
  require(a.q_heads <= 16384 && a.kv_heads <= 16384, "too many heads");
  // of no tokens, an input may be null beside its output: the address of no elements
  require(a.tokens == 0 ||
              ((a.q != nullptr) == (a.q_out != nullptr) && (a.k != nullptr) == (a.k_out != nullptr) &&
               (a.v != nullptr) == (a.v_out != nullptr)),
          "an input without its output, or an output without its input");
  require(a.tokens == 0 || a.q || a.k || a.v, "nothing to do: q, k and v are all null");
  require(!a.q || a.q_heads > 0, "q without q_heads");
  require(!(a.k || a.v) || a.kv_heads > 0, "k or v without kv_heads");
  if (a.rot_dim && (a.q || a.k)) {
    require(a.freqs, "null freqs");
    for (size_t i = 0; i < a.rot_dim / 2; ++i) require(std::isfinite(a.freqs[i]), "freqs must be finite");
    require(a.positions || a.tokens == 0, "null positions");
  }
  require(aligned_to(a.positions, 4) && aligned_to(a.rows, 4), "positions and rows must be 4-byte aligned");
  if (a.k || a.v) {
    require(a.out_rows <= 0x7fffffff, "too many cache rows");
    if (!a.rows) require(a.out_rows >= a.tokens, "out_rows is less than tokens, and there are no rows");
  }
  Buffer ins[3], outs[3];
  int sides = 0;
  auto side = [&](const void* in, int64_t it, int64_t ih, void* out, int64_t orow, int64_t oh, size_t heads,
                  size_t out_rows, bool by_row, const char* what) {
    if (!in) return;
    require(aligned_to(in, (size_t)w) && aligned_to(out, (size_t)w), "pointers must be aligned to their elements");
    span_of(d, {{a.tokens, it}, {heads, ih}}, what);
    written_span(d, {{out_rows, orow}, {heads, oh}}, what);
    const Buffer x(in, d, {{a.tokens, it}, {heads, ih}}, w), y(out, d, {{by_row ? out_rows : a.tokens, orow}, {heads, oh}}, w);
    if (share(x, y))
      require(in == out && (a.tokens == 1 || it == orow) && (heads == 1 || ih == oh) && !by_row,
              "an output overlaps its input without being the same (for k and v: the same, and no rows)");
    ins[sides] = x;
    outs[sides++] = y;
  };
  side(a.q, a.q_token_stride, a.q_head_stride, a.q_out, a.q_out_token_stride, a.q_out_head_stride, a.q_heads, a.tokens,
       false, "q or q_out");
  side(a.k, a.k_token_stride, a.k_head_stride, a.k_out, a.k_out_row_stride, a.k_out_head_stride, a.kv_heads, a.out_rows,
       a.rows != nullptr, "k or k_out");
  side(a.v, a.v_token_stride, a.v_head_stride, a.v_out, a.v_out_row_stride, a.v_out_head_stride, a.kv_heads, a.out_rows,
       a.rows != nullptr, "v or v_out");
  if (a.tokens) {
    const dim3 grid = make_plan(a).grid;
    require((int64_t)grid.x * grid.y <= max_blocks(kThreads), "too many tokens for one launch");
    const Buffer numbers[] = {{a.positions, (int64_t)a.tokens, {}, 4}, {a.rows, (int64_t)a.tokens, {}, 4}};
    for (int i = 0; i < sides; ++i) {
      for (int j = 0; j < sides; ++j)
        require(i == j || !share(outs[i], ins[j]), "an output overlaps the input of another");
      for (int j = 0; j < i; ++j) require(!share(outs[i], outs[j]), "two outputs overlap");
      for (const Buffer& x : numbers) require(!share(outs[i], x), "an output overlaps positions or rows");
    }
  }
}

void launch_rope(const KuHipRopeArgs& a, hipStream_t s) {
  if (a.tokens == 0) return;
  const RopePlan p = make_plan(a);
  const bool half = a.layout == KU_ROPE_HALF;
  switch (a.dtype) {
    case KU_BF16: launch_t<GT_BF16, uint16_t>(p, half, s); break;
    case KU_F16: launch_t<GT_F16, uint16_t>(p, half, s); break;
    default: launch_t<GT_F32, float>(p, half, s); break;
  }
}

}  // namespace ku::hipbk
