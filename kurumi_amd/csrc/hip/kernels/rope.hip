// Rotary positions with the store into a key / value cache (ku_hip_rope).
//
// Pair i of a head of token t turns by a = position_t * f_i:
//   y_lo = s (x_lo cos a - x_hi sin a),  y_hi = s (x_hi cos a + x_lo sin a)
// with (lo, hi) = (i, i + rot/2) or (2i, 2i + 1); the features from rot on, and v, are copied.
//
// The angle is formed in f64 as a number of turns, position * (f_i / 2 pi), of which only the
// fraction is kept: in f32 a position of 10^5 would leave the fastest pair 2^-8 of a turn. The
// fraction is then exact enough in f32 for sine and cosine to half a step of f32.
#include <hip/hip_runtime.h>

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
  int q_heads, kv_heads, head_dim, rot;
  float scale;
  double turns[kMaxPairs];  // f_i / 2 pi, negated for the inverse
};

template <int DT, class T>
__device__ __forceinline__ float ld(const T* p) { return load_elem<DT, T, float>(*p); }

// One work-group per (token, head): heads are q's, then k's, then v's.
template <int DT, class T, bool HALF>
__global__ void __launch_bounds__(64) rope_k(RopeDev a) {
  const int64_t t = blockIdx.x;
  int h = blockIdx.y;
  const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
  const RopeSide& sd = is_q ? a.q : is_v ? a.v : a.k;
  h = is_q ? h : is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads;
  if (!sd.in) return;
  int64_t row = t;
  if (!is_q) {
    if (a.rows) row = a.rows[t];
    if (row < 0 || row >= a.out_rows) return;
  }
  const T* x = static_cast<const T*>(sd.in) + t * sd.in_token + h * sd.in_head;
  T* y = static_cast<T*>(sd.out) + row * sd.out_row + h * sd.out_head;
  const int rot = is_v ? 0 : a.rot;
  const double p = rot ? (double)a.positions[t] : 0.0;
  for (int i = threadIdx.x; i < rot / 2; i += 64) {
    const double turns = p * a.turns[i];
    float sn, cs;
    sincospif(2.f * (float)(turns - rint(turns)), &sn, &cs);
    sn *= a.scale;
    cs *= a.scale;
    const int lo = HALF ? i : 2 * i, hi = HALF ? i + rot / 2 : 2 * i + 1;
    const float xl = ld<DT>(x + lo), xh = ld<DT>(x + hi);
    y[lo] = store_elem<DT, T>(fmaf(xl, cs, -xh * sn));
    y[hi] = store_elem<DT, T>(fmaf(xh, cs, xl * sn));
  }
  for (int i = rot + threadIdx.x; i < a.head_dim; i += 64) y[i] = x[i];
}

template <int DT, class T>
void launch_t(const RopeDev& d, bool half, hipStream_t s) {
  const dim3 grid((unsigned)d.tokens, (unsigned)(d.q_heads + 2 * d.kv_heads));
  if (half)
    hipLaunchKernelGGL((rope_k<DT, T, true>), grid, dim3(64), 0, s, d);
  else
    hipLaunchKernelGGL((rope_k<DT, T, false>), grid, dim3(64), 0, s, d);
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
  require((a.q != nullptr) == (a.q_out != nullptr) && (a.k != nullptr) == (a.k_out != nullptr) &&
              (a.v != nullptr) == (a.v_out != nullptr),
          "an input without its output, or an output without its input");
  require(a.q || a.k || a.v, "nothing to do: q, k and v are all null");
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
  auto side = [&](const void* in, int64_t it, int64_t ih, void* out, int64_t orow, int64_t oh, size_t heads,
                  size_t out_rows, bool by_row, const char* what) {
    if (!in) return;
    require(aligned_to(in, (size_t)w) && aligned_to(out, (size_t)w), "pointers must be aligned to their elements");
    const int64_t ni = span_of(d, {{a.tokens, it}, {heads, ih}}, what) * w;
    const int64_t no = written_span(d, {{out_rows, orow}, {heads, oh}}, what) * w;
    if (a.tokens && overlap(in, ni, out, no))
      require(in == out && it == orow && ih == oh && !by_row,
              "an output overlaps its input without being the same (for k and v: the same, and no rows)");
  };
  side(a.q, a.q_token_stride, a.q_head_stride, a.q_out, a.q_out_token_stride, a.q_out_head_stride, a.q_heads, a.tokens,
       false, "q or q_out");
  side(a.k, a.k_token_stride, a.k_head_stride, a.k_out, a.k_out_row_stride, a.k_out_head_stride, a.kv_heads, a.out_rows,
       a.rows != nullptr, "k or k_out");
  side(a.v, a.v_token_stride, a.v_head_stride, a.v_out, a.v_out_row_stride, a.v_out_head_stride, a.kv_heads, a.out_rows,
       a.rows != nullptr, "v or v_out");
}

void launch_rope(const KuHipRopeArgs& a, hipStream_t s) {
  if (a.tokens == 0) return;
  RopeDev d;
  d.q = {a.q, a.q_out, a.q_token_stride, a.q_head_stride, a.q_out_token_stride, a.q_out_head_stride};
  d.k = {a.k, a.k_out, a.k_token_stride, a.k_head_stride, a.k_out_row_stride, a.k_out_head_stride};
  d.v = {a.v, a.v_out, a.v_token_stride, a.v_head_stride, a.v_out_row_stride, a.v_out_head_stride};
  d.positions = a.positions;
  d.rows = a.rows;
  d.tokens = (int64_t)a.tokens;
  d.out_rows = (int64_t)a.out_rows;
  d.q_heads = a.q ? (int)a.q_heads : 0;
  d.kv_heads = a.k || a.v ? (int)a.kv_heads : 0;
  d.head_dim = (int)a.head_dim;
  d.rot = a.q || a.k ? (int)a.rot_dim : 0;
  d.scale = a.scale;
  for (int i = 0; i < d.rot / 2; ++i) d.turns[i] = (a.inverse ? -a.freqs[i] : a.freqs[i]) / 6.283185307179586476925;
  const bool half = a.layout == KU_ROPE_HALF;
  switch (a.dtype) {
    case KU_BF16: launch_t<GT_BF16, uint16_t>(d, half, s); break;
    case KU_F16: launch_t<GT_F16, uint16_t>(d, half, s); break;
    default: launch_t<GT_F32, float>(d, half, s); break;
  }
  check_launch();
}

}  // namespace ku::hipbk
