// Attention of a batch that shares its first keys (ku_hip_sdpa_prefix).
//
//   out[b, t, h] = sum_j softmax_j(scale q[b, t, h] . K_j) V_j
// over the shared prefix and the keys of sequence b that query t sees.
#include <hip/hip_runtime.h>

#include <cmath>

#include "decode.h"
#include "sdpa_prefix.h"

namespace ku::hipbk {

namespace {

template <int DT>
__global__ void __launch_bounds__(64) sdpa_rows_k(SdpaDev a) {
  __shared__ float lds[kSdpaMaxDim];
  const int64_t i = blockIdx.x;
  sdpa_one<DT>(a, (int)(i / a.q_heads / a.q_len), (int)(i / a.q_heads % a.q_len), (int)(i % a.q_heads), lds);
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

size_t sdpa_prefix_scratch_bytes(const KuHipSdpaPrefixArgs&) { return 0; }

void launch_sdpa_prefix(const KuHipSdpaPrefixArgs& a, void*, hipStream_t s) {
  if (a.batch == 0) return;
  const SdpaDev d = device_args(a);
  const dim3 grid((unsigned)(a.batch * a.q_len * a.q_heads));
  switch (a.dtype) {
    case KU_BF16: hipLaunchKernelGGL((sdpa_rows_k<GT_BF16>), grid, dim3(64), 0, s, d); break;
    case KU_F16: hipLaunchKernelGGL((sdpa_rows_k<GT_F16>), grid, dim3(64), 0, s, d); break;
    default: hipLaunchKernelGGL((sdpa_rows_k<GT_F32>), grid, dim3(64), 0, s, d); break;
  }
  check_launch();
}

}  // namespace ku::hipbk
