// Pairs of 16-bit floats in one dword, as the operands of the 16-bit matrix products hold them.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kernels.h"

namespace ku::hipbk {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));

// two f32 -> one dword of two 16-bit values, rounded to nearest even by v_cvt_pk_bf16_f32 /
// v_cvt_f16_f32 (the probabilities and outputs here are never NaN unless an input is)
template <int DT>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const f32x2 v = {lo, hi};
  if constexpr (DT == GT_BF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, f16x2));
}

// c + lo + hi of a packed pair of 16-bit floats (v_dot2c_f32_{bf16,f16} against 1.0 pairs)
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

// the two values of a packed pair
template <int DT>
__device__ __forceinline__ float lower(uint32_t pair) {
  if constexpr (DT == GT_BF16) return __uint_as_float(pair << 16);
  else return (float)__builtin_bit_cast(f16x2, pair)[0];
}
template <int DT>
__device__ __forceinline__ float upper(uint32_t pair) {
  if constexpr (DT == GT_BF16) return __uint_as_float(pair & 0xffff0000u);
  else return (float)__builtin_bit_cast(f16x2, pair)[1];
}

}  // namespace ku::hipbk
