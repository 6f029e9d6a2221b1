// Arithmetic that the attentions over a paged cache share: matrix products of 16 bytes a lane, and what a softmax's
// probabilities become in 16 bits.
#pragma once

#include "tmh_f8.h"

namespace tmh {

constexpr float kNone = -__builtin_inff();
typedef uint32_t uint2_t __attribute__((ext_vector_type(2)));

__device__ __forceinline__ uint32_t scan64(uint32_t v) {  // the sum over the lanes up to this one
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t up = __shfl_up(v, o);
    if ((threadIdx.x & 63) >= o) v += up;
  }
  return v;
}

// (By value: __builtin_bit_cast of a vector's element, an lvalue, reads element 0.)
__device__ __forceinline__ float as_float(uint32_t v) { return __builtin_bit_cast(float, v); }

template <int DT>
struct Lane16 {  // 16 bytes of a lane as MFMA operands
  typedef _Float16 vec __attribute__((ext_vector_type(8)));
};
template <>
struct Lane16<DT_BF16> {
  typedef __bf16 vec __attribute__((ext_vector_type(8)));
};

template <int DT>
__device__ __forceinline__ float4_t mfma16(uint4_t a, uint4_t b, float4_t c) {
  typedef typename Lane16<DT>::vec vec;
  if constexpr (DT == DT_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(vec, a), __builtin_bit_cast(vec, b), c, 0, 0, 0);
}

// Two probabilities as the sums of two 16-bit parts each: cut off, and the rest, rounded. What is cut is a little less
// than the probability, so that the rest is not 0 beside a first part that is not, and an infinity in V stays what
// it is in both products (f16: of probabilities of 2^-23, 2^-38 of the largest, and more; others give NaN with it).
// A probability of 0 gives zeros: a token without weight has no part in the answer, whatever its value.
template <int DT>
__device__ __forceinline__ uint2 split2(float a, float b) {
  constexpr float less = 1.f - 0x1p-20f;
  if constexpr (DT == DT_F16) {
    const auto h = __builtin_amdgcn_cvt_pkrtz(fmaf(a, less, -0x1p-24f), fmaf(b, less, -0x1p-24f));
    return make_uint2(__builtin_bit_cast(uint32_t, h), pack2<DT>(a - static_cast<float>(h[0]), b - static_cast<float>(h[1])));
  } else {
    const uint32_t hi = __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b * less), __builtin_bit_cast(uint32_t, a * less), 0x07060302u);
    return make_uint2(hi, pack2<DT>(a - __builtin_bit_cast(float, hi << 16), b - __builtin_bit_cast(float, hi & 0xFFFF0000u)));
  }
}

// The maximum (sum) over the four lanes of one column of an MFMA tile, in all of them.
__device__ __forceinline__ float column_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float column_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

}  // namespace tmh
