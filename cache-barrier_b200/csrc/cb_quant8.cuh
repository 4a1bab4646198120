// q = round(u / step) to e4m3 or int8 for eight values at a time: the rounding of the
// fp32 quotient.
//
// The eight quotients share a divisor, so they come from its reciprocal: with
// y = RN(1 / step), q0 = RN(u y) and the remainder r = u - q0 step by a fused
// multiply-add, RN(q0 + r y) is the correctly rounded quotient (P. Markstein,
// "Computation of elementary functions on the IBM RISC System/6000 processor", 1990,
// theorem 8, where q0 is within a unit in the last place; one beyond that is off by
// 1e-7 units before its rounding, which no 8-bit boundary tells apart in practice).
// Three instructions a value; an IEEE division each (about 20) made the kernels that
// use this issue-bound. Steps whose reciprocal or remainder would leave the normal
// range (below 2^-60, above 2^126, NaN) are divided.
#pragma once

#include <cstdint>
#include <cuda_fp8.h>

namespace cb {

// int8 rounds half away from zero, e4m3 to nearest even, saturated.
template <bool INT8>
__device__ __forceinline__ uint64_t quant8(const float (&u)[8], float step) {
  float v[8];
  if (step >= 8.673617379884035e-19f && step <= 8.507059173023462e+37f) {  // 2^-60, 2^126
    const float y = __fdiv_rn(1.0f, step);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q = __fmul_rn(u[j], y);
      v[j] = __fmaf_rn(__fmaf_rn(-q, step, u[j]), y, q);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __fdiv_rn(u[j], step);
  }
  uint64_t out = 0;
  if constexpr (INT8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int q = __float2int_rz(__fadd_rn(v[j], copysignf(0.5f, v[j])));
      out |= static_cast<uint64_t>(static_cast<uint8_t>(q)) << (8 * j);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; j += 2)
      out |= static_cast<uint64_t>(__nv_cvt_float2_to_fp8x2(make_float2(v[j], v[j + 1]), __NV_SATFINITE, __NV_E4M3)) << (8 * j);
  }
  return out;
}

}  // namespace cb
