// q = round(u / step) to e4m3 or int8 for eight values at a time: the rounding of the
// fp32 quotient.
//
// The eight quotients share a divisor, so they come from its reciprocal: with
// y = RN(1 / step), q = RN(u y) and the remainder r = q step - u by a fused
// multiply-add, RN(q - r y) is the correctly rounded quotient where q is within a unit in
// the last place (P. Markstein, "Computation of elementary functions on the IBM RISC
// System/6000 processor", 1990, theorem 8). q may be up to 1.5 units off, and r then
// rounds too: before its own rounding the result is within 2^-22 units of u / step. So
// the 8-bit result can differ from that of a division only where u / step is that close
// to the midpoint between a tie of the 8-bit type and the next fp32 value. For e4m3 and
// 16-bit u that leaves one family, step = (1 - 2^-24) 2^n under a power of two, which comes
// out right (the test of the append holds all 16-bit u against 4096 divisors); the norm's
// fp32 u have no such bound and may round the other way there.
// Three instructions a value; an IEEE division each (about 20) made the kernels that
// use this issue-bound. The remainder is taken with its sign turned, so that a zero
// quotient keeps its sign. Steps whose reciprocal or remainder would leave the normal
// range (below 2^-60, above 2^126, NaN) are divided, and so are eight values of which one
// may be beyond 512 steps (`bounded` false): where q is infinite, q - r y is not a number.
// Values whose step comes from their own maximum are bounded (an infinity among them makes
// the step infinite).
#pragma once

#include <cstdint>
#include <cuda_fp8.h>

namespace cb {

// int8 rounds half away from zero, e4m3 to nearest even, saturated.
template <bool INT8>
__device__ __forceinline__ uint64_t quant8(const float (&u)[8], float step, bool bounded = true) {
  float v[8];
  if (bounded && step >= 8.673617379884035e-19f && step <= 8.507059173023462e+37f) {  // 2^-60, 2^126
    const float y = __fdiv_rn(1.0f, step);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q = __fmul_rn(u[j], y);
      v[j] = __fmaf_rn(-__fmaf_rn(q, step, -u[j]), y, q);
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
