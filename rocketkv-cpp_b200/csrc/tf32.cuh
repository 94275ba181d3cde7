// tf32.cuh -- fp32 operands of tf32 matrix instructions as two parts.
#pragma once

#include <stdint.h>

namespace rkv {

// x = hi + lo.  A tf32 operand is the top 19 bits of what it is given, so hi
// is x itself; lo is what those bits leave, exactly, plus half a step of its
// own cut, so that this cut rounds to nearest.  Relative to x the parts leave
// 2^-22 or so.  Errors of an fp32 attention's output against 64 bits, and the
// decode's rate with 3 heads of 128 columns a KV head: this 0.6e-6 to 0.9e-6
// at 6.6 TB/s; lo cut too 1.0e-6 to 1.5e-6 at 6.6; hi rounded by the
// conversion instruction 0.5e-6 to 0.8e-6 at 5.7.
__device__ __forceinline__ void tf32_split(uint32_t x, uint32_t& hi, uint32_t& lo) {
    hi = x;
    lo = __float_as_uint(__uint_as_float(x) - __uint_as_float(x & 0xFFFFE000u)) + 0x1000u;
}

}  // namespace rkv
