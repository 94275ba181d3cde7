// weight_list.cuh -- which tokens a lane of the weight selection lists.
// Plain integer arithmetic, compiled for the host too (tests/weight_list_check.cpp).
#pragma once

#ifdef __CUDACC__
#define RKV_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define RKV_HOST_DEVICE inline
#endif

namespace rkv {

// Bits 0 .. n - 1 of 16.
RKV_HOST_DEVICE unsigned first_bits16(int n) { return n <= 0 ? 0u : n >= 16 ? 0xFFFFu : (1u << n) - 1u; }

// Bit e for token i0 + e, of the 16 that a lane looks at.  marked: bits of the tokens whose key is at or above
// the threshold (of any token where all keys are).  Tokens outside [c0, c1) are sinks or recent: they do not
// compete and are listed.  Nothing is listed from t1 on, where the next warp's stretch begins and lists its own:
// a token listed twice would be counted and written twice.
RKV_HOST_DEVICE unsigned listed_tokens(unsigned marked, int i0, int c0, int c1, int t1) {
    const unsigned competes = first_bits16(c1 - i0) & ~first_bits16(c0 - i0);
    return (marked | ~competes) & first_bits16(t1 - i0);
}

}  // namespace rkv
