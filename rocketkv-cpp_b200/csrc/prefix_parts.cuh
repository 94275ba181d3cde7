// prefix_parts.cuh -- what the joins may read of the tcgen05 kernel's parts, and how that kernel's roles divide its
// registers.
// Plain integer arithmetic, compiled for the host too (tests/prefix_parts_check.cpp).
#pragma once

#ifdef __CUDACC__
#define RKV_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define RKV_HOST_DEVICE inline
#endif

namespace rkv {

constexpr int kTcSms = 148;   // CTAs of the tcgen05 kernel
constexpr int kTcRows = 256;  // rows that each has in the buffer of stretches that begin inside a unit
// Parts of a row's shared tokens at most.
constexpr int kMaxShared = 152;
static_assert(kMaxShared >= kTcSms, "a unit may have a stretch per CTA");

// Whether `behind` stretches can follow a unit's first one, the first of them at row `row` of that buffer and each
// other kTcRows further.  Where the kernel gave up a wait it has left the pair unwritten, and it may be anything.
RKV_HOST_DEVICE bool parts_in_buffer(int behind, int row) {
    return behind == 0 || (behind > 0 && behind < kTcSms && row >= 0 && row < (kTcSms - (behind - 1)) * kTcRows);
}

// Threads of the tcgen05 kernel, and the registers that a thread of either half of them asks for once it has its role.
constexpr int kTcThreads = 512, kTcFewRegs = 56, kTcManyRegs = 200;
// Whether a kernel compiled to `regs` registers a thread was launched with as many as the roles ask for: where it was
// not, those that ask for more would wait for ever.
RKV_HOST_DEVICE bool split_fits(int regs) { return (long long)regs * kTcThreads >= (long long)(kTcFewRegs + kTcManyRegs) * (kTcThreads / 2); }

}  // namespace rkv
