// Index arithmetic of the 8-bit operators that the host can run too: division by a launch constant.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define LCB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LCB_HOST_DEVICE inline
#endif

namespace lcb {

// ---- division by a launch constant ----------------------------------------------------------------------------
// magic = floor((2^bits - 1) / d): the high half of n * magic is the quotient or one less, for every n of `bits` bits.
LCB_HOST_DEVICE uint64_t high_half(uint64_t a, uint64_t b) {
#ifdef __CUDA_ARCH__
    return __umul64hi(a, b);
#else
    return (uint64_t)((unsigned __int128)a * b >> 64);
#endif
}
LCB_HOST_DEVICE uint32_t high_half(uint32_t a, uint32_t b) {
#ifdef __CUDA_ARCH__
    return __umulhi(a, b);
#else
    return (uint32_t)((uint64_t)a * b >> 32);
#endif
}

template <typename U>
struct FastDivide {
    U magic, d;
    static FastDivide of(U d) { return {(U)(~(U)0 / d), d}; }
    LCB_HOST_DEVICE U divmod(U n, U &rest) const {
        U q = high_half(n, magic);
        rest = n - q * d;
        if (rest >= d) {
            rest -= d;
            ++q;
        }
        return q;
    }
};
using FastDiv = FastDivide<uint64_t>;
using FastDiv32 = FastDivide<uint32_t>;

}  // namespace lcb
