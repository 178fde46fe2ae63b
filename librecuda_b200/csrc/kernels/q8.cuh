// The 8-bit row format on the device: e4m3 codes with one power-of-two scale byte per group of 32 values.
//
// A group with largest finite magnitude A gets the scale s = 2^(b - 127), b the smallest of 0..246 with
// A <= 448 s.  From the bits of A = 1.m * 2^(f - 127): 448 = 1.75 * 2^8, so s = 2^(f - 135) holds A exactly when
// 1.m <= 1.75, i.e. m <= 0x600000, and twice that otherwise.  Adding 0x7fffff - 0x600000 to the bits carries into the
// exponent field in just that second case, so b = ((bits + 0x1fffff) >> 23) - 8, clamped to [0, 246].  Subnormal A and
// zero land below 0 and get b = 0, s = 2^-127.  Multiplying by 1 / s = 2^(127 - b) is exact wherever the result matters to
// e4m3 (its smallest step is 2^-9), so the conversion to e4m3 is the only rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "lcb200_types.h"

namespace lcb {

constexpr int kGroup = 32;          // values per scale byte
constexpr int kMaxScaleByte = 246;  // 448 * 2^(246 - 127) is finite in f32 and bf16, so no value of a code overflows
constexpr unsigned kInfBits = 0x7f800000u;

// ---- division of a unit index by a launch constant ---------------------------------------------------------
// magic = floor((2^64 - 1) / d): the high half of n * magic is the quotient or one less, for every 64-bit n.
struct FastDiv {
    uint64_t magic, d;
    static FastDiv of(uint64_t d) { return {~0ull / d, d}; }
    __device__ __forceinline__ uint64_t divmod(uint64_t n, uint64_t &rest) const {
        uint64_t q = __umul64hi(n, magic);
        rest = n - q * d;
        if (rest >= d) {
            rest -= d;
            ++q;
        }
        return q;
    }
};

// ---- wide elements -------------------------------------------------------------------------------------------
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// What a read back returns: rounded once, saturating at the type's largest finite value.  The value of a code is at
// most 448 * 2^119, which only f16 cannot hold; NaN stays NaN.
template <typename T>
__device__ __forceinline__ T from_f32_finite(float x) { return from_f32<T>(x); }
template <>
__device__ __forceinline__ __half from_f32_finite<__half>(float x) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(0.0f), "f"(x));
    return __ushort_as_half((unsigned short)r);
}

// ---- scales and codes ---------------------------------------------------------------------------------------
__device__ __forceinline__ int scale_byte(unsigned top_bits) {
    const int b = (int)((top_bits + 0x1fffffu) >> 23) - 8;
    return min(max(b, 0), kMaxScaleByte);
}
__device__ __forceinline__ float scale_inverse(int b) { return __uint_as_float((unsigned)(254 - b) << 23); }
// 2^(b - 127); b = 0 is the subnormal 2^-127
__device__ __forceinline__ float scale_value(unsigned b) { return __uint_as_float(max(b << 23, 0x00400000u)); }

// bits of |x| where x is finite, 0 where it is not
__device__ __forceinline__ unsigned finite_magnitude(float x) {
    const unsigned a = __float_as_uint(x) & 0x7fffffffu;
    return a < kInfBits ? a : 0u;
}

__device__ __forceinline__ uint16_t to_codes(float lo, float hi) {  // saturates at +-448, NaN -> 0x7f
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}
// infinities are stored as NaN
__device__ __forceinline__ float nan_if_infinite(float x) {
    return (__float_as_uint(x) & 0x7fffffffu) == kInfBits ? __uint_as_float(0x7fffffffu) : x;
}
__device__ __forceinline__ __half2 from_codes(uint16_t c) {  // exact: every code is an f16 value
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(c));
    return *reinterpret_cast<__half2 *>(&r);
}
__device__ __forceinline__ float from_code(uint8_t c) { return __low2float(from_codes(c)); }

// ---- an index out of range in device memory -----------------------------------------------------------------------
__device__ __forceinline__ void raise_error(const ErrorSink &e, unsigned bits) {
    atomicOr(e.word, bits);
    unsigned int *m = *e.mirror;
    if (m != nullptr) {
        atomicOr_system(m, bits);
        __threadfence_system();
    }
}

}  // namespace lcb
