// The 8-bit row format on the device: e4m3 codes with one power-of-two scale byte per group of 32 values.
//
// A group with largest finite magnitude A gets the scale s = 2^(b - 127), b the smallest of 0..246 with A <= 448 s.
// From the bits of A = 1.m * 2^(f - 127): 448 = 1.75 * 2^8, so s = 2^(f - 135) holds A exactly when 1.m <= 1.75, i.e.
// m <= 0x600000, and twice that otherwise.  Adding 0x7fffff - 0x600000 to the bits carries into the exponent field in
// just that second case, so b = ((bits + 0x1fffff) >> 23) - 8, clamped to [0, 246].  Subnormal A and zero land below
// 0 and get b = 0, s = 2^-127.  Multiplying by 1 / s = 2^(127 - b) is exact wherever the result matters to e4m3 (its
// smallest step is 2^-9), so the conversion to e4m3 is the only rounding.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <initializer_list>
#include <type_traits>

#include "common.cuh"
#include "lcb200_types.h"
#include "q8_tiling.h"

namespace lcb {

constexpr int kMaxScaleByte = 246;  // 448 * 2^(246 - 127) is finite in f32 and bf16, so no value of a code overflows
constexpr unsigned kInfBits = 0x7f800000u;

// ---- a lane's place (tilings: q8_tiling.h) ------------------------------------------------------------------------
struct Lane {
    uint64_t line;  // of the first pass; the next ones are side_by_side further each
    uint64_t unit;  // of the line
    bool in;        // has a unit; lanes without one still take part in a warp's votes and shuffles
    __device__ __forceinline__ Lane(const Tiling &t, uint32_t block, uint32_t passes) {
        uint32_t chunk;
        const uint32_t tile = t.by_chunks.divmod(block, chunk);
        *this = Lane(t, tile, chunk, passes);
    }
    __device__ __forceinline__ Lane(const Tiling &t, uint32_t tile, uint32_t chunk, uint32_t passes) {
        if (t.by_chunks.d == 1) {
            uint32_t place;
            const uint32_t local = t.by_width.divmod(threadIdx.x, place);
            line = (uint64_t)tile * (t.side_by_side * passes) + local;
            unit = place;
            in = local < t.side_by_side;
        } else {
            line = (uint64_t)tile * passes;
            unit = (uint64_t)chunk * t.threads + threadIdx.x;
            in = unit < t.width && threadIdx.x < t.threads;  // a CTA may be wider than this tiling asks for
        }
    }
};

// ---- a warp's run of values -----------------------------------------------------------------------------------------
// Up to 512 values of T that lie behind each other at any address, 16 to a lane, accessed in aligned words, lane by
// lane side by side.  In shared memory a lane's words have one word of room behind them, so that the accesses by word
// and those by lane both find 32 different banks.
template <typename T>
struct Run {
    static constexpr int kLaneWords = 16 * (int)sizeof(T) / 4;
    static constexpr int kSteps = kLaneWords + (sizeof(T) == 2);  // a run that starts inside a word covers one more
    static constexpr int kScratch = 32 * (kLaneWords + 1) + 1;
    __device__ static __forceinline__ int slot(int word) { return word + word / kLaneWords; }
    __device__ static __forceinline__ int lane() { return threadIdx.x & 31; }
    // values of the run, from every lane's columns to the end of the row
    __device__ static __forceinline__ int values(int left) { return (int)__reduce_add_sync(0xffffffffu, (unsigned)min(left, 16)); }

    // p: the lane's first value.  Words that hold at least one value of the run are read whole.
    __device__ static __forceinline__ bool odd(const T *p) { return sizeof(T) == 2 && (reinterpret_cast<uintptr_t>(p) & 2); }
    __device__ static __forceinline__ void load(uint32_t (&r)[kSteps], const T *p, int left) {
        const int n = values(left), words = sizeof(T) == 2 ? (n + (int)odd(p) + 1) / 2 : n;
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p - lane() * 16 - (int)odd(p));
#pragma unroll
        for (int k = 0; k < kSteps; ++k) r[k] = n > 0 && k * 32 + lane() < words ? q[k * 32 + lane()] : 0u;
    }
    __device__ static __forceinline__ void hand_out(const uint32_t (&r)[kSteps], uint32_t (&w)[kLaneWords], const T *p, uint32_t *scratch) {
#pragma unroll
        for (int k = 0; k < kSteps; ++k)
            if (k < kLaneWords || lane() == 0) scratch[slot(k * 32 + lane())] = r[k];
        __syncwarp();
        uint32_t t[kLaneWords + 1];
#pragma unroll
        for (int i = 0; i < kLaneWords; ++i) t[i] = scratch[lane() * (kLaneWords + 1) + i];
        t[kLaneWords] = sizeof(T) == 2 ? scratch[(lane() + 1) * (kLaneWords + 1)] : 0u;
#pragma unroll
        for (int i = 0; i < kLaneWords; ++i) w[i] = __funnelshift_r(t[i], t[i + 1], odd(p) ? 16 : 0);
        __syncwarp();
    }
    __device__ static __forceinline__ void store(const uint32_t (&w)[kLaneWords], T *p, int left, uint32_t *scratch) {
        const int n = values(left);
#pragma unroll
        for (int i = 0; i < kLaneWords; ++i) scratch[lane() * (kLaneWords + 1) + i] = w[i];
        __syncwarp();
        T *first = p - lane() * 16;
        if (!odd(p)) {
            uint32_t *q = reinterpret_cast<uint32_t *>(first);
            const int words = sizeof(T) == 2 ? n / 2 : n;
#pragma unroll
            for (int k = 0; k < kLaneWords; ++k)
                if (k * 32 + lane() < words) q[k * 32 + lane()] = scratch[slot(k * 32 + lane())];
        } else {
            uint32_t *q = reinterpret_cast<uint32_t *>(first + 1);  // the words from the second value on
            const int words = (n - 1) / 2;
#pragma unroll
            for (int k = 0; k < kLaneWords; ++k) {
                const int word = k * 32 + lane();
                if (word < words) q[word] = __funnelshift_r(scratch[slot(word)], scratch[slot(word + 1)], 16);
            }
            if (lane() == 0 && n > 0) *reinterpret_cast<uint16_t *>(first) = (uint16_t)scratch[0];
        }
        if constexpr (sizeof(T) == 2) {  // a last value that no word holds
            if (lane() == 1 && n > (int)odd(p) && ((n - (int)odd(p)) & 1))
                reinterpret_cast<uint16_t *>(first)[n - 1] = (uint16_t)(scratch[slot((n - 1) / 2)] >> (16 * ((n - 1) & 1)));
        }
        __syncwarp();
    }
};
// a warp's scratch for runs of T
template <typename T, int A>
__device__ __forceinline__ uint32_t *run_scratch() {
    if constexpr (A == kWarp) {
        __shared__ uint32_t all[kMaxThreads / 32][Run<T>::kScratch];
        return all[threadIdx.x / 32];
    } else {
        return nullptr;
    }
}

// ---- pairs: two 32-bit operations in one instruction ----------------------------------------------------------------
struct Pair {
    uint64_t v;
    Pair() = default;
    __device__ __forceinline__ Pair(float x, float y) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y)); }
    __device__ __forceinline__ explicit Pair(float x) : Pair(x, x) {}
    __device__ __forceinline__ float2 get() const {
        float2 f;
        asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(v));
        return f;
    }
};
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}

// ---- wide elements -------------------------------------------------------------------------------------------
// Two values rounded to a 16-bit type, `lo` in the lower half.  FINITE: saturating at the largest finite value, what a
// read back returns (the value of a code is at most 448 * 2^119, which only f16 cannot hold; NaN stays NaN).
template <typename T, bool FINITE>
__device__ __forceinline__ uint32_t pair_from_f32(float lo, float hi) {
    uint32_t r;
    if constexpr (std::is_same_v<T, __half>) {
        if constexpr (FINITE) asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
        else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    } else {
        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    }
    return r;
}

template <typename T, int A>
struct Unit {  // as it lies in memory
    static constexpr int kValues = Form<A>::kValues;
    static constexpr int kWords = kValues * (int)sizeof(T) / 4;
    static constexpr int kPerWord = 4 / (int)sizeof(T);
    uint32_t w[kWords];
    uint32_t run[A == kWarp ? Run<T>::kSteps : 1];  // kWarp: as loaded, before it is handed out
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    // `left`: columns from the unit's first one to the end of the row, 0: no unit.  Values behind the end are 0.
    // Every lane of the warp calls this, take() before it looks at a value, and store().
    __device__ __forceinline__ void load(const T *p, int left) {
        const uint32_t *q = reinterpret_cast<const uint32_t *>(p);
        clear();
        if constexpr (A == kWarp) {
            Run<T>::load(run, p, left);
            return;
        }
        if (left <= 0) return;
        if constexpr (A == 32) {
#pragma unroll
            for (int i = 0; i < kWords; i += 8)
                asm volatile("ld.global.L1::no_allocate.v8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                             : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]), "=r"(w[i + 4]),
                               "=r"(w[i + 5]), "=r"(w[i + 6]), "=r"(w[i + 7])
                             : "l"(q + i));
        } else if constexpr (A == 16) {  // the lanes' accesses interleave: the second one finds its sectors in L1
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 v = i * kPerWord < left ? ld_stream<1>(reinterpret_cast<const uint4 *>(q + i)) : make_uint4(0, 0, 0, 0);
                w[i] = v.x, w[i + 1] = v.y, w[i + 2] = v.z, w[i + 3] = v.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = i < left ? q[i] : 0u;
        } else {
            // the aligned words that hold at least one of the values, shifted by half a word where the address asks
            // for it
            const uint32_t odd = (uint32_t)(reinterpret_cast<uintptr_t>(p) >> 1) & 1u;
            q = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
            const int n = min(left, kValues) + (int)odd;
            uint32_t r[kWords + 1];
#pragma unroll
            for (int i = 0; i <= kWords; ++i) r[i] = 2 * i < n ? q[i] : 0u;
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(r[i], r[i + 1], 16 * odd);
            end_at(left);
        }
    }
    __device__ __forceinline__ void end_at(int left) {
        if (left >= kValues) return;
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = i < left ? w[i] : 0u;
            else w[i] = 2 * i + 1 < left ? w[i] : 2 * i < left ? w[i] & 0xffffu : 0u;
        }
    }
    __device__ __forceinline__ void take(const T *p, int left, uint32_t *scratch) {
        if constexpr (A == kWarp) {
            Run<T>::hand_out(run, w, p, scratch);
            end_at(left);
        }
    }
    __device__ __forceinline__ void store(T *p, int left, uint32_t *scratch) const {
        uint32_t *q = reinterpret_cast<uint32_t *>(p);
        if constexpr (A == kWarp) {
            Run<T>::store(w, p, left, scratch);
            return;
        }
        if (left <= 0) return;
        if constexpr (A == 32) {
#pragma unroll
            for (int i = 0; i < kWords; i += 8)
                asm volatile("st.global.L1::no_allocate.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
                             :: "l"(q + i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]),
                                "r"(w[i + 5]), "r"(w[i + 6]), "r"(w[i + 7])
                             : "memory");
        } else if constexpr (A == 16) {
#pragma unroll
            for (int i = 0; i < kWords; i += 4)
                if (i * kPerWord < left) st_stream<1>(reinterpret_cast<uint4 *>(q + i), make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]));
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                if (i < left) q[i] = w[i];
        } else {
            uint16_t *h = reinterpret_cast<uint16_t *>(p);
            if (left < kValues) {
#pragma unroll
                for (int j = 0; j < kValues; ++j)
                    if (j < left) h[j] = (uint16_t)(w[j / 2] >> (16 * (j & 1)));
            } else if ((reinterpret_cast<uintptr_t>(p) & 2) == 0) {
#pragma unroll
                for (int i = 0; i < kWords; ++i) q[i] = w[i];
            } else {
                h[0] = (uint16_t)w[0];
#pragma unroll
                for (int i = 0; i + 1 < kWords; ++i) *reinterpret_cast<uint32_t *>(h + 1 + 2 * i) = __funnelshift_r(w[i], w[i + 1], 16);
                h[kValues - 1] = (uint16_t)(w[kWords - 1] >> 16);
            }
        }
    }
    __device__ __forceinline__ float value(int j) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[j]);
        else if constexpr (std::is_same_v<T, __half>) return __half2float(__ushort_as_half((unsigned short)(w[j / 2] >> (16 * (j & 1)))));
        else return __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
    }
    __device__ __forceinline__ Pair pair(int j) const { return Pair(value(j), value(j + 1)); }  // j even
    template <bool FINITE>
    __device__ __forceinline__ void set_pair(int j, Pair x) {
        const float2 f = x.get();
        if constexpr (sizeof(T) == 4) w[j] = __float_as_uint(f.x), w[j + 1] = __float_as_uint(f.y);
        else w[j / 2] = pair_from_f32<T, FINITE>(f.x, f.y);
    }
    // Bits, as f32, of the largest magnitude that is not NaN.  16-bit values compare two at a time; the sign that the
    // instruction leaves is dropped at the end.
    __device__ __forceinline__ unsigned top_bits() const {
        if constexpr (sizeof(T) == 4) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < kWords; ++i) m = fmaxf(m, fabsf(__uint_as_float(w[i])));
            return __float_as_uint(m);
        } else {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < kWords; ++i) {
                if constexpr (std::is_same_v<T, __half>) asm("max.xorsign.abs.f16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
                else asm("max.xorsign.abs.bf16x2 %0, %0, %1;" : "+r"(m) : "r"(w[i]));
            }
            m &= 0x7fff7fffu;
            m = max(m & 0xffffu, m >> 16);
            if constexpr (std::is_same_v<T, __half>) return __float_as_uint(__half2float(__ushort_as_half((unsigned short)m)));
            else return m << 16;
        }
    }
};
// ---- scales and codes ---------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned scale_byte(unsigned top_bits) {
    const int b = (int)((top_bits + 0x1fffffu) >> 23) - 8;
    return (unsigned)min(max(b, 0), kMaxScaleByte);
}
__device__ __forceinline__ float scale_inverse(unsigned b) { return __uint_as_float((254u - b) << 23); }
// 2^(b - 127); b = 0 is the subnormal 2^-127
__device__ __forceinline__ float scale_value(unsigned b) { return __uint_as_float(max(b << 23, 0x00400000u)); }

// bits of |x| where x is finite, 0 where it is not
__device__ __forceinline__ unsigned finite_magnitude(float x) {
    const unsigned a = __float_as_uint(x) & 0x7fffffffu;
    return a < kInfBits ? a : 0u;
}
// infinities are stored as NaN
__device__ __forceinline__ float nan_if_infinite(float x) {
    return (__float_as_uint(x) & 0x7fffffffu) == kInfBits ? __uint_as_float(0x7fffffffu) : x;
}

// Largest over the lanes of a group; every lane of the warp calls it.
template <int A>
__device__ __forceinline__ unsigned group_max(unsigned m) {
#pragma unroll
    for (int o = 1; o < Form<A>::kLanes; o *= 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    return m;
}

__device__ __forceinline__ uint16_t to_codes(float lo, float hi) {  // saturates at +-448, NaN -> 0x7f
    uint16_t r;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

template <int A>
struct Codes {  // of one unit, four to a word
    static constexpr int kValues = Form<A>::kValues;
    static constexpr int kWords = kValues / 4;
    uint32_t w[kWords];
    __device__ __forceinline__ void load(const uint8_t *p, int left) {
        if (left <= 0) return;
        if constexpr (A == 32) {
            const uint4 v = ld_stream<2>(reinterpret_cast<const uint4 *>(p));
            w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
        } else if constexpr (A == 16) {
            const uint2 *q = reinterpret_cast<const uint2 *>(p);
            const uint2 lo = q[0], hi = left > 8 ? q[1] : make_uint2(0, 0);
            w[0] = lo.x, w[1] = lo.y, w[2] = hi.x, w[3] = hi.y;
        } else {
            // the aligned words that hold at least one of the codes; codes behind the row's end are whatever lies there
            const uint32_t shift = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3);
            const uint32_t *q = reinterpret_cast<const uint32_t *>(reinterpret_cast<uintptr_t>(p) & ~(uintptr_t)3);
            const int n = min(left, kValues) + (int)shift;
            uint32_t r[kWords + 1];
#pragma unroll
            for (int i = 0; i <= kWords; ++i) r[i] = 4 * i < n ? q[i] : 0u;
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __funnelshift_r(r[i], r[i + 1], 8 * shift);
        }
    }
    __device__ __forceinline__ void store(uint8_t *p, int left) const {
        if (left <= 0) return;
        if constexpr (A == 32) st_stream<2>(reinterpret_cast<uint4 *>(p), make_uint4(w[0], w[1], w[2], w[3]));
        else if constexpr (A == 16) {
            uint2 *q = reinterpret_cast<uint2 *>(p);
            q[0] = make_uint2(w[0], w[1]);
            if (left > 8) q[1] = make_uint2(w[2], w[3]);
        } else if (left < kValues) {
#pragma unroll
            for (int j = 0; j < kValues; ++j)
                if (j < left) p[j] = (uint8_t)(w[j / 4] >> (8 * (j & 3)));
        } else {
            const uint32_t m = (uint32_t)(reinterpret_cast<uintptr_t>(p) & 3);
            if (m == 0) {
#pragma unroll
                for (int i = 0; i < kWords; ++i) reinterpret_cast<uint32_t *>(p)[i] = w[i];
            } else {
                // up to the first word's boundary, the words between, and what is left of the last word
                if (m == 2) *reinterpret_cast<uint16_t *>(p) = (uint16_t)w[0];
                else p[0] = (uint8_t)w[0];
                if (m == 1) *reinterpret_cast<uint16_t *>(p + 1) = (uint16_t)(w[0] >> 8);
                uint32_t *q = reinterpret_cast<uint32_t *>(p + (4 - m));
#pragma unroll
                for (int i = 0; i + 1 < kWords; ++i) q[i] = __funnelshift_r(w[i], w[i + 1], 8 * (4 - m));
                const uint32_t rest = w[kWords - 1] >> (8 * (4 - m));
                uint8_t *e = reinterpret_cast<uint8_t *>(q + kWords - 1);
                if (m != 1) *reinterpret_cast<uint16_t *>(e) = (uint16_t)rest;
                if (m == 1) e[0] = (uint8_t)rest;
                if (m == 3) e[2] = (uint8_t)(rest >> 16);
            }
        }
    }
    // values j and j + 1 (j even), in 32 bits: a code is an f16 value exactly, and its product with a power of two is
    // exact
    __device__ __forceinline__ Pair pair(int j, Pair scale) const {
        uint32_t r;
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)(w[j / 4] >> (8 * (j & 2)))));
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r));
        return Pair(f.x, f.y) * scale;
    }
};

// Packs a unit; returns the scale byte of its group.  Every lane of the warp calls it; lanes without values come with
// a cleared unit.  The maximum ignores NaN, which convert to the NaN code by themselves; infinities are rare, so only
// when one is found somewhere in the warp the values are looked at one by one.
template <typename T, int A>
__device__ __forceinline__ unsigned pack_unit(const Unit<T, A> &in, Codes<A> &out) {
    constexpr int N = Form<A>::kValues;
    float x[N];
#pragma unroll
    for (int j = 0; j < N; ++j) x[j] = in.value(j);
    unsigned top = group_max<A>(in.top_bits());
    if (__any_sync(0xffffffffu, top >= kInfBits)) {
        top = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) {
            top = max(top, finite_magnitude(x[j]));
            x[j] = nan_if_infinite(x[j]);
        }
        top = group_max<A>(top);
    }
    const unsigned b = scale_byte(top);
    const Pair inverse(scale_inverse(b));
    auto codes = [&](int j) {
        const float2 y = (Pair(x[j], x[j + 1]) * inverse).get();
        return (uint32_t)to_codes(y.x, y.y);
    };
#pragma unroll
    for (int j = 0; j < N; j += 4) out.w[j / 4] = codes(j) | codes(j + 2) << 16;
    return b;
}

// ---- sigmoid --------------------------------------------------------------------------------------------------
// s = 1 / (1 + e) and q = 1 - s = e * s with e = exp(-g): no term cancels.  e = 2^t * (1 - ln2 * rest) with t = -g
// log2(e) rounded and rest what the rounding left of g log2(e), since an error of t counts |t| times.  s and q are good to 12
// units of 2^-24 where they are normal numbers.
//
// s is below 2^-126 from g = -87.34 down, where a reciprocal is flushed, while g * s and what it is multiplied with may
// still be large.  So the reciprocal is taken of k (1 + e), k = 1/4 or 1/2, and s = k r is held in steps of 2^-149.
//   AT_CODES false  g is any number, only s is asked for.  k = 1/4: r is normal for every finite e; below g = -88.7228 e
//                   is beyond the largest number, infinite, and s is 0.
//   AT_CODES true   g is the value of a code: 88 and 96 are neighbours.  Down to -88, k e stays below 2^126 with k = 1/2;
//                   from -96 on e is that of -88.72, k e is beyond 2^126, r is flushed and s = q = 0, where an infinite e
//                   would make q NaN.  (Infinite e and a saturating product for q: 107 us against 103 in the gradient of
//                   8192 x 10240 bf16.)
// g is held to [-100, 100] for t and rest to be finite; an infinite or NaN g still shows in g * s.
struct Sigmoid {
    Pair s, q;
};
template <bool AT_CODES>
__device__ __forceinline__ Sigmoid sigmoid(Pair g) {
    constexpr float kLog2e = 1.4426950216293335f, kLog2eRest = 1.9259629911266175e-8f, kLn2 = 0.69314718246459961f;
    constexpr float kLow = AT_CODES ? -88.72f : -100.0f, k = AT_CODES ? 0.5f : 0.25f;
    const float2 f = g.get();
    const Pair m(fminf(fmaxf(f.x, kLow), 100.0f), fminf(fmaxf(f.y, kLow), 100.0f));
    const Pair t = m * Pair(-kLog2e);
    const Pair rest = fma2(m, Pair(kLog2eRest), fma2(m, Pair(kLog2e), t));
    float2 e = t.get();
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.x));
    asm("ex2.approx.ftz.f32 %0, %0;" : "+f"(e.y));
    const Pair p = Pair(e.x, e.y) * fma2(rest, Pair(-k * kLn2), Pair(k));  // k e
    float2 d = (p + Pair(k)).get();
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.x));
    asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(d.y));
    const Pair r(d.x, d.y);
    return {r * Pair(k), p * r};
}

// calls fn with a null pointer of the element type
template <typename Fn>
int with_type(int type, Fn fn) {
    switch (type) {
        case LCB_F32: return fn(static_cast<float *>(nullptr));
        case LCB_F16: return fn(static_cast<__half *>(nullptr));
        default: return fn(static_cast<__nv_bfloat16 *>(nullptr));
    }
}

// calls fn with std::integral_constant of the access form; 0: the loose one.  WARP: whether kWarp is among the forms
template <int LOOSE, bool WARP, typename Fn>
int with_access(int a, Fn fn) {
    if (a == 32) return fn(std::integral_constant<int, 32>());
    if (a == 16) return fn(std::integral_constant<int, 16>());
    if constexpr (WARP)
        if (a == kWarp) return fn(std::integral_constant<int, kWarp>());
    return fn(std::integral_constant<int, LOOSE>());
}

// calls fn with std::integral_constant of the passes: 1 or MOST
template <int MOST, typename Fn>
int with_passes(uint32_t passes, Fn fn) {
    return passes == 1 ? fn(std::integral_constant<int, 1>()) : fn(std::integral_constant<int, MOST>());
}

// Loads a kernel onto the current device, before its first launch.
template <typename... KArgs>
int load_kernel(void (*kernel)(KArgs...)) {
    cudaFuncAttributes a;
    return (int)cudaFuncGetAttributes(&a, kernel);
}
// the first error of a list
inline int first_error(std::initializer_list<int> codes) {
    for (int c : codes)
        if (c != 0) return c;
    return 0;
}

}  // namespace lcb
