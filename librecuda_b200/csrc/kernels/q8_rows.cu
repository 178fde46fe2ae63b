// 8-bit activation checkpoints for sm_100a: packing and unpacking a matrix, and the gated unit gate * up / (1 + exp(-gate))
// that leaves its checkpoint in the forward pass and reads it in the backward pass.
//
// One lane per value, one warp per group: a warp's 32 lanes hold the 32 consecutive values of a group, so the largest
// magnitude is one warp-wide maximum over the bits and any number of columns, stride and alignment is the same case.
#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct Rows {  // rows of the wide type
    T *p;
    size_t stride;
};
struct Packed {
    uint8_t *codes, *scales;
};

struct Shape {
    uint64_t cols, groups;  // per row
    uint64_t total;         // lanes of all rows, a row padded to whole groups
    FastDiv per_row;        // by the lanes of a row
    static Shape of(size_t rows, size_t cols) {
        const uint64_t groups = groups_of(cols);
        return {cols, groups, rows * groups * kGroup, FastDiv::of(groups * kGroup)};
    }
};

struct Lane {
    uint64_t row, col;
    bool in;  // a value of the matrix; lanes behind the last column of a row belong to its last group all the same
    __device__ __forceinline__ Lane(const Shape &s) {
        const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
        row = s.per_row.divmod(i, col);
        in = i < s.total && col < s.cols;
    }
};

// Called by whole warps: packs the warp's group.
__device__ __forceinline__ void pack_group(const Packed &out, const Shape &s, const Lane &at, float x) {
    const unsigned top = __reduce_max_sync(0xffffffffu, at.in ? finite_magnitude(x) : 0u);
    const int b = scale_byte(top);
    if (!at.in) return;
    const uint16_t c = to_codes(nan_if_infinite(x) * scale_inverse(b), 0.0f);
    out.codes[at.row * s.cols + at.col] = (uint8_t)c;
    if ((at.col & (kGroup - 1)) == 0) out.scales[at.row * s.groups + at.col / kGroup] = (uint8_t)b;
}

__device__ __forceinline__ float unpack_one(const Packed &in, const Shape &s, const Lane &at) {
    return from_code(in.codes[at.row * s.cols + at.col]) * scale_value(in.scales[at.row * s.groups + at.col / kGroup]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pack_kernel(Packed out, Rows<const T> src, Shape s) {
    pdl_launch_dependents();
    pdl_wait();
    const Lane at(s);
    const float x = at.in ? to_f32(src.p[at.row * src.stride + at.col]) : 0.0f;
    pack_group(out, s, at, x);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) unpack_kernel(Rows<T> dst, Packed in, Shape s) {
    pdl_launch_dependents();
    pdl_wait();
    const Lane at(s);
    if (at.in) dst.p[at.row * dst.stride + at.col] = from_f32_finite<T>(unpack_one(in, s, at));
}

__device__ __forceinline__ float sigmoid(float x) { return 1.0f / (1.0f + expf(-x)); }

template <typename T>
__global__ void __launch_bounds__(kThreads) silu_mul_pack_kernel(Rows<T> h, Packed gate_out, Packed up_out, Rows<const T> gate,
                                                                 Rows<const T> up, Shape s) {
    pdl_launch_dependents();
    pdl_wait();
    const Lane at(s);
    const float g = at.in ? to_f32(gate.p[at.row * gate.stride + at.col]) : 0.0f;
    const float u = at.in ? to_f32(up.p[at.row * up.stride + at.col]) : 0.0f;
    if (at.in) h.p[at.row * h.stride + at.col] = from_f32<T>(g * sigmoid(g) * u);
    pack_group(gate_out, s, at, g);
    pack_group(up_out, s, at, u);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) silu_mul_grad_kernel(Rows<T> dgate, Rows<T> dup, Rows<T> h, Rows<const T> dh, Packed gate,
                                                                 Packed up, Shape s) {
    pdl_launch_dependents();
    pdl_wait();
    const Lane at(s);
    if (!at.in) return;
    const float g = unpack_one(gate, s, at), u = unpack_one(up, s, at);
    const float d = to_f32(dh.p[at.row * dh.stride + at.col]);
    const float sg = sigmoid(g), silu = g * sg;
    dup.p[at.row * dup.stride + at.col] = from_f32<T>(d * silu);
    dgate.p[at.row * dgate.stride + at.col] = from_f32<T>(d * u * (sg + silu * (1.0f - sg)));
    if (h.p != nullptr) h.p[at.row * h.stride + at.col] = from_f32<T>(silu * u);
}

template <typename... KArgs, typename... Args>
int launch_rows(void (*kernel)(KArgs...), const Shape &s, lcbStream stream, Args... args) {
    const uint64_t blocks = (s.total + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffffu) return 1;
    return launch_kernel(kernel, (unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream), args..., s);
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

Packed packed(const void *codes, const void *scales) {
    return {static_cast<uint8_t *>(const_cast<void *>(codes)), static_cast<uint8_t *>(const_cast<void *>(scales))};
}

}  // namespace
}  // namespace lcb

using namespace lcb;

extern "C" int lcb_pack_q8(void *codes, void *scales, const void *src, size_t src_stride, int type, size_t rows, size_t cols,
                           lcbStream stream) {
    if (!pack_ok(codes, scales, src, src_stride, type, rows, cols, false)) return 1;
    if (rows == 0 || cols == 0) return 0;
    const Shape s = Shape::of(rows, cols);
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows(pack_kernel<T>, s, stream, packed(codes, scales), Rows<const T>{static_cast<const T *>(src), src_stride});
    });
}

extern "C" int lcb_unpack_q8(void *dst, size_t dst_stride, int type, const void *codes, const void *scales, size_t rows, size_t cols,
                             lcbStream stream) {
    if (!pack_ok(codes, scales, dst, dst_stride, type, rows, cols, true)) return 1;
    if (rows == 0 || cols == 0) return 0;
    const Shape s = Shape::of(rows, cols);
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows(unpack_kernel<T>, s, stream, Rows<T>{static_cast<T *>(dst), dst_stride}, packed(codes, scales));
    });
}

extern "C" int lcb_silu_mul_pack_q8(void *h, size_t h_stride, void *gate_codes, void *gate_scales, void *up_codes, void *up_scales,
                                    const void *gate, size_t gate_stride, const void *up, size_t up_stride, int type, size_t rows,
                                    size_t cols, lcbStream stream) {
    if (!silu_pack_ok(h, h_stride, gate_codes, gate_scales, up_codes, up_scales, gate, gate_stride, up, up_stride, type, rows, cols)) return 1;
    if (rows == 0 || cols == 0) return 0;
    const Shape s = Shape::of(rows, cols);
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows(silu_mul_pack_kernel<T>, s, stream, Rows<T>{static_cast<T *>(h), h_stride}, packed(gate_codes, gate_scales),
                           packed(up_codes, up_scales), Rows<const T>{static_cast<const T *>(gate), gate_stride},
                           Rows<const T>{static_cast<const T *>(up), up_stride});
    });
}

extern "C" int lcb_silu_mul_grad_q8(void *dgate, size_t dgate_stride, void *dup, size_t dup_stride, void *h, size_t h_stride,
                                    const void *dh, size_t dh_stride, const void *gate_codes, const void *gate_scales,
                                    const void *up_codes, const void *up_scales, int type, size_t rows, size_t cols, lcbStream stream) {
    if (!silu_grad_ok(dgate, dgate_stride, dup, dup_stride, h, h_stride, dh, dh_stride, gate_codes, gate_scales, up_codes, up_scales, type,
                      rows, cols))
        return 1;
    if (rows == 0 || cols == 0) return 0;
    const Shape s = Shape::of(rows, cols);
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return launch_rows(silu_mul_grad_kernel<T>, s, stream, Rows<T>{static_cast<T *>(dgate), dgate_stride},
                           Rows<T>{static_cast<T *>(dup), dup_stride}, Rows<T>{static_cast<T *>(h), h_stride},
                           Rows<const T>{static_cast<const T *>(dh), dh_stride}, packed(gate_codes, gate_scales), packed(up_codes, up_scales));
    });
}
