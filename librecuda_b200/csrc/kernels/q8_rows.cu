// 8-bit activation checkpoints for sm_100a: packing and unpacking a matrix, and the gated unit gate * up / (1 + exp(-gate))
// that leaves its checkpoint in the forward pass and reads it in the backward pass.
//
// All loads of a CTA are issued before its first store.
#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

// units in flight per lane, at most
constexpr int kPasses = 4;
constexpr int kPassesUnpack = 2;
constexpr int kPassesSilu = 2;  // of each input
constexpr int kPassesGrad = 1;

template <typename T>
struct Rows {  // rows of the wide type
    T *p;
    size_t stride;
};
struct Packed {
    uint8_t *codes, *scales;
};

struct Shape {
    uint64_t rows, cols, groups;
    Tiling tiling;
    template <int V>
    static Shape of(size_t rows, size_t cols, int max_passes) {
        const uint64_t groups = groups_of(cols);
        return {rows, cols, groups, Tiling::of(rows, Form<V>::per_row(groups), max_passes)};
    }
};

// A lane's column and its rows.
template <int V>
struct Place {
    uint64_t row, column, group;
    uint64_t rows_left;  // from `row` on
    uint32_t step, passes;
    int left;    // columns from the unit's first one on; 0 where it lies behind the row (V > 1: a row ends with a whole unit)
    bool leads;  // its group, and so writes the scale
    __device__ __forceinline__ explicit Place(const Shape &s) {
        const Lane lane(s.tiling, blockIdx.x);
        row = lane.line;
        column = lane.unit * Form<V>::kValues;
        group = lane.unit / Form<V>::kLanes;
        leads = lane.unit % Form<V>::kLanes == 0;
        step = s.tiling.side_by_side;
        passes = s.tiling.passes;
        left = lane.in && column < s.cols ? (int)min(s.cols - column, (uint64_t)INT32_MAX) : 0;
        rows_left = row < s.rows ? s.rows - row : 0;
    }
    __device__ __forceinline__ bool in(int pass) const { return left > 0 && pass * step < rows_left; }
    __device__ __forceinline__ uint8_t *code(const Packed &p, const Shape &s, int pass) const {
        return p.codes + (row * s.cols + column) + pass * (step * s.cols);
    }
    __device__ __forceinline__ uint8_t *scale(const Packed &p, const Shape &s, int pass) const {
        return p.scales + (row * s.groups + group) + pass * (step * s.groups);
    }
    template <typename T>
    __device__ __forceinline__ T *wide(const Rows<T> &r, int pass) const { return r.p + (row * r.stride + column) + pass * (step * r.stride); }
};

template <typename T, int V>
__device__ __forceinline__ void pack_and_store(const Packed &out, const Shape &s, const Place<V> &at, int pass, const Unit<T, V> &x) {
    Codes<V> c;
    const unsigned b = pack_unit(x, c);
    if (!at.in(pass)) return;
    c.store(at.code(out, s, pass), at.left);
    if (at.leads) *at.scale(out, s, pass) = (uint8_t)b;
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) pack_kernel(Packed out, Rows<const T> src, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s);
    Unit<T, V> x[kPasses];
    pdl_wait();
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        x[u].clear();
        if (u < at.passes && at.in(u)) x[u].load(at.wide(src, u), at.left);
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u)
        if (u < at.passes) pack_and_store(out, s, at, u, x[u]);
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) unpack_kernel(Rows<T> dst, Packed in, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s);
    Codes<V> c[kPassesUnpack];
    unsigned b[kPassesUnpack];
    pdl_wait();
#pragma unroll
    for (int u = 0; u < kPassesUnpack; ++u) {
        if (u < at.passes && at.in(u)) {
            c[u].load(at.code(in, s, u), at.left);
            b[u] = *at.scale(in, s, u);
        }
    }
#pragma unroll
    for (int u = 0; u < kPassesUnpack; ++u) {
        if (u >= at.passes || !at.in(u)) continue;
        const Pair scale(scale_value(b[u]));
        Unit<T, V> y;
#pragma unroll
        for (int j = 0; j < Form<V>::kValues; j += 2) y.template set_pair<true>(j, c[u].pair(j, scale));
        y.store(at.wide(dst, u), at.left);
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) silu_mul_pack_kernel(Rows<T> h, Packed gate_out, Packed up_out, Rows<const T> gate,
                                                                    Rows<const T> up, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s);
    Unit<T, V> g[kPassesSilu], u[kPassesSilu];
    pdl_wait();
#pragma unroll
    for (int k = 0; k < kPassesSilu; ++k) {
        g[k].clear();
        u[k].clear();
        if (k < at.passes && at.in(k)) {
            g[k].load(at.wide(gate, k), at.left);
            u[k].load(at.wide(up, k), at.left);
        }
    }
#pragma unroll
    for (int k = 0; k < kPassesSilu; ++k) {
        if (k >= at.passes) break;
        if (at.in(k)) {
            Unit<T, V> out;
#pragma unroll
            for (int j = 0; j < Form<V>::kValues; j += 2) {
                const Pair x = g[k].pair(j);
                out.template set_pair<false>(j, x * sigmoid(x).s * u[k].pair(j));
            }
            out.store(at.wide(h, k), at.left);
        }
        pack_and_store(gate_out, s, at, k, g[k]);
        pack_and_store(up_out, s, at, k, u[k]);
    }
}

template <typename T, int V, bool AGAIN>
__global__ void __launch_bounds__(kMaxThreads) silu_mul_grad_kernel(Rows<T> dgate, Rows<T> dup, Rows<T> h, Rows<const T> dh, Packed gate,
                                                                    Packed up, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s);
    pdl_wait();
    if (!at.in(0)) return;
    Unit<T, V> d;
    Codes<V> g, u;
    d.load(at.wide(dh, 0), at.left);
    g.load(at.code(gate, s, 0), at.left);
    u.load(at.code(up, s, 0), at.left);
    const Pair gs(scale_value(*at.scale(gate, s, 0))), us(scale_value(*at.scale(up, s, 0)));
    Unit<T, V> dg, du, y;
#pragma unroll
    for (int j = 0; j < Form<V>::kValues; j += 2) {
        const Pair x = g.pair(j, gs), z = u.pair(j, us), dj = d.pair(j);
        const Sigmoid sg = sigmoid(x);
        const Pair silu = x * sg.s;
        du.template set_pair<false>(j, dj * silu);
        dg.template set_pair<false>(j, dj * z * fma2(silu, sg.q, sg.s));
        if constexpr (AGAIN) y.template set_pair<false>(j, silu * z);
    }
    du.store(at.wide(dup, 0), at.left);
    dg.store(at.wide(dgate, 0), at.left);
    if constexpr (AGAIN) y.store(at.wide(h, 0), at.left);
}

// The widest unit whose accesses are aligned in every row: codes and values of a unit start at multiples of its size.
// A row's codes lie behind each other, so the columns must be a multiple of the unit; 16 values take 32-byte accesses of the
// wide type (f32: two) and 16-byte ones of the codes, 8 values half of that.
struct Fit {
    uint64_t wide = 0, codes = 0;
    template <typename T>
    void add(const Rows<T> &r, size_t rows) {
        if (r.p != nullptr) wide |= reinterpret_cast<uintptr_t>(r.p) | (rows > 1 ? r.stride * sizeof(T) : 0);
    }
    void add(const Packed &p) { codes |= reinterpret_cast<uintptr_t>(p.codes); }
    int unit(size_t cols) const {
        if (cols % 16 == 0 && wide % 32 == 0 && codes % 16 == 0) return 16;
        if (cols % 8 == 0 && wide % 16 == 0 && codes % 8 == 0) return 8;
        return 1;
    }
};

template <typename... KArgs, typename... Args>
int launch_rows(void (*kernel)(KArgs...), const Shape &s, lcbStream stream, Args... args) {
    const uint64_t blocks = s.tiling.blocks();
    if (blocks > 0x7fffffffu) return 1;
    return launch_kernel(kernel, (unsigned)blocks, s.tiling.threads, 0, static_cast<cudaStream_t>(stream), args..., s);
}

Packed packed(const void *codes, const void *scales) {
    return {static_cast<uint8_t *>(const_cast<void *>(codes)), static_cast<uint8_t *>(const_cast<void *>(scales))};
}
template <typename T, typename P>
Rows<T> rows_at(P *p, size_t stride) { return {static_cast<T *>(p), stride}; }

}  // namespace
}  // namespace lcb

using namespace lcb;

extern "C" int lcb_pack_q8(void *codes, void *scales, const void *src, size_t src_stride, int type, size_t rows, size_t cols,
                           lcbStream stream) {
    if (!pack_ok(codes, scales, src, src_stride, type, rows, cols, false)) return 1;
    if (rows == 0 || cols == 0) return 0;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto in = rows_at<const T>(src, src_stride);
        const Packed out = packed(codes, scales);
        Fit fit;
        fit.add(in, rows);
        fit.add(out);
        return with_unit(fit.unit(cols), [&](auto v) {
            return launch_rows(pack_kernel<T, v()>, Shape::of<v()>(rows, cols, kPasses), stream, out, in);
        });
    });
}

extern "C" int lcb_unpack_q8(void *dst, size_t dst_stride, int type, const void *codes, const void *scales, size_t rows, size_t cols,
                             lcbStream stream) {
    if (!pack_ok(codes, scales, dst, dst_stride, type, rows, cols, true)) return 1;
    if (rows == 0 || cols == 0) return 0;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto out = rows_at<T>(dst, dst_stride);
        const Packed in = packed(codes, scales);
        Fit fit;
        fit.add(out, rows);
        fit.add(in);
        return with_unit(fit.unit(cols), [&](auto v) {
            return launch_rows(unpack_kernel<T, v()>, Shape::of<v()>(rows, cols, kPassesUnpack), stream, out, in);
        });
    });
}

extern "C" int lcb_silu_mul_pack_q8(void *h, size_t h_stride, void *gate_codes, void *gate_scales, void *up_codes, void *up_scales,
                                    const void *gate, size_t gate_stride, const void *up, size_t up_stride, int type, size_t rows,
                                    size_t cols, lcbStream stream) {
    if (!silu_pack_ok(h, h_stride, gate_codes, gate_scales, up_codes, up_scales, gate, gate_stride, up, up_stride, type, rows, cols)) return 1;
    if (rows == 0 || cols == 0) return 0;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto out = rows_at<T>(h, h_stride);
        const auto g = rows_at<const T>(gate, gate_stride), u = rows_at<const T>(up, up_stride);
        const Packed gp = packed(gate_codes, gate_scales), upk = packed(up_codes, up_scales);
        Fit fit;
        fit.add(out, rows);
        fit.add(g, rows);
        fit.add(u, rows);
        fit.add(gp);
        fit.add(upk);
        return with_unit(fit.unit(cols), [&](auto v) {
            return launch_rows(silu_mul_pack_kernel<T, v()>, Shape::of<v()>(rows, cols, kPassesSilu), stream, out, gp, upk, g, u);
        });
    });
}

extern "C" int lcb_silu_mul_grad_q8(void *dgate, size_t dgate_stride, void *dup, size_t dup_stride, void *h, size_t h_stride,
                                    const void *dh, size_t dh_stride, const void *gate_codes, const void *gate_scales,
                                    const void *up_codes, const void *up_scales, int type, size_t rows, size_t cols, lcbStream stream) {
    if (!silu_grad_ok(dgate, dgate_stride, dup, dup_stride, h, h_stride, dh, dh_stride, gate_codes, gate_scales, up_codes, up_scales, type,
                      rows, cols))
        return 1;
    if (rows == 0 || cols == 0) return 0;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto dg = rows_at<T>(dgate, dgate_stride), du = rows_at<T>(dup, dup_stride), out = rows_at<T>(h, h_stride);
        const auto d = rows_at<const T>(dh, dh_stride);
        const Packed gp = packed(gate_codes, gate_scales), upk = packed(up_codes, up_scales);
        Fit fit;
        fit.add(dg, rows);
        fit.add(du, rows);
        fit.add(out, rows);
        fit.add(d, rows);
        fit.add(gp);
        fit.add(upk);
        return with_unit(fit.unit(cols), [&](auto v) {
            return launch_rows(h != nullptr ? silu_mul_grad_kernel<T, v(), true> : silu_mul_grad_kernel<T, v(), false>,
                               Shape::of<v()>(rows, cols, kPassesGrad), stream, dg, du, out, d, gp, upk);
        });
    });
}
