// 8-bit activation checkpoints for sm_100a: packing and unpacking a matrix, and the gated unit gate * up / (1 + exp(-gate))
// that leaves its checkpoint in the forward pass and reads it in the backward pass.
//
// All loads of a CTA are issued before its first store.
#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

constexpr int kPasses = 4;      // units in flight per lane: pack, unpack
constexpr int kPassesSilu = 2;  // the gated unit holds two inputs
constexpr int kPassesGrad = 1;  // and its gradient three, with three outputs

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
    static Shape of(size_t rows, size_t cols, int v) {
        const uint64_t groups = groups_of(cols);
        return {rows, cols, groups, Tiling::of(rows, groups * (kGroup / v))};
    }
};

// A lane's column and its rows.  The columns of a unit are all inside the matrix or all behind it; lanes behind the last
// column of a row still belong to its last group.
template <int V>
struct Place {
    uint64_t row, unit, left;  // left: rows from `row` on
    uint32_t step;
    bool in_row;
    __device__ __forceinline__ Place(const Shape &s, int passes) {
        const Lane lane(s.tiling, blockIdx.x, passes);
        row = lane.line;
        unit = lane.unit;
        step = s.tiling.side_by_side;
        in_row = lane.in && unit * V < s.cols && row < s.rows;
        left = s.rows - row;
    }
    __device__ __forceinline__ bool in(int pass) const { return in_row && pass * step < left; }
    __device__ __forceinline__ bool leads() const { return (unit & (kGroup / V - 1)) == 0; }
    __device__ __forceinline__ uint8_t *code(const Packed &p, const Shape &s, int pass) const {
        return p.codes + (row * s.cols + unit * V) + pass * (step * s.cols);
    }
    __device__ __forceinline__ uint8_t *scale(const Packed &p, const Shape &s, int pass) const {
        return p.scales + (row * s.groups + unit / (kGroup / V)) + pass * (step * s.groups);
    }
    template <typename T>
    __device__ __forceinline__ T *wide(const Rows<T> &r, int pass) const { return r.p + (row * r.stride + unit * V) + pass * (step * r.stride); }
};

template <typename T, int V>
__device__ __forceinline__ void pack_and_store(const Packed &out, const Shape &s, const Place<V> &at, int pass, const Unit<T, V> &x) {
    Codes<V> c;
    const int b = pack_unit(x, c);
    if (!at.in(pass)) return;
    c.store(at.code(out, s, pass));
    if (at.leads()) *at.scale(out, s, pass) = (uint8_t)b;
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) pack_kernel(Packed out, Rows<const T> src, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s, kPasses);
    Unit<T, V> x[kPasses];
    pdl_wait();
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        x[u].clear();
        if (at.in(u)) x[u].load(at.wide(src, u));
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) pack_and_store(out, s, at, u, x[u]);
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) unpack_kernel(Rows<T> dst, Packed in, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s, kPasses);
    Codes<V> c[kPasses];
    unsigned b[kPasses];
    pdl_wait();
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        if (at.in(u)) {
            c[u].load(at.code(in, s, u));
            b[u] = *at.scale(in, s, u);
        }
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        if (!at.in(u)) continue;
        Unit<T, V> y;
#pragma unroll
        for (int j = 0; j < V; j += 2) y.template set_pair<true>(j, c[u].pair(j, scale_value(b[u])));
        y.store(at.wide(dst, u));
    }
}

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) silu_mul_pack_kernel(Rows<T> h, Packed gate_out, Packed up_out, Rows<const T> gate,
                                                                    Rows<const T> up, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s, kPassesSilu);
    Unit<T, V> g[kPassesSilu], u[kPassesSilu];
    pdl_wait();
#pragma unroll
    for (int k = 0; k < kPassesSilu; ++k) {
        g[k].clear();
        u[k].clear();
        if (at.in(k)) {
            g[k].load(at.wide(gate, k));
            u[k].load(at.wide(up, k));
        }
    }
#pragma unroll
    for (int k = 0; k < kPassesSilu; ++k) {
        if (at.in(k)) {
            Unit<T, V> out;
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const Pair x = g[k].pair(j);
                out.template set_pair<false>(j, x * sigmoid(x).s * u[k].pair(j));
            }
            out.store(at.wide(h, k));
        }
        pack_and_store(gate_out, s, at, k, g[k]);
        pack_and_store(up_out, s, at, k, u[k]);
    }
}

template <typename T, int V, bool AGAIN>
__global__ void __launch_bounds__(kMaxThreads) silu_mul_grad_kernel(Rows<T> dgate, Rows<T> dup, Rows<T> h, Rows<const T> dh, Packed gate,
                                                                    Packed up, Shape s) {
    pdl_launch_dependents();
    const Place<V> at(s, kPassesGrad);
    Unit<T, V> d[kPassesGrad];
    Codes<V> g[kPassesGrad], u[kPassesGrad];
    unsigned gb[kPassesGrad], ub[kPassesGrad];
    pdl_wait();
#pragma unroll
    for (int k = 0; k < kPassesGrad; ++k) {
        if (at.in(k)) {
            d[k].load(at.wide(dh, k));
            g[k].load(at.code(gate, s, k));
            u[k].load(at.code(up, s, k));
            gb[k] = *at.scale(gate, s, k);
            ub[k] = *at.scale(up, s, k);
        }
    }
#pragma unroll
    for (int k = 0; k < kPassesGrad; ++k) {
        if (!at.in(k)) continue;
        const float gs = scale_value(gb[k]), us = scale_value(ub[k]);
        Unit<T, V> dg, du, y;
#pragma unroll
        for (int j = 0; j < V; j += 2) {
            const Pair x = g[k].pair(j, gs), z = u[k].pair(j, us), dj = d[k].pair(j);
            const Sigmoid sg = sigmoid(x);
            const Pair silu = x * sg.s;
            du.template set_pair<false>(j, dj * silu);
            dg.template set_pair<false>(j, dj * z * fma2(silu, sg.q, sg.s));
            if constexpr (AGAIN) y.template set_pair<false>(j, silu * z);
        }
        du.store(at.wide(dup, k));
        dg.store(at.wide(dgate, k));
        if constexpr (AGAIN) y.store(at.wide(h, k));
    }
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
int launch_rows(void (*kernel)(KArgs...), int passes, const Shape &s, lcbStream stream, Args... args) {
    const uint64_t blocks = s.tiling.blocks(passes);
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
            return launch_rows(pack_kernel<T, v()>, kPasses, Shape::of(rows, cols, v()), stream, out, in);
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
            return launch_rows(unpack_kernel<T, v()>, kPasses, Shape::of(rows, cols, v()), stream, out, in);
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
            return launch_rows(silu_mul_pack_kernel<T, v()>, kPassesSilu, Shape::of(rows, cols, v()), stream, out, gp, upk, g, u);
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
            return launch_rows(h != nullptr ? silu_mul_grad_kernel<T, v(), true> : silu_mul_grad_kernel<T, v(), false>, kPassesGrad,
                               Shape::of(rows, cols, v()), stream, dg, du, out, d, gp, upk);
        });
    });
}
