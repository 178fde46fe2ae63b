// 8-bit activation checkpoints for sm_100a: packing and unpacking a matrix, and the gated unit gate * up / (1 +
// exp(-gate)) that leaves its checkpoint in the forward pass and reads it in the backward pass.
//
// What they compute (format and rounding: q8.cuh).  pack: codes and scales of every group.  unpack: code * s, rounded
// once. silu_mul_pack: h = g u s(g) with s(g) = 1 / (1 + exp(-g)), and g and u packed.  silu_mul_grad, with g and u
// the values of the packed pair: dup = dh g s(g), dgate = dh u s(g) (1 + g (1 - s(g))), and h again.
//
// What bounds them: HBM.  Every byte is moved once; per value of bf16 that is 3.03 bytes for pack and unpack, 8.06
// for the gated unit, 8.06 for its gradient, 10.06 with h again.  The arithmetic (about 7, 25 and 25 instructions per
// value, shared addresses counted) is the next limit, at 45-65 % of the issue slots, and what any form that spends
// more per value runs into first.  So a lane holds 16 values, 32-bit arithmetic goes two to an instruction,
// magnitudes are compared before they are converted, addresses are found once per lane, and all loads of a CTA are
// issued before its first store.  No tensor cores: there is no product.
//
// Measured on a B200 (bf16 unless said; share of 6548 GB/s, what a copy of the same bytes by torch reaches): pack
// 16384 x 8192 59 us, 105 %; unpack 61 us, 102 %; unpack 16400 x 5120 to f32 63.6 us, 101 %; gated unit 8192 x 10240
// 101 us, 102 %; its gradient with h again 125.5 us, 103 %, without 101 us.  Rows of 16-byte alignment: pack 16384 x
// 8200 67 us, 93 %.  Rows at any address: pack 16384 x 8191 101-104 us, unpack 88 us, gated unit 8192 x 10241 194 us,
// gradient 175 us: 53-70 %, held by two to three times the instructions and, but for unpack, by a third of the warps that an
// SM holds; f32 with 1001 columns: pack 32, unpack 29 of 23 us.  Small calls in a graph: unpack of a row 1.1 us, pack 129 x
// 1001 and the gated unit 7 x 1416 1.7, gradient 33 x 2731 3.0.  One lane per value instead of 16: pack 542 us, unpack to
// f32 339, gated unit 503, gradient 405.
#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

// Units in flight per lane, where there is work for that many.  Pack: 4 (59.1 us; 3 and 2 within 1 %, 1: 64).
// Unpack: 2 (60.9 us; 1: 69), in the warp form 1 (88 us at 16384 x 8191; 2 within 1 %).  Gated unit: 2 of each input
// (101 us; 1: 106), in the warp form 1, its registers held to 6 CTAs per SM (194 us at 8192 x 10241, 201 without that limit;
// 2: 226 and 236, whose loads no longer fit L1).  Gradient: 1, which already has three inputs in flight and three outputs to
// hold; 2 take 86 registers and 169 us against 125.
template <int A>
constexpr int kPassesPack = A >= 16 ? 4 : 2;
template <int A>
constexpr int kPassesUnpack = A == kWarp ? 1 : 2;
template <int A>
constexpr int kPassesSilu = A == kWarp ? 1 : 2;
constexpr int kPassesGrad = 1;
template <typename T>
struct Rows {  // rows of the wide type
    T *p;
    size_t stride;
};
struct Packed {
    uint8_t *codes, *scales;
};

// A matrix whose rows lie behind each other without a gap and end with whole groups is one long row, and so is a
// single row.  It is cut into lines of kMaxThreads units, which keeps every lane busy whatever the number of columns.
struct Shape {
    uint64_t rows, cols, groups;
    uint64_t flat;  // values of one long row, else 0
    Tiling tiling;
    template <int A>
    static Shape of(size_t rows, size_t cols, bool flat, int passes) {
        if (flat) {
            const uint64_t line = kMaxThreads * Form<A>::kValues, total = (uint64_t)rows * cols, lines = (total + line - 1) / line;
            return {lines, line, line / kGroup, total, Tiling::of(lines, kMaxThreads, passes)};
        }
        return {rows, cols, groups_of(cols), 0, Tiling::of(rows, units_of<A>(cols), passes)};
    }
};

// A lane's column and its rows, P passes of them.
template <int A, int P>
struct Place {
    uint64_t row, column;
    uint64_t code, scale;  // of the unit in the packed matrix
    uint32_t step;         // rows from pass to pass
    uint32_t live;         // passes in which this lane has a unit: the first ones
    int left, last;        // columns from the unit's first one on, and in the last live pass
    bool leads;            // its group, and so writes the scale
    __device__ __forceinline__ explicit Place(const Shape &s) {
        const Lane lane(s.tiling, blockIdx.x, P);
        row = lane.line;
        column = lane.unit * Form<A>::kValues;
        code = row * s.cols + column;
        scale = row * s.groups + lane.unit / Form<A>::kLanes;
        leads = lane.unit % Form<A>::kLanes == 0;
        step = s.tiling.side_by_side;
        const uint64_t end = s.flat != 0 ? s.flat : s.rows, at = s.flat != 0 ? code : row;
        const uint32_t rest = lane.in && column < s.cols && at < end ? (uint32_t)min(end - at, (uint64_t)INT32_MAX) : 0;
        const uint32_t stride = s.flat != 0 ? step * (uint32_t)s.cols : step;
        live = 0;
#pragma unroll
        for (uint32_t u = 0; u < P; ++u) live += u * stride < rest;
        left = last = (int)min(s.cols - column, (uint64_t)INT32_MAX);
        if (s.flat != 0 && live != 0) last = min(left, (int)(rest - (live - 1) * stride));
    }
    __device__ __forceinline__ int columns(uint32_t pass) const { return pass >= live ? 0 : pass + 1 == live ? last : left; }
    template <typename T>
    __device__ __forceinline__ T *wide(const Rows<T> &r) const { return r.p + (row * r.stride + column); }
};

template <typename T, int A, int P>
__device__ __forceinline__ void pack_and_store(const Packed &out, const Shape &s, const Place<A, P> &at, uint32_t pass, const Unit<T, A> &x) {
    Codes<A> c;
    const unsigned b = pack_unit(x, c);
    c.store(out.codes + at.code + pass * (at.step * s.cols), at.columns(pass));
    if (pass < at.live && at.leads) out.scales[at.scale + pass * (at.step * s.groups)] = (uint8_t)b;
}

template <typename T, int A, int P>
__global__ void __launch_bounds__(kMaxThreads) pack_kernel(Packed out, Rows<const T> src, Shape s) {
    pdl_launch_dependents();
    const Place<A, P> at(s);
    uint32_t *scratch = run_scratch<T, A>();
    const T *from = at.wide(src);
    Unit<T, A> x[P];
    pdl_wait();
#pragma unroll
    for (uint32_t u = 0; u < P; ++u) x[u].load(from + u * (at.step * src.stride), at.columns(u));
#pragma unroll
    for (uint32_t u = 0; u < P; ++u) {
        x[u].take(from + u * (at.step * src.stride), at.columns(u), scratch);
        pack_and_store(out, s, at, u, x[u]);
    }
}

template <typename T, int A, int P>
__global__ void __launch_bounds__(kMaxThreads) unpack_kernel(Rows<T> dst, Packed in, Shape s) {
    pdl_launch_dependents();
    const Place<A, P> at(s);
    uint32_t *scratch = run_scratch<T, A>();
    T *to = at.wide(dst);
    const uint8_t *codes = in.codes + at.code, *scales = in.scales + at.scale;
    Codes<A> c[P];
    unsigned b[P];
    pdl_wait();
#pragma unroll
    for (uint32_t u = 0; u < P; ++u) {
        c[u].load(codes + u * (at.step * s.cols), at.columns(u));
        b[u] = u < at.live ? scales[u * (at.step * s.groups)] : 0;
    }
#pragma unroll
    for (uint32_t u = 0; u < P; ++u) {
        if (A != kWarp && u >= at.live) break;
        const Pair scale(scale_value(b[u]));
        Unit<T, A> y;
#pragma unroll
        for (int j = 0; j < Form<A>::kValues; j += 2) y.template set_pair<true>(j, c[u].pair(j, scale));
        y.store(to + u * (at.step * dst.stride), at.columns(u), scratch);
    }
}

template <typename T, int A, int P>
__global__ void __launch_bounds__(kMaxThreads, A == kWarp ? 6 : 0) silu_mul_pack_kernel(Rows<T> h, Packed gate_out, Packed up_out, Rows<const T> gate,
                                                                    Rows<const T> up, Shape s) {
    pdl_launch_dependents();
    const Place<A, P> at(s);
    uint32_t *scratch = run_scratch<T, A>();
    const T *from_gate = at.wide(gate), *from_up = at.wide(up);
    T *to = at.wide(h);
    Unit<T, A> g[P], u[P];
    pdl_wait();
#pragma unroll
    for (uint32_t k = 0; k < P; ++k) {
        g[k].load(from_gate + k * (at.step * gate.stride), at.columns(k));
        u[k].load(from_up + k * (at.step * up.stride), at.columns(k));
    }
#pragma unroll
    for (uint32_t k = 0; k < P; ++k) {
        g[k].take(from_gate + k * (at.step * gate.stride), at.columns(k), scratch);
        u[k].take(from_up + k * (at.step * up.stride), at.columns(k), scratch);
        if (A == kWarp || k < at.live) {
            Unit<T, A> out;
#pragma unroll
            for (int j = 0; j < Form<A>::kValues; j += 2) {
                const Pair x = g[k].pair(j);
                out.template set_pair<false>(j, x * sigmoid<false>(x).s * u[k].pair(j));
            }
            out.store(to + k * (at.step * h.stride), at.columns(k), scratch);
        }
        pack_and_store(gate_out, s, at, k, g[k]);
        pack_and_store(up_out, s, at, k, u[k]);
    }
}

template <typename T, int A, bool AGAIN>
__global__ void __launch_bounds__(kMaxThreads) silu_mul_grad_kernel(Rows<T> dgate, Rows<T> dup, Rows<T> h, Rows<const T> dh, Packed gate,
                                                                    Packed up, Shape s) {
    pdl_launch_dependents();
    const Place<A, 1> at(s);
    uint32_t *scratch = run_scratch<T, A>();
    pdl_wait();
    if (A != kWarp && at.live == 0) return;
    const int left = at.columns(0);
    Unit<T, A> d;
    Codes<A> g, u;
    d.load(at.wide(dh), left);
    g.load(gate.codes + at.code, left);
    u.load(up.codes + at.code, left);
    const Pair gs(scale_value(left > 0 ? gate.scales[at.scale] : 0u)), us(scale_value(left > 0 ? up.scales[at.scale] : 0u));
    d.take(at.wide(dh), left, scratch);
    Unit<T, A> dg, du, y;
#pragma unroll
    for (int j = 0; j < Form<A>::kValues; j += 2) {
        const Pair x = g.pair(j, gs), z = u.pair(j, us), dj = d.pair(j);
        const Sigmoid sg = sigmoid<true>(x);
        const Pair silu = x * sg.s;
        du.template set_pair<false>(j, dj * silu);
        dg.template set_pair<false>(j, dj * z * fma2(silu, sg.q, sg.s));
        if constexpr (AGAIN) y.template set_pair<false>(j, silu * z);
    }
    du.store(at.wide(dup), left, scratch);
    dg.store(at.wide(dgate), left, scratch);
    if constexpr (AGAIN) y.store(at.wide(h), left, scratch);
}

// The widest accesses that are aligned in every row.  A row's codes lie behind each other, so the columns must be a
// multiple of what an access covers.
struct Fit {
    size_t rows, cols;
    bool flat;
    uint64_t wide = 0, codes = 0;
    Fit(size_t rows, size_t cols) : rows(rows), cols(cols), flat(rows == 1 || cols % kGroup == 0) {}
    template <typename T>
    void add(const Rows<T> &r) {
        if (r.p == nullptr) return;
        wide |= reinterpret_cast<uintptr_t>(r.p) | (rows > 1 ? r.stride * sizeof(T) : 0);
        if (rows > 1 && r.stride != cols) flat = false;
    }
    void add(const Packed &p) { codes |= reinterpret_cast<uintptr_t>(p.codes); }
    template <typename T>
    int access(RowOp op) const {
        if (cols % 16 == 0 && wide % 32 == 0 && codes % 16 == 0) return 32;
        if (cols % 8 == 0 && wide % 16 == 0 && codes % 8 == 0) return 16;
        return flat || warp_form_pays(op, sizeof(T) == 4, cols) ? kWarp : 0;
    }
    // one long row is addressed in lines that lie behind each other
    template <typename T>
    Rows<T> lines(const Rows<T> &r, const Shape &s) const { return {r.p, flat ? (size_t)s.cols : r.stride}; }
};

// A single row whose number of columns is no multiple of a group is done in two parts, so that the last group does not
// decide how all the others are read.  part(first column, columns)
template <typename Part>
int in_parts(size_t rows, size_t cols, Part part) {
    const size_t body = cols / kGroup * kGroup;
    if (rows != 1 || body == cols || body == 0) return part(0, cols);
    const int rc = part(0, body);
    return rc != 0 ? rc : part(body, cols - body);
}

template <typename... KArgs, typename... Args>
int launch_rows(void (*kernel)(KArgs...), const Shape &s, lcbStream stream, Args... args) {
    const uint64_t blocks = s.tiling.blocks();
    if (blocks > kMostBlocks) return 1;
    return launch_kernel(kernel, (unsigned)blocks, s.tiling.threads, 0, static_cast<cudaStream_t>(stream), args..., s);
}

Packed packed(const void *codes, const void *scales) {
    return {static_cast<uint8_t *>(const_cast<void *>(codes)), static_cast<uint8_t *>(const_cast<void *>(scales))};
}
Packed from(const Packed &p, size_t column) { return {p.codes + column, p.scales + column / kGroup}; }
template <typename T, typename P>
Rows<T> rows_at(P *p, size_t stride, size_t column) { return {p != nullptr ? static_cast<T *>(p) + column : nullptr, stride}; }

template <typename T, int A>
int load_pack_kernels() { return first_error({load_kernel(pack_kernel<T, A, 1>), load_kernel(pack_kernel<T, A, kPassesPack<A>>)}); }
template <typename T, int A>
int load_storing_kernels() {
    return first_error({load_kernel(unpack_kernel<T, A, 1>), load_kernel(unpack_kernel<T, A, kPassesUnpack<A>>),
                        load_kernel(silu_mul_pack_kernel<T, A, 1>), load_kernel(silu_mul_pack_kernel<T, A, kPassesSilu<A>>),
                        load_kernel(silu_mul_grad_kernel<T, A, false>), load_kernel(silu_mul_grad_kernel<T, A, true>)});
}
template <typename T>
int load_row_kernels() {
    constexpr bool f32 = sizeof(T) == 4;
    return first_error({load_pack_kernels<T, 32>(), load_pack_kernels<T, 16>(), load_pack_kernels<T, kWarp>(),
                        load_pack_kernels<T, loose_form(RowOp::Pack, f32)>(), load_storing_kernels<T, 32>(), load_storing_kernels<T, 16>(),
                        load_storing_kernels<T, kWarp>(), load_storing_kernels<T, loose_form(RowOp::Unpack, f32)>()});
}

}  // namespace

int preload_q8_row_kernels() { return first_error({load_row_kernels<float>(), load_row_kernels<__half>(), load_row_kernels<__nv_bfloat16>()}); }
}  // namespace lcb

using namespace lcb;

extern "C" int lcb_pack_q8(void *codes, void *scales, const void *src, size_t src_stride, int type, size_t rows, size_t cols,
                           lcbStream stream) {
    if (!pack_ok(codes, scales, src, src_stride, type, rows, cols, false)) return 1;
    if (rows == 0 || cols == 0) return 0;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return in_parts(rows, cols, [&](size_t column, size_t n) {
            const auto in = rows_at<const T>(src, src_stride, column);
            const Packed out = from(packed(codes, scales), column);
            Fit fit(rows, n);
            fit.add(in);
            fit.add(out);
            return with_access<loose_form(RowOp::Pack, sizeof(T) == 4), true>(fit.template access<T>(RowOp::Pack), [&](auto a) {
                const Shape s = Shape::of<a()>(rows, n, fit.flat, kPassesPack<a()>);
                return with_passes<kPassesPack<a()>>(s.tiling.passes, [&](auto p) {
                    return launch_rows(pack_kernel<T, a(), p()>, s, stream, out, fit.lines(in, s));
                });
            });
        });
    });
}

extern "C" int lcb_unpack_q8(void *dst, size_t dst_stride, int type, const void *codes, const void *scales, size_t rows, size_t cols,
                             lcbStream stream) {
    if (!pack_ok(codes, scales, dst, dst_stride, type, rows, cols, true)) return 1;
    if (rows == 0 || cols == 0) return 0;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return in_parts(rows, cols, [&](size_t column, size_t n) {
            const auto out = rows_at<T>(dst, dst_stride, column);
            const Packed in = from(packed(codes, scales), column);
            Fit fit(rows, n);
            fit.add(out);
            fit.add(in);
            return with_access<loose_form(RowOp::Unpack, sizeof(T) == 4), true>(fit.template access<T>(RowOp::Unpack), [&](auto a) {
                const Shape s = Shape::of<a()>(rows, n, fit.flat, kPassesUnpack<a()>);
                return with_passes<kPassesUnpack<a()>>(s.tiling.passes, [&](auto p) {
                    return launch_rows(unpack_kernel<T, a(), p()>, s, stream, fit.lines(out, s), in);
                });
            });
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
        return in_parts(rows, cols, [&](size_t column, size_t n) {
            const auto out = rows_at<T>(h, h_stride, column);
            const auto g = rows_at<const T>(gate, gate_stride, column), u = rows_at<const T>(up, up_stride, column);
            const Packed gp = from(packed(gate_codes, gate_scales), column), upk = from(packed(up_codes, up_scales), column);
            Fit fit(rows, n);
            fit.add(out);
            fit.add(g);
            fit.add(u);
            fit.add(gp);
            fit.add(upk);
            return with_access<loose_form(RowOp::Unit, sizeof(T) == 4), true>(fit.template access<T>(RowOp::Unit), [&](auto a) {
                const Shape s = Shape::of<a()>(rows, n, fit.flat, kPassesSilu<a()>);
                return with_passes<kPassesSilu<a()>>(s.tiling.passes, [&](auto p) {
                    return launch_rows(silu_mul_pack_kernel<T, a(), p()>, s, stream, fit.lines(out, s), gp, upk, fit.lines(g, s), fit.lines(u, s));
                });
            });
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
        return in_parts(rows, cols, [&](size_t column, size_t n) {
            const auto dg = rows_at<T>(dgate, dgate_stride, column), du = rows_at<T>(dup, dup_stride, column), out = rows_at<T>(h, h_stride, column);
            const auto d = rows_at<const T>(dh, dh_stride, column);
            const Packed gp = from(packed(gate_codes, gate_scales), column), upk = from(packed(up_codes, up_scales), column);
            Fit fit(rows, n);
            fit.add(dg);
            fit.add(du);
            fit.add(out);
            fit.add(d);
            fit.add(gp);
            fit.add(upk);
            return with_access<loose_form(RowOp::Gradient, sizeof(T) == 4), true>(fit.template access<T>(RowOp::Gradient), [&](auto a) {
                const Shape s = Shape::of<a()>(rows, n, fit.flat, kPassesGrad);
                return launch_rows(h != nullptr ? silu_mul_grad_kernel<T, a(), true> : silu_mul_grad_kernel<T, a(), false>, s, stream,
                                   fit.lines(dg, s), fit.lines(du, s), fit.lines(out, s), fit.lines(d, s), gp, upk);
            });
        });
    });
}
