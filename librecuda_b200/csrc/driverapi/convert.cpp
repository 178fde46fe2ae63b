// The 8-bit operators as stream operations: quantising copies into and out of a paged cache, packing and unpacking of
// matrices, and the gated unit with its 8-bit checkpoint.  A call is checked when it is recorded, with the checks of
// the kernel layer and the stream layer's own rules for pointers, and launched by Commence like every other
// operation. The reference has no operation that changes a number format (driverapi/include/librecuda.h:37-114).
#include <initializer_list>

#include "internal.h"
#include "q8_check.h"

using namespace lcu;

namespace {

// An operand: device memory that the stream's GPU may access (NULL where an operand is optional and left out).
struct Operand {
    const void *p;
    size_t bytes;   // from its first to behind its last byte
    bool written;
};

libreCudaStatus_t record_convert(LibreCUstream stream, bool async, std::initializer_list<Operand> operands, std::function<int(cudaStream_t)> enqueue) {
    Command c;
    c.kind = Command::Convert;
    c.async = async;
    for (const Operand &o : operands) {
        if (o.p == nullptr) continue;
        LIBRECUDA_VALIDATE(classify(o.p) == PtrClass::Device, LIBRECUDA_ERROR_INVALID_VALUE);
        const int owner = owner_device(o.p);  // same rule as for kernel copies
        LIBRECUDA_VALIDATE(owner < 0 || stream->ctx->peers.count(owner) != 0, LIBRECUDA_ERROR_INVALID_VALUE);
        if (o.written) c.writes.emplace_back(o.p, o.bytes);
    }
    c.enqueue = std::move(enqueue);
    return record(stream, std::move(c));
}

Operand wide(const void *p, size_t stride, int type, size_t rows, size_t cols, bool written) {
    return {p, lcb::span_bytes(rows, rows > 1 ? stride : 0, 1, 0, cols, lcb::type_size(type)), written};
}
Operand codes(const void *p, size_t rows, size_t cols, bool written) { return {p, rows * cols, written}; }
Operand scales(const void *p, size_t rows, size_t cols, bool written) { return {p, rows * lcb::groups_of(cols), written}; }

}  // namespace

libreCudaStatus_t libreCuPackQ8(void *pCodes, void *pScales, const void *src, size_t srcStride, int type, size_t rows, size_t cols,
                                LibreCUstream stream, bool async) {
    return lcu_guarded([&]() -> libreCudaStatus_t {
        LIBRECUDA_VALIDATE(stream != nullptr, LIBRECUDA_ERROR_INVALID_VALUE);
        LCU_ENSURE_CTX();
        LIBRECUDA_VALIDATE(lcb::pack_ok(pCodes, pScales, src, srcStride, type, rows, cols, false), LIBRECUDA_ERROR_INVALID_VALUE);
        if (rows == 0 || cols == 0) LIBRECUDA_SUCCEED();
        return record_convert(stream, async,
                              {codes(pCodes, rows, cols, true), scales(pScales, rows, cols, true), wide(src, srcStride, type, rows, cols, false)},
                              [=](cudaStream_t s) { return lcb_pack_q8(pCodes, pScales, src, srcStride, type, rows, cols, s); });
    });
}

libreCudaStatus_t libreCuUnpackQ8(void *dst, size_t dstStride, int type, const void *pCodes, const void *pScales, size_t rows, size_t cols,
                                  LibreCUstream stream, bool async) {
    return lcu_guarded([&]() -> libreCudaStatus_t {
        LIBRECUDA_VALIDATE(stream != nullptr, LIBRECUDA_ERROR_INVALID_VALUE);
        LCU_ENSURE_CTX();
        LIBRECUDA_VALIDATE(lcb::pack_ok(pCodes, pScales, dst, dstStride, type, rows, cols, true), LIBRECUDA_ERROR_INVALID_VALUE);
        if (rows == 0 || cols == 0) LIBRECUDA_SUCCEED();
        return record_convert(stream, async,
                              {wide(dst, dstStride, type, rows, cols, true), codes(pCodes, rows, cols, false), scales(pScales, rows, cols, false)},
                              [=](cudaStream_t s) { return lcb_unpack_q8(dst, dstStride, type, pCodes, pScales, rows, cols, s); });
    });
}

libreCudaStatus_t libreCuSiluMulPackQ8(void *h, size_t hStride, void *gateCodes, void *gateScales, void *upCodes, void *upScales, const void *gate,
                                       size_t gateStride, const void *up, size_t upStride, int type, size_t rows, size_t cols,
                                       LibreCUstream stream, bool async) {
    return lcu_guarded([&]() -> libreCudaStatus_t {
        LIBRECUDA_VALIDATE(stream != nullptr, LIBRECUDA_ERROR_INVALID_VALUE);
        LCU_ENSURE_CTX();
        LIBRECUDA_VALIDATE(lcb::silu_pack_ok(h, hStride, gateCodes, gateScales, upCodes, upScales, gate, gateStride, up, upStride, type, rows, cols),
                           LIBRECUDA_ERROR_INVALID_VALUE);
        if (rows == 0 || cols == 0) LIBRECUDA_SUCCEED();
        return record_convert(stream, async,
                              {wide(h, hStride, type, rows, cols, true), codes(gateCodes, rows, cols, true), scales(gateScales, rows, cols, true),
                               codes(upCodes, rows, cols, true), scales(upScales, rows, cols, true), wide(gate, gateStride, type, rows, cols, false),
                               wide(up, upStride, type, rows, cols, false)},
                              [=](cudaStream_t s) {
                                  return lcb_silu_mul_pack_q8(h, hStride, gateCodes, gateScales, upCodes, upScales, gate, gateStride, up, upStride, type,
                                                              rows, cols, s);
                              });
    });
}

libreCudaStatus_t libreCuSiluMulGradQ8(void *dGate, size_t dGateStride, void *dUp, size_t dUpStride, void *h, size_t hStride, const void *dH,
                                       size_t dHStride, const void *gateCodes, const void *gateScales, const void *upCodes, const void *upScales,
                                       int type, size_t rows, size_t cols, LibreCUstream stream, bool async) {
    return lcu_guarded([&]() -> libreCudaStatus_t {
        LIBRECUDA_VALIDATE(stream != nullptr, LIBRECUDA_ERROR_INVALID_VALUE);
        LCU_ENSURE_CTX();
        LIBRECUDA_VALIDATE(lcb::silu_grad_ok(dGate, dGateStride, dUp, dUpStride, h, hStride, dH, dHStride, gateCodes, gateScales, upCodes, upScales,
                                             type, rows, cols),
                           LIBRECUDA_ERROR_INVALID_VALUE);
        if (rows == 0 || cols == 0) LIBRECUDA_SUCCEED();
        return record_convert(stream, async,
                              {wide(dGate, dGateStride, type, rows, cols, true), wide(dUp, dUpStride, type, rows, cols, true),
                               wide(h, hStride, type, rows, cols, true), wide(dH, dHStride, type, rows, cols, false), codes(gateCodes, rows, cols, false),
                               scales(gateScales, rows, cols, false), codes(upCodes, rows, cols, false), scales(upScales, rows, cols, false)},
                              [=](cudaStream_t s) {
                                  return lcb_silu_mul_grad_q8(dGate, dGateStride, dUp, dUpStride, h, hStride, dH, dHStride, gateCodes, gateScales,
                                                              upCodes, upScales, type, rows, cols, s);
                              });
    });
}

libreCudaStatus_t libreCuCacheWriteQ8(const lcbCacheQ8 *cache, const void *k, size_t kTokenStride, size_t kHeadStride, const void *v,
                                      size_t vTokenStride, size_t vHeadStride, int type, const int64_t *slots, size_t tokens,
                                      LibreCUstream stream, bool async) {
    return lcu_guarded([&]() -> libreCudaStatus_t {
        LIBRECUDA_VALIDATE(stream != nullptr, LIBRECUDA_ERROR_INVALID_VALUE);
        LCU_ENSURE_CTX();
        LIBRECUDA_VALIDATE(lcb::cache_write_ok(cache, k, kTokenStride, kHeadStride, v, vTokenStride, vHeadStride, type, slots, tokens),
                           LIBRECUDA_ERROR_INVALID_VALUE);
        if (tokens == 0) LIBRECUDA_SUCCEED();
        const lcbCacheQ8 c = *cache;  // the caller's descriptor may be gone when the stream commences
        const size_t slots_total = c.pages * c.page_tokens * c.heads;
        return record_convert(stream, async,
                              {codes(c.k_codes, slots_total, c.k_dim, true), scales(c.k_scales, slots_total, c.k_dim, true),
                               codes(c.v_codes, slots_total, c.v_dim, true), scales(c.v_scales, slots_total, c.v_dim, true),
                               {k, 0, false}, {c.v_dim != 0 ? v : nullptr, 0, false}, {slots, 0, false}},
                              [=](cudaStream_t s) {
                                  return lcb_cache_write_q8(&c, k, kTokenStride, kHeadStride, v, vTokenStride, vHeadStride, type, slots, tokens, s);
                              });
    });
}

libreCudaStatus_t libreCuCacheReadQ8(const lcbCacheQ8 *cache, void *k, size_t kTokenStride, size_t kHeadStride, void *v, size_t vTokenStride,
                                     size_t vHeadStride, int type, const int32_t *pageTable, size_t tableStride, const int32_t *lengths,
                                     const int64_t *firstRows, size_t sequences, size_t maxLength, size_t rows, LibreCUstream stream,
                                     bool async) {
    return lcu_guarded([&]() -> libreCudaStatus_t {
        LIBRECUDA_VALIDATE(stream != nullptr, LIBRECUDA_ERROR_INVALID_VALUE);
        LCU_ENSURE_CTX();
        LIBRECUDA_VALIDATE(lcb::cache_read_ok(cache, k, kTokenStride, kHeadStride, v, vTokenStride, vHeadStride, type, pageTable, tableStride, lengths,
                                              firstRows, sequences, maxLength, rows),
                           LIBRECUDA_ERROR_INVALID_VALUE);
        if (sequences == 0 || maxLength == 0) LIBRECUDA_SUCCEED();
        const lcbCacheQ8 c = *cache;
        const size_t e = lcb::type_size(type);
        auto out = [&](const void *p, size_t token_stride, size_t head_stride, size_t dim) -> Operand {
            return {dim != 0 ? p : nullptr, lcb::span_bytes(rows, rows > 1 ? token_stride : 0, c.heads, c.heads > 1 ? head_stride : 0, dim, e), true};
        };
        return record_convert(stream, async,
                              {out(k, kTokenStride, kHeadStride, c.k_dim), out(v, vTokenStride, vHeadStride, c.v_dim), {c.k_codes, 0, false},
                               {c.k_scales, 0, false}, {c.v_codes, 0, false}, {c.v_scales, 0, false}, {pageTable, 0, false}, {lengths, 0, false},
                               {firstRows, 0, false}},
                              [=](cudaStream_t s) {
                                  return lcb_cache_read_q8(&c, k, kTokenStride, kHeadStride, v, vTokenStride, vHeadStride, type, pageTable, tableStride,
                                                           lengths, firstRows, sequences, maxLength, rows, s);
                              });
    });
}
