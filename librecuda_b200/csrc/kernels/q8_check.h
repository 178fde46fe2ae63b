// Argument checks of the 8-bit operators, shared by the kernel launchers (which return 1) and by the stream layer
// (which refuses a call when it is recorded, not when it is submitted).  Host code without CUDA calls.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <initializer_list>

#include "lcb200_types.h"
#include "q8_tiling.h"

namespace lcb {

inline size_t type_size(int type) { return type == LCB_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type == LCB_F32 || type == LCB_F16 || type == LCB_BF16; }
inline size_t groups_of(size_t n) { return n / 32 + (n % 32 != 0); }
inline bool aligned(const void *p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// Bytes from the first to behind the last element of outer x inner rows of n elements; 0 where that does not fit
// 62 bits.  Empty shapes have 0 bytes too; the callers have dealt with them before.
inline size_t span_bytes(size_t outer, size_t outer_stride, size_t inner, size_t inner_stride, size_t n, size_t size) {
    if (outer == 0 || inner == 0 || n == 0) return 0;
    size_t a, b, s;
    if (__builtin_mul_overflow(outer - 1, outer_stride, &a) || __builtin_mul_overflow(inner - 1, inner_stride, &b)) return 0;
    if (__builtin_add_overflow(a, b, &s) || __builtin_add_overflow(s, n, &s) || __builtin_mul_overflow(s, size, &s)) return 0;
    return s >> 62 ? 0 : s;
}
inline bool product_ok(size_t a, size_t b, size_t c, size_t d) {  // a * b * c * d below 2^62
    size_t p;
    return !__builtin_mul_overflow(a, b, &p) && !__builtin_mul_overflow(p, c, &p) && !__builtin_mul_overflow(p, d, &p) && !(p >> 62);
}

// outputs that begin at the same address write over each other (NULL: left out)
inline bool apart(std::initializer_list<const void *> outputs) {
    for (auto a = outputs.begin(); a != outputs.end(); ++a)
        for (auto b = a + 1; b != outputs.end(); ++b)
            if (*a != nullptr && *a == *b) return false;
    return true;
}
// rows of an output: none may overlap another
inline bool rows_apart(size_t rows, size_t stride, size_t cols) { return rows <= 1 || stride >= cols; }
// the same for rows (t, h), whichever of the two is the outer dimension
inline bool heads_apart(size_t tokens, size_t token_stride, size_t heads, size_t head_stride, size_t dim) {
    if (tokens <= 1) return rows_apart(heads, head_stride, dim);
    if (heads <= 1) return rows_apart(tokens, token_stride, dim);
    const size_t across_heads = span_bytes(1, 0, heads, head_stride, dim, 1);
    const size_t across_tokens = span_bytes(1, 0, tokens, token_stride, dim, 1);
    return (head_stride >= dim && across_heads != 0 && token_stride >= across_heads) ||
           (token_stride >= dim && across_tokens != 0 && head_stride >= across_tokens);
}

inline bool wide_matrix_ok(const void *p, size_t stride, int type, size_t rows, size_t cols, bool output) {
    return p != nullptr && aligned(p, type_size(type)) && span_bytes(rows, rows > 1 ? stride : 0, 1, 0, cols, type_size(type)) != 0 &&
           (!output || rows_apart(rows, stride, cols));
}
inline bool packed_matrix_ok(const void *codes, const void *scales, size_t rows, size_t cols) {
    return codes != nullptr && scales != nullptr && cols < SIZE_MAX - 31 && product_ok(rows, groups_of(cols), 32, 1);
}
// A grid has at most 2^31 - 1 CTAs.  The form with the fewest values per lane and one pass has the most.
constexpr uint64_t kMostBlocks = 0x7fffffffu;
inline bool grid_ok(size_t rows, size_t cols, int type) {
    return (type == LCB_F32 ? Tiling::of(rows, units_of<kLooseTiny>(cols), 1) : Tiling::of(rows, units_of<kLooseShort>(cols), 1)).blocks() <= kMostBlocks;
}

inline bool pack_ok(const void *codes, const void *scales, const void *wide, size_t stride, int type, size_t rows, size_t cols, bool wide_is_output) {
    if (!type_ok(type)) return false;
    if (rows == 0 || cols == 0) return true;
    return codes != scales && codes != wide && scales != wide && packed_matrix_ok(codes, scales, rows, cols) &&
           grid_ok(rows, cols, type) && wide_matrix_ok(wide, stride, type, rows, cols, wide_is_output);
}

inline bool silu_pack_ok(const void *h, size_t h_stride, const void *gate_codes, const void *gate_scales, const void *up_codes, const void *up_scales,
                         const void *gate, size_t gate_stride, const void *up, size_t up_stride, int type, size_t rows, size_t cols) {
    if (!type_ok(type)) return false;
    if (rows == 0 || cols == 0) return true;
    return apart({h, gate_codes, gate_scales, up_codes, up_scales}) && packed_matrix_ok(gate_codes, gate_scales, rows, cols) &&
           packed_matrix_ok(up_codes, up_scales, rows, cols) && grid_ok(rows, cols, type) && wide_matrix_ok(h, h_stride, type, rows, cols, true) &&
           wide_matrix_ok(gate, gate_stride, type, rows, cols, false) &&
           wide_matrix_ok(up, up_stride, type, rows, cols, false);
}
inline bool silu_grad_ok(const void *dgate, size_t dgate_stride, const void *dup, size_t dup_stride, const void *h, size_t h_stride, const void *dh,
                         size_t dh_stride, const void *gate_codes, const void *gate_scales, const void *up_codes, const void *up_scales, int type,
                         size_t rows, size_t cols) {
    if (!type_ok(type)) return false;
    if (rows == 0 || cols == 0) return true;
    return apart({dgate, dup, h}) && packed_matrix_ok(gate_codes, gate_scales, rows, cols) && packed_matrix_ok(up_codes, up_scales, rows, cols) &&
           grid_ok(rows, cols, type) && wide_matrix_ok(dgate, dgate_stride, type, rows, cols, true) && wide_matrix_ok(dup, dup_stride, type, rows, cols, true) &&
           (h == nullptr || wide_matrix_ok(h, h_stride, type, rows, cols, true)) && wide_matrix_ok(dh, dh_stride, type, rows, cols, false);
}

inline bool cache_ok(const lcbCacheQ8 *c) {
    if (c == nullptr || (c->order != LCB_CACHE_TOKENS_FIRST && c->order != LCB_CACHE_HEADS_FIRST)) return false;
    if (c->pages == 0 || c->page_tokens == 0 || c->heads == 0 || c->k_dim == 0) return false;
    if (c->k_codes == nullptr || c->k_scales == nullptr) return false;
    const bool two = c->v_dim != 0;
    if ((c->v_codes != nullptr) != two || (c->v_scales != nullptr) != two) return false;
    size_t slots;
    if (__builtin_mul_overflow(c->pages, c->page_tokens, &slots) || (slots >> 62)) return false;
    // a token's rows together stay below 2^31 values, padded, and a page below 2^31 tokens: both are 32-bit numbers
    if (c->page_tokens > (size_t)INT32_MAX) return false;
    for (size_t dim : {c->k_dim, c->v_dim})
        if (dim > (size_t)INT32_MAX - 31 || c->heads > ((size_t)1 << 31) / 32 / (groups_of(dim) + 1)) return false;
    return product_ok(slots, c->heads, groups_of(c->k_dim), 32) &&
           product_ok(slots, c->heads, groups_of(c->v_dim), 32);
}
inline size_t cache_codes_bytes(const lcbCacheQ8 &c, size_t dim) { return c.pages * c.page_tokens * c.heads * dim; }
inline size_t cache_scales_bytes(const lcbCacheQ8 &c, size_t dim) { return c.pages * c.page_tokens * c.heads * groups_of(dim); }

// the wide side of a cache operator: `tokens` rows per head
inline bool cache_rows_ok(const lcbCacheQ8 &c, const void *k, size_t kts, size_t khs, const void *v, size_t vts, size_t vhs, int type,
                          size_t tokens, bool output) {
    if (!type_ok(type)) return false;
    const size_t e = type_size(type);
    auto side = [&](const void *p, size_t ts, size_t hs, size_t dim) {
        return p != nullptr && aligned(p, e) && product_ok(tokens, c.heads, groups_of(dim), 32) &&
               span_bytes(tokens, tokens > 1 ? ts : 0, c.heads, c.heads > 1 ? hs : 0, dim, e) != 0 &&
               (!output || heads_apart(tokens, ts, c.heads, hs, dim));
    };
    return side(k, kts, khs, c.k_dim) && (c.v_dim == 0 || side(v, vts, vhs, c.v_dim));
}
// CTAs of one line of heads in the form with the fewest values per lane that the operator takes, keys and values
template <int A>
uint64_t most_parts(const lcbCacheQ8 &c) {
    uint64_t parts = 0;
    for (size_t dim : {c.k_dim, c.v_dim})
        if (dim != 0) parts += Tiling::of(1, c.heads * units_of<A>(dim), 1).by_chunks.d;
    return parts;
}
// a write: a CTA takes at least one token of a part
template <int A>
uint64_t most_write_blocks(const lcbCacheQ8 &c, size_t tokens) {
    uint64_t blocks = 0;
    for (size_t dim : {c.k_dim, c.v_dim})
        if (dim != 0) blocks += Tiling::of(tokens, c.heads * units_of<A>(dim), 1).blocks();
    return blocks;
}
inline bool cache_write_ok(const lcbCacheQ8 *c, const void *k, size_t kts, size_t khs, const void *v, size_t vts, size_t vhs, int type,
                           const int64_t *slots, size_t tokens) {
    if (!cache_ok(c) || !type_ok(type)) return false;
    if (tokens == 0) return true;
    return apart({c->k_codes, c->k_scales, c->v_codes, c->v_scales}) && slots != nullptr && aligned(slots, 8) &&
           cache_rows_ok(*c, k, kts, khs, v, vts, vhs, type, tokens, false) &&
           (type == LCB_F32 ? most_write_blocks<kLooseShort>(*c, tokens) : most_write_blocks<kLoose>(*c, tokens)) <= kMostBlocks;
}
inline bool cache_read_ok(const lcbCacheQ8 *c, const void *k, size_t kts, size_t khs, const void *v, size_t vts, size_t vhs, int type,
                          const int32_t *table, size_t table_stride, const int32_t *lengths, const int64_t *first_rows, size_t sequences,
                          size_t max_length, size_t rows) {
    if (!cache_ok(c) || !type_ok(type)) return false;
    if (sequences == 0 || max_length == 0) return true;
    size_t reach, entries;
    if (__builtin_mul_overflow(table_stride, c->page_tokens, &reach)) reach = SIZE_MAX;
    if (max_length > reach || max_length > (size_t)INT32_MAX || c->pages > (size_t)INT32_MAX) return false;
    if (__builtin_mul_overflow(sequences, table_stride, &entries) || (entries >> 60)) return false;
    if (table == nullptr || lengths == nullptr || first_rows == nullptr) return false;
    if (!aligned(table, 4) || !aligned(lengths, 4) || !aligned(first_rows, 8) || (rows >> 62)) return false;
    return product_ok(sequences, max_length, c->heads, groups_of(c->k_dim) * 32) &&
           product_ok(sequences, max_length, c->heads, groups_of(c->v_dim) * 32) &&
           (c->v_dim == 0 || apart({k, v})) && cache_rows_ok(*c, k, kts, khs, v, vts, vhs, type, rows, true) &&
           sequences <= (kMostBlocks - (1u << 20)) / most_parts<kLooseShort>(*c);  // the launcher shares the tokens out among 2^20 CTAs
}

}  // namespace lcb
