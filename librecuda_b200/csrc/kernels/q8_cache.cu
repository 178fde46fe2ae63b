// Paged key/value cache in the 8-bit row format for sm_100a: quantising rows as they are written to their slots, and
// reading sequences back through a page table.
//
// One lane per value, one warp per group, as in q8_rows.cu.  Every index that comes from device memory (slots, pages,
// lengths, first rows) is checked before it forms an address.
#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

constexpr int kThreads = 256;

template <typename T>
struct Side {  // keys or values
    T *wide;
    uint64_t token_stride, head_stride;
    uint8_t *codes, *scales;
    uint64_t dim, groups;
    FastDiv per_head;   // by the lanes of a row, padded to whole groups
    uint64_t blocks;    // of the grid (write), or of one sequence (read)
};

struct Pool {
    uint64_t pages, heads;
    FastDiv page_tokens, by_heads;
    int heads_first;
    // row of (page, offset in the page, head)
    __device__ __forceinline__ uint64_t row(uint64_t page, uint64_t offset, uint64_t head) const {
        return heads_first ? (page * heads + head) * page_tokens.d + offset : (page * page_tokens.d + offset) * heads + head;
    }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(Side<const T> k, Side<const T> v, Pool pool, const int64_t *slots,
                                                               uint64_t tokens, ErrorSink errors) {
    pdl_launch_dependents();
    pdl_wait();
    const bool first = blockIdx.x < k.blocks;
    const Side<const T> &s = first ? k : v;
    const uint64_t i = (blockIdx.x - (first ? 0 : k.blocks)) * kThreads + threadIdx.x;
    uint64_t col, head;
    const uint64_t token = pool.by_heads.divmod(s.per_head.divmod(i, col), head);
    if (token >= tokens) return;  // the same for all lanes of a warp
    const int64_t slot = slots[token];
    if (slot < 0) return;
    uint64_t offset;
    const uint64_t page = pool.page_tokens.divmod((uint64_t)slot, offset);
    if (page >= pool.pages) {
        if (col == 0 && head == 0) raise_error(errors, kErrIndexRange);
        return;
    }
    const bool in = col < s.dim;
    const float x = in ? to_f32(s.wide[token * s.token_stride + head * s.head_stride + col]) : 0.0f;
    const unsigned top = __reduce_max_sync(0xffffffffu, in ? finite_magnitude(x) : 0u);
    const int b = scale_byte(top);
    if (!in) return;
    const uint64_t row = pool.row(page, offset, head);
    s.codes[row * s.dim + col] = (uint8_t)to_codes(nan_if_infinite(x) * scale_inverse(b), 0.0f);
    if ((col & (kGroup - 1)) == 0) s.scales[row * s.groups + col / kGroup] = (uint8_t)b;
}

struct Sequences {
    const int32_t *table, *lengths;
    const int64_t *first_rows;
    uint64_t table_stride, max_length, rows;
    FastDiv blocks;  // of one sequence, keys and values
};

template <typename T>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(Side<T> k, Side<T> v, Pool pool, Sequences q, ErrorSink errors) {
    pdl_launch_dependents();
    pdl_wait();
    uint64_t block;
    const uint64_t b = q.blocks.divmod(blockIdx.x, block);
    const bool first = block < k.blocks;
    const Side<T> &s = first ? k : v;
    const uint64_t i = (block - (first ? 0 : k.blocks)) * kThreads + threadIdx.x;
    const int32_t length = q.lengths[b];
    if (block == 0 && threadIdx.x == 0 && (length < 0 || length > (int64_t)q.max_length)) raise_error(errors, kErrIndexRange);
    const uint64_t n = length < 0 ? 0 : min((uint64_t)length, q.max_length);
    uint64_t col, head, offset;
    const uint64_t p = pool.by_heads.divmod(s.per_head.divmod(i, col), head);
    if (p >= n) return;
    const uint64_t entry = pool.page_tokens.divmod(p, offset);
    const int32_t page = q.table[b * q.table_stride + entry];
    const int64_t row = q.first_rows[b] + (int64_t)p;
    if (page < 0 || (uint64_t)page >= pool.pages || row < 0 || (uint64_t)row >= q.rows) {
        if (col == 0 && head == 0) raise_error(errors, kErrIndexRange);
        return;
    }
    if (col >= s.dim) return;
    const uint64_t at = pool.row((uint64_t)page, offset, head);
    const float x = from_code(s.codes[at * s.dim + col]) * scale_value(s.scales[at * s.groups + col / kGroup]);
    s.wide[(uint64_t)row * s.token_stride + head * s.head_stride + col] = from_f32_finite<T>(x);
}

Pool pool_of(const lcbCacheQ8 &c) {
    return {c.pages, c.heads, FastDiv::of(c.page_tokens), FastDiv::of(c.heads), c.order == LCB_CACHE_HEADS_FIRST};
}

// `tokens`: rows per head that the side's blocks cover
template <typename T>
Side<T> side_of(T *wide, size_t token_stride, size_t head_stride, void *codes, void *scales, size_t dim, const lcbCacheQ8 &c, uint64_t tokens) {
    if (dim == 0) return {nullptr, 0, 0, nullptr, nullptr, 0, 0, FastDiv::of(1), 0};
    const uint64_t groups = groups_of(dim), lanes = tokens * c.heads * groups * kGroup;
    return {wide, token_stride, head_stride, static_cast<uint8_t *>(codes), static_cast<uint8_t *>(scales), dim, groups,
            FastDiv::of(groups * kGroup), (lanes + kThreads - 1) / kThreads};
}

template <typename Fn>
int with_type(int type, Fn fn) {
    switch (type) {
        case LCB_F32: return fn(static_cast<float *>(nullptr));
        case LCB_F16: return fn(static_cast<__half *>(nullptr));
        default: return fn(static_cast<__nv_bfloat16 *>(nullptr));
    }
}

}  // namespace

int preload_q8_kernels() {
    ErrorSink errors;
    return error_sink(&errors);
}
}  // namespace lcb

using namespace lcb;

extern "C" int lcb_cache_write_q8(const lcbCacheQ8 *cache, const void *k, size_t k_token_stride, size_t k_head_stride, const void *v,
                                  size_t v_token_stride, size_t v_head_stride, int type, const int64_t *slots, size_t tokens,
                                  lcbStream stream) {
    if (!cache_write_ok(cache, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, type, slots, tokens)) return 1;
    if (tokens == 0) return 0;
    ErrorSink errors;
    const int rc = error_sink(&errors);
    if (rc != 0) return rc;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto ks = side_of<const T>(static_cast<const T *>(k), k_token_stride, k_head_stride, cache->k_codes, cache->k_scales, cache->k_dim, *cache, tokens);
        const auto vs = side_of<const T>(static_cast<const T *>(v), v_token_stride, v_head_stride, cache->v_codes, cache->v_scales, cache->v_dim, *cache, tokens);
        const uint64_t blocks = ks.blocks + vs.blocks;
        if (blocks > 0x7fffffffu) return 1;
        return launch_kernel(cache_write_kernel<T>, (unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream), ks, vs, pool_of(*cache),
                             slots, (uint64_t)tokens, errors);
    });
}

extern "C" int lcb_cache_read_q8(const lcbCacheQ8 *cache, void *k, size_t k_token_stride, size_t k_head_stride, void *v, size_t v_token_stride,
                                 size_t v_head_stride, int type, const int32_t *page_table, size_t table_stride, const int32_t *lengths,
                                 const int64_t *first_rows, size_t sequences, size_t max_length, size_t rows, lcbStream stream) {
    if (!cache_read_ok(cache, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, type, page_table, table_stride, lengths,
                       first_rows, sequences, max_length, rows))
        return 1;
    if (sequences == 0 || max_length == 0) return 0;
    ErrorSink errors;
    const int rc = error_sink(&errors);
    if (rc != 0) return rc;
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        const auto ks = side_of<T>(static_cast<T *>(k), k_token_stride, k_head_stride, cache->k_codes, cache->k_scales, cache->k_dim, *cache, max_length);
        const auto vs = side_of<T>(static_cast<T *>(v), v_token_stride, v_head_stride, cache->v_codes, cache->v_scales, cache->v_dim, *cache, max_length);
        const uint64_t each = ks.blocks + vs.blocks;
        if (each * sequences > 0x7fffffffu) return 1;
        const Sequences q{page_table, lengths, first_rows, table_stride, max_length, rows, FastDiv::of(each)};
        return launch_kernel(cache_read_kernel<T>, (unsigned)(each * sequences), kThreads, 0, static_cast<cudaStream_t>(stream), ks, vs,
                             pool_of(*cache), q, errors);
    });
}
