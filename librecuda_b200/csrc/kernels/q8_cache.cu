// Paged key/value cache in the 8-bit row format for sm_100a: quantising rows as they are written to their slots, and
// reading sequences back through a page table.
//
// Units and groups are those of q8_rows.cu; a row is a token's head here.  Every index that comes from device memory (slots,
// pages, lengths, first rows) is checked before it forms an address.
#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;  // units in flight per lane

template <typename T>
struct Side {  // keys or values
    T *wide;
    uint64_t token_stride, head_stride;
    uint8_t *codes, *scales;
    uint64_t dim, groups;
    FastDiv per_row;                 // by the units of a row, padded to whole groups
    uint64_t skip_rows, skip_units;  // a CTA's threads as rows and units: from one unit of a lane to its next
    uint64_t blocks;                 // of the grid (write), or of one sequence (read)
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

template <int V>
struct Place {  // of a lane's unit among the rows (token, head)
    uint64_t row, unit;
    template <typename T>
    __device__ __forceinline__ Place(const Side<T> &s, uint64_t block) {
        row = s.per_row.divmod(block * (kThreads * kUnits) + threadIdx.x, unit);
    }
    template <typename T>
    __device__ __forceinline__ void next(const Side<T> &s) {
        row += s.skip_rows;
        unit += s.skip_units;
        if (unit >= s.per_row.d) {
            unit -= s.per_row.d;
            ++row;
        }
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(Side<const T> k, Side<const T> v, Pool pool, const int64_t *slots,
                                                               uint64_t tokens, ErrorSink errors) {
    pdl_launch_dependents();
    const bool first = blockIdx.x < k.blocks;
    const Side<const T> &s = first ? k : v;
    Place<V> at(s, blockIdx.x - (first ? 0 : k.blocks));
    Unit<T, V> x[kUnits];
    int64_t slot[kUnits];
    uint64_t head[kUnits], unit[kUnits];
    pdl_wait();
    // The rows of skipped tokens are loaded too: waiting for the slot first would put a second memory latency in front of
    // every row.
#pragma unroll
    for (int u = 0; u < kUnits; ++u, at.next(s)) {
        const uint64_t token = pool.by_heads.divmod(at.row, head[u]);
        unit[u] = at.unit;
        slot[u] = -1;
        x[u].clear();
        if (token < tokens) {
            slot[u] = slots[token];
            if (at.unit * V < s.dim) x[u].load(s.wide + token * s.token_stride + head[u] * s.head_stride + at.unit * V);
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        Codes<V> c;
        const int b = pack_unit(x[u], c);
        if (slot[u] < 0 || unit[u] * V >= s.dim) continue;
        uint64_t offset;
        const uint64_t page = pool.page_tokens.divmod((uint64_t)slot[u], offset);
        if (page >= pool.pages) {
            if (unit[u] == 0 && head[u] == 0) raise_error(errors, kErrIndexRange);
            continue;
        }
        const uint64_t row = pool.row(page, offset, head[u]);
        c.store(s.codes + row * s.dim + unit[u] * V);
        if ((unit[u] & (kGroup / V - 1)) == 0) s.scales[row * s.groups + unit[u] / (kGroup / V)] = (uint8_t)b;
    }
}

struct Sequences {
    const int32_t *table, *lengths;
    const int64_t *first_rows;
    uint64_t table_stride, max_length, rows;
    FastDiv blocks;  // of one sequence, keys and values
};

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(Side<T> k, Side<T> v, Pool pool, Sequences q, ErrorSink errors) {
    pdl_launch_dependents();
    uint64_t block;
    const uint64_t b = q.blocks.divmod(blockIdx.x, block);
    const bool first = block < k.blocks;
    const Side<T> &s = first ? k : v;
    Place<V> at(s, block - (first ? 0 : k.blocks));
    uint64_t head[kUnits], unit[kUnits], p[kUnits], offset[kUnits];
    int32_t page[kUnits];
    pdl_wait();
    const int32_t length = q.lengths[b];
    const int64_t first_row = q.first_rows[b];
    // page numbers are loaded beside the length; positions below max_length have an entry in the table
#pragma unroll
    for (int u = 0; u < kUnits; ++u, at.next(s)) {
        p[u] = pool.by_heads.divmod(at.row, head[u]);
        unit[u] = at.unit;
        const uint64_t entry = pool.page_tokens.divmod(p[u], offset[u]);
        page[u] = p[u] < q.max_length ? q.table[b * q.table_stride + entry] : 0;
    }
    if (block == 0 && threadIdx.x == 0 && (length < 0 || length > (int64_t)q.max_length)) raise_error(errors, kErrIndexRange);
    const uint64_t n = length < 0 ? 0 : min((uint64_t)length, q.max_length);
    Codes<V> c[kUnits];
    unsigned scale[kUnits];
    bool live[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t row = first_row + (int64_t)p[u];
        live[u] = p[u] < n && unit[u] * V < s.dim;
        if (live[u] && (page[u] < 0 || (uint64_t)page[u] >= pool.pages || row < 0 || (uint64_t)row >= q.rows)) {
            if (unit[u] == 0 && head[u] == 0) raise_error(errors, kErrIndexRange);
            live[u] = false;
        }
        if (live[u]) {
            const uint64_t from = pool.row((uint64_t)page[u], offset[u], head[u]);
            c[u].load(s.codes + from * s.dim + unit[u] * V);
            scale[u] = s.scales[from * s.groups + unit[u] / (kGroup / V)];
        }
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        if (!live[u]) continue;
        float x[V];
        c[u].values(x, scale_value(scale[u]));
        Unit<T, V> y;
        y.template set<true>(x);
        y.store(s.wide + (uint64_t)(first_row + (int64_t)p[u]) * s.token_stride + head[u] * s.head_stride + unit[u] * V);
    }
}

Pool pool_of(const lcbCacheQ8 &c) {
    return {c.pages, c.heads, FastDiv::of(c.page_tokens), FastDiv::of(c.heads), c.order == LCB_CACHE_HEADS_FIRST};
}

// `tokens`: rows per head that the side's blocks cover
template <typename T>
Side<T> side_of(T *wide, size_t token_stride, size_t head_stride, void *codes, void *scales, size_t dim, const lcbCacheQ8 &c, uint64_t tokens,
                int v) {
    const uint64_t groups = groups_of(dim), per_row = groups * (kGroup / v), tile = (uint64_t)kThreads * kUnits;
    return {wide, token_stride, head_stride, static_cast<uint8_t *>(codes), static_cast<uint8_t *>(scales), dim, groups, FastDiv::of(per_row),
            kThreads / per_row, kThreads % per_row, (tokens * c.heads * per_row + tile - 1) / tile};
}

struct Wide {  // the wide tensor of a side, as given
    const void *p;
    size_t token_stride, head_stride, dim;
    void *codes, *scales;
    // The widest unit whose accesses are aligned in every row (see q8_rows.cu).
    int unit(const lcbCacheQ8 &c, size_t tokens, size_t e) const {
        const uint64_t w = reinterpret_cast<uintptr_t>(p) | (tokens > 1 ? token_stride * e : 0) | (c.heads > 1 ? head_stride * e : 0);
        const uint64_t q = reinterpret_cast<uintptr_t>(codes);
        if (dim % 16 == 0 && w % 32 == 0 && q % 16 == 0) return 16;
        if (dim % 8 == 0 && w % 16 == 0 && q % 8 == 0) return 8;
        return 1;
    }
};

// Keys and values go to one launch where their units are the same, else to one each.
// launch(v, k side, v side): either side may have no blocks.
template <typename T, typename Launch>
int by_sides(const lcbCacheQ8 &c, const Wide &k, const Wide &v, size_t tokens, size_t rows, Launch launch) {
    const int ku = k.unit(c, rows, sizeof(T)), vu = c.v_dim != 0 ? v.unit(c, rows, sizeof(T)) : ku;
    auto side = [&](const Wide &w, int unit, bool on) {
        if (!on || w.dim == 0) return Side<T>{nullptr, 0, 0, nullptr, nullptr, 0, 0, FastDiv::of(1), 0, 0, 0};
        return side_of<T>(static_cast<T *>(const_cast<void *>(w.p)), w.token_stride, w.head_stride, w.codes, w.scales, w.dim, c, tokens, unit);
    };
    const bool both = ku == vu;
    const int rc = with_unit(ku, [&](auto u) { return launch(u, side(k, ku, true), side(v, vu, both)); });
    if (rc != 0 || both) return rc;
    return with_unit(vu, [&](auto u) { return launch(u, side(k, ku, false), side(v, vu, true)); });
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
    const Wide kw{k, k_token_stride, k_head_stride, cache->k_dim, cache->k_codes, cache->k_scales};
    const Wide vw{v, v_token_stride, v_head_stride, cache->v_dim, cache->v_codes, cache->v_scales};
    return with_type(type, [&](auto *t) {
        using T = const std::remove_pointer_t<decltype(t)>;
        return by_sides<T>(*cache, kw, vw, tokens, tokens, [&](auto u, const Side<T> &ks, const Side<T> &vs) {
            const uint64_t blocks = ks.blocks + vs.blocks;
            if (blocks > 0x7fffffffu) return 1;
            return launch_kernel(cache_write_kernel<std::remove_const_t<T>, u()>, (unsigned)blocks, kThreads, 0, static_cast<cudaStream_t>(stream),
                                 ks, vs, pool_of(*cache), slots, (uint64_t)tokens, errors);
        });
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
    const Wide kw{k, k_token_stride, k_head_stride, cache->k_dim, cache->k_codes, cache->k_scales};
    const Wide vw{v, v_token_stride, v_head_stride, cache->v_dim, cache->v_codes, cache->v_scales};
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        return by_sides<T>(*cache, kw, vw, max_length, rows, [&](auto u, const Side<T> &ks, const Side<T> &vs) {
            const uint64_t each = ks.blocks + vs.blocks;
            if (each * sequences > 0x7fffffffu) return 1;
            const Sequences q{page_table, lengths, first_rows, table_stride, max_length, rows, FastDiv::of(each)};
            return launch_kernel(cache_read_kernel<T, u()>, (unsigned)(each * sequences), kThreads, 0, static_cast<cudaStream_t>(stream), ks, vs,
                                 pool_of(*cache), q, errors);
        });
    });
}
