// Paged key/value cache in the 8-bit row format for sm_100a: quantising rows as they are written to their slots, and
// reading sequences back through a page table.
//
// Units and groups are those of q8_rows.cu; a row is a token's head here.  Every index that comes from device memory (slots,
// pages, lengths, first rows) is checked before it forms an address.
#include <algorithm>

#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

constexpr int kPasses = 4;  // tokens per lane

template <typename T>
struct Side {  // keys or values
    T *wide;
    uint64_t token_stride, head_stride;  // in elements of the wide type
    uint8_t *codes, *scales;
    uint32_t dim, groups;
    uint32_t token_rows, head_rows;  // rows of the pool from token to token and from head to head of a page
    FastDiv32 per_row;               // by the units of a row, padded to whole groups
    Tiling tiling;                   // a line is a token with all its heads
    uint32_t blocks;                 // of the grid (write), or of one sequence (read); 0: no such side in this launch
};

struct Pool {
    uint64_t slots, pages, page_rows;  // rows of a page: its tokens times the heads
    FastDiv page_tokens;               // of a slot
    FastDiv32 page_tokens32;           // of a position
    bool heads_first;
};

// A lane's tokens and its place in their heads.
template <int V>
struct Place {
    uint64_t token, wide;  // wide: offset of the lane's values from the token's
    uint64_t code, scale;  // the same in the pool
    uint32_t step, passes;
    int left;          // columns from the unit's first one on; 0: no unit
    bool leads, first; // leads its group, and so writes the scale; is the token's first unit
    template <typename T>
    __device__ __forceinline__ Place(const Side<T> &s, uint32_t block) {
        const Lane lane(s.tiling, block);
        token = lane.line;
        step = s.tiling.side_by_side;
        passes = s.tiling.passes;
        uint32_t unit;
        const uint32_t head = s.per_row.divmod((uint32_t)lane.unit, unit);
        const uint32_t column = unit * Form<V>::kValues;
        const uint64_t row = (uint64_t)head * s.head_rows;
        wide = head * s.head_stride + column;
        code = row * s.dim + column;
        scale = row * s.groups + unit / Form<V>::kLanes;
        left = lane.in && column < s.dim ? (int)(s.dim - column) : 0;
        leads = unit % Form<V>::kLanes == 0;
        first = lane.unit == 0;
    }
};

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) cache_write_kernel(Side<const T> k, Side<const T> v, Pool pool, const int64_t *slots,
                                                                  uint64_t tokens, ErrorSink errors) {
    pdl_launch_dependents();
    const bool keys = blockIdx.x < k.blocks;
    const Side<const T> s = keys ? k : v;
    const Place<V> at(s, blockIdx.x - (keys ? 0 : k.blocks));
    const T *from = s.wide + at.token * s.token_stride + at.wide;
    Unit<T, V> x[kPasses];
    int64_t slot[kPasses];
    pdl_wait();
    // The rows of skipped tokens are loaded too: waiting for the slot first would put a second memory latency in front of
    // every row.
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const uint64_t token = at.token + u * at.step;
        slot[u] = -1;
        x[u].clear();
        if (u < at.passes && at.left > 0 && token < tokens) {
            slot[u] = slots[token];
            x[u].load(from + u * (at.step * s.token_stride), at.left);
        }
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        if (u >= at.passes) break;
        Codes<V> c;
        const unsigned b = pack_unit(x[u], c);
        if (slot[u] < 0) continue;
        if ((uint64_t)slot[u] >= pool.slots) {
            if (at.first) raise_error(errors, kErrIndexRange);
            continue;
        }
        uint64_t row = (uint64_t)slot[u] * s.token_rows;
        if (pool.heads_first) {
            uint64_t offset;
            row = pool.page_tokens.divmod((uint64_t)slot[u], offset) * pool.page_rows;
            row += offset;
        }
        c.store(s.codes + row * s.dim + at.code, at.left);
        if (at.leads) s.scales[row * s.groups + at.scale] = (uint8_t)b;
    }
}

struct Sequences {
    const int32_t *table, *lengths;
    const int64_t *first_rows;
    uint64_t table_stride, rows;
    uint32_t max_length;
    FastDiv32 blocks;  // of one sequence, keys and values
};

template <typename T, int V>
__global__ void __launch_bounds__(kMaxThreads) cache_read_kernel(Side<T> k, Side<T> v, Pool pool, Sequences q, ErrorSink errors) {
    pdl_launch_dependents();
    uint32_t block;
    const uint32_t b = q.blocks.divmod(blockIdx.x, block);
    const bool keys = block < k.blocks;
    const Side<T> s = keys ? k : v;
    const Place<V> at(s, block - (keys ? 0 : k.blocks));
    const int32_t *table = q.table + b * q.table_stride;
    uint32_t offset[kPasses];
    int32_t page[kPasses];
    pdl_wait();
    const int32_t length = q.lengths[b];
    const int64_t first_row = q.first_rows[b];
    // page numbers are loaded beside the length; positions below max_length have an entry in the table
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const uint32_t p = (uint32_t)at.token + u * at.step;
        const uint32_t entry = pool.page_tokens32.divmod(p, offset[u]);
        page[u] = u < at.passes && p < q.max_length ? table[entry] : 0;
    }
    if (block == 0 && threadIdx.x == 0 && (length < 0 || (uint32_t)length > q.max_length)) raise_error(errors, kErrIndexRange);
    const uint32_t n = length < 0 ? 0 : min((uint32_t)length, q.max_length);
    const int64_t row = first_row + (int64_t)at.token;
    T *to = s.wide + (uint64_t)row * s.token_stride + at.wide;  // not formed into an access before its row is checked
    Codes<V> c[kPasses];
    unsigned scale[kPasses];
    bool live[kPasses];
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        const uint32_t p = (uint32_t)at.token + u * at.step;
        live[u] = u < at.passes && at.left > 0 && p < n;
        if (live[u] && ((uint32_t)page[u] >= pool.pages || (uint64_t)(row + (int64_t)(u * at.step)) >= q.rows)) {
            if (at.first) raise_error(errors, kErrIndexRange);
            live[u] = false;
        }
        if (live[u]) {
            const uint64_t from = (uint32_t)page[u] * pool.page_rows + (uint64_t)offset[u] * s.token_rows;
            c[u].load(s.codes + from * s.dim + at.code, at.left);
            scale[u] = s.scales[from * s.groups + at.scale];
        }
    }
#pragma unroll
    for (int u = 0; u < kPasses; ++u) {
        if (!live[u]) continue;
        const Pair by(scale_value(scale[u]));
        Unit<T, V> y;
#pragma unroll
        for (int j = 0; j < Form<V>::kValues; j += 2) y.template set_pair<true>(j, c[u].pair(j, by));
        y.store(to + u * (at.step * s.token_stride), at.left);
    }
}

Pool pool_of(const lcbCacheQ8 &c) {
    return {c.pages * c.page_tokens, c.pages, c.page_tokens * c.heads, FastDiv::of(c.page_tokens),
            FastDiv32::of((uint32_t)c.page_tokens), c.order == LCB_CACHE_HEADS_FIRST};
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
int by_sides(const lcbCacheQ8 &c, const Wide &k, const Wide &v, size_t tokens, size_t rows, size_t sequences, Launch launch) {
    const int ku = k.unit(c, rows, sizeof(T)), vu = c.v_dim != 0 ? v.unit(c, rows, sizeof(T)) : ku;
    auto side = [&](const Wide &w, int unit, bool on) {
        Side<T> s{};
        if (!on || w.dim == 0) return s;
        const uint64_t groups = groups_of(w.dim);
        const uint64_t per_row = unit == 16 ? Form<16>::per_row(groups) : unit == 8 ? Form<8>::per_row(groups) : Form<1>::per_row(groups);
        const bool heads_first = c.order == LCB_CACHE_HEADS_FIRST;
        s = {static_cast<T *>(const_cast<void *>(w.p)), w.token_stride, w.head_stride, static_cast<uint8_t *>(w.codes), static_cast<uint8_t *>(w.scales),
             (uint32_t)w.dim, (uint32_t)groups, heads_first ? 1u : (uint32_t)c.heads, heads_first ? (uint32_t)c.page_tokens : 1u,
             FastDiv32::of((uint32_t)per_row), Tiling::of(tokens, c.heads * per_row, kPasses, 2 * sequences), 0};
        s.blocks = (uint32_t)std::min<uint64_t>(s.tiling.blocks(), 0x80000000u);  // too many: refused by the launch
        return s;
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
        return by_sides<T>(*cache, kw, vw, tokens, tokens, 1, [&](auto u, const Side<T> &ks, const Side<T> &vs) {
            const uint64_t blocks = (uint64_t)ks.blocks + vs.blocks;
            if (blocks > 0x7fffffffu) return 1;
            const unsigned threads = std::max(ks.tiling.threads, vs.tiling.threads);
            return launch_kernel(cache_write_kernel<std::remove_const_t<T>, u()>, (unsigned)blocks, threads, 0, static_cast<cudaStream_t>(stream),
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
        return by_sides<T>(*cache, kw, vw, max_length, rows, sequences, [&](auto u, const Side<T> &ks, const Side<T> &vs) {
            const uint64_t each = (uint64_t)ks.blocks + vs.blocks;
            if (each > 0x7fffffffu || sequences > 0x7fffffffu / each) return 1;
            const Sequences q{page_table, lengths, first_rows, table_stride, rows, (uint32_t)max_length, FastDiv32::of((uint32_t)each)};
            const unsigned threads = std::max(ks.tiling.threads, vs.tiling.threads);
            return launch_kernel(cache_read_kernel<T, u()>, (unsigned)(each * sequences), threads, 0, static_cast<cudaStream_t>(stream), ks, vs,
                                 pool_of(*cache), q, errors);
        });
    });
}
