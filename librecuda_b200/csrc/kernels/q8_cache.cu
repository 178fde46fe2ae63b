// Paged key/value cache in the 8-bit row format for sm_100a: quantising rows as they are written to their slots, and
// reading sequences back through a page table.
//
// Units, groups and rounding are those of q8.cuh; a row is a token's head, a line a token with all its heads, so that
// a lane keeps its place in the heads and steps from token to token.  Keys and values share a launch.  Every index
// that comes from device memory (slots, pages, lengths, first rows) is checked before it forms an address.
//
// What bounds them: HBM, 3.03 bytes per value of bf16, and for a read the chain length -> page -> code in front of
// it.  A CTA of 128 threads holds few tokens, so the chain is walked by many CTAs at once; a write loads its rows
// beside their slots.
//
// Measured on a B200 (bf16, 8 heads of 128; share of 6548 GB/s): write of 65000 tokens, a sixteenth of them padding,
// 60 us, 96 % (64 us and 90 % heads first: 128-byte pieces); read of 48 sequences of 1 to 16384 tokens 377 us, 99 %;
// in f32 99 %.  A cache of one tensor, 576 wide: 20.7 us and 84 %, 117 us and 90 %.  Heads of 65: 84 us and 35 %, 515 us and
// 37 %, rows at any address in words lane by lane.
// One token: write 1.05 us in a graph. One lane per value instead of 16: 997 and 9805 us.  Rows loaded only once
// their slots are known: 65 us against 61.
#include <algorithm>

#include "lcb200_kernels.h"
#include "q8.cuh"
#include "q8_check.h"

namespace lcb {
namespace {

__device__ unsigned int g_index_word = 0;              // kErrIndexRange, once an index was out of range
__device__ unsigned int *g_index_mirror = nullptr;     // its host-mapped copy, NULL before lcb_preload
__device__ __forceinline__ void raise_index_error() {
    atomicOr(&g_index_word, kErrIndexRange);
    unsigned int *m = g_index_mirror;
    if (m != nullptr) {
        atomicOr_system(m, kErrIndexRange);
        __threadfence_system();
    }
}

// Tokens in flight per lane, where there is work for that many.  Write: 4 (61 us; 2: 65; 1: 76).  Read: 2 (377 us; 4:
// 378; 1: 422).
template <int A>
constexpr int kPassesWrite = A >= 16 ? 4 : 2;
constexpr int kPassesRead = 2;
// Heads at any address: values per lane of a write (65 columns: bf16 84 us with 16, f32 48 with 8, 52 with 16); a
// read takes 8.
template <typename T>
constexpr int kWriteForm = sizeof(T) == 4 ? kLooseShort : kLoose;
constexpr int kRunTiles = 4, kRunWaves = 4, kMostWaves = 64;  // tiles that a CTA of a read takes, see its launcher

template <typename T>
struct Side {  // keys or values
    T *wide;
    uint64_t token_stride, head_stride;  // in elements of the wide type
    uint8_t *codes, *scales;
    uint32_t dim, groups;
    uint64_t head_rows;              // rows of the pool from head to head of a page
    uint64_t page_codes, page_scales;    // bytes of a page
    uint32_t token_codes, token_scales;  // bytes from token to token of a page
    FastDiv32 per_row;               // by the units of a row, padded to whole groups
    Tiling tiling;                   // a line is a token with all its heads
    uint32_t blocks;                 // of the grid (write), or of one sequence (read); 0: no such side in this launch
    uint64_t all_blocks() const { return dim != 0 ? tiling.blocks() : 0; }
};

struct Pool {
    uint64_t slots, pages;
    FastDiv page_tokens;      // of a slot
    FastDiv32 page_tokens32;  // of a position, and of a slot where the slots are few enough
    bool heads_first, few_slots;
};

// A lane's tokens and its place in their heads.
template <int A, int P>
struct Place {
    uint64_t token, wide;  // wide: offset of the lane's values from the token's
    uint64_t code, scale;  // the same in the pool
    uint32_t step;
    int left;          // columns from the unit's first one on; 0: no unit
    bool leads, first; // leads its group, and so writes the scale; is the token's first unit
    template <typename T>
    __device__ __forceinline__ Place(const Side<T> &s, const Lane &lane) {
        token = lane.line;
        step = s.tiling.side_by_side;
        uint32_t unit;
        const uint32_t head = s.per_row.divmod((uint32_t)lane.unit, unit);
        const uint32_t column = unit * Form<A>::kValues;
        const uint64_t row = (uint64_t)head * s.head_rows;
        wide = head * s.head_stride + column;
        code = row * s.dim + column;
        scale = row * s.groups + unit / Form<A>::kLanes;
        left = lane.in && column < s.dim ? (int)(s.dim - column) : 0;
        leads = unit % Form<A>::kLanes == 0;
        first = lane.unit == 0;
    }
};

template <typename T, int A, int P>
__global__ void __launch_bounds__(kMaxThreads) cache_write_kernel(Side<const T> k, Side<const T> v, Pool pool, const int64_t *slots,
                                                                  uint64_t tokens) {
    pdl_launch_dependents();
    const bool keys = blockIdx.x < k.blocks;
    const Side<const T> s = keys ? k : v;
    const Place<A, P> at(s, Lane(s.tiling, blockIdx.x - (keys ? 0 : k.blocks), P));
    const T *from = s.wide + at.token * s.token_stride + at.wide;
    uint8_t *codes = s.codes + at.code, *scales = s.scales + at.scale;
    Unit<T, A> x[P];
    int64_t slot[P];
    pdl_wait();
    // The rows of skipped tokens are loaded too: waiting for the slot first would put a second memory latency in
    // front of every row.  65000 tokens, a sixteenth of them skipped: 59 us, 65 with the slots first; half of them skipped
    // 53 us, fifteen sixteenths 42.
#pragma unroll
    for (int u = 0; u < P; ++u) {
        const uint64_t token = at.token + u * at.step;
        const int left = token < tokens ? at.left : 0;
        slot[u] = left > 0 ? slots[token] : -1;
        x[u].load(from + u * (at.step * s.token_stride), left);
    }
#pragma unroll
    for (int u = 0; u < P; ++u) {
        Codes<A> c;
        const unsigned b = pack_unit(x[u], c);
        if (slot[u] < 0) continue;
        if ((uint64_t)slot[u] >= pool.slots) {
            if (at.first) raise_index_error();
            continue;
        }
        uint64_t page = 0, offset = (uint64_t)slot[u];  // tokens first: pages lie behind each other like their tokens
        if (pool.heads_first) {
            if (pool.few_slots) {
                uint32_t o;
                page = pool.page_tokens32.divmod((uint32_t)slot[u], o);
                offset = o;
            } else {
                page = pool.page_tokens.divmod((uint64_t)slot[u], offset);
            }
        }
        c.store(codes + (page * s.page_codes + offset * s.token_codes), at.left);
        if (at.leads) scales[page * s.page_scales + offset * s.token_scales] = (uint8_t)b;
    }
}

struct Sequences {
    const int32_t *table, *lengths;
    const int64_t *first_rows;
    uint64_t table_stride, rows;
    uint32_t max_length;
    uint32_t tiles;    // of a CTA
    FastDiv32 blocks;  // of one sequence, keys and values
};

// A CTA takes `tiles` tiles of one sequence, one behind the other: in a ragged batch much of the grid lies behind the
// ends of the sequences, and a CTA that finds nothing to do costs a launch and a memory latency all the same (377 us
// with up to 4 tiles, 404 with one, 384 with 8, which leave too few CTAs to even out the sequences).
template <typename T, int A, int P>
__global__ void __launch_bounds__(kMaxThreads) cache_read_kernel(Side<T> k, Side<T> v, Pool pool, Sequences q) {
    pdl_launch_dependents();
    uint32_t block;
    const uint32_t b = q.blocks.divmod(blockIdx.x, block);
    const bool keys = block < k.blocks;
    const Side<T> s = keys ? k : v;
    const uint32_t in_side = block - (keys ? 0 : k.blocks);
    uint32_t chunk;
    const uint32_t run = s.tiling.by_chunks.divmod(in_side, chunk);
    const Place<A, P> at(s, Lane(s.tiling, run * q.tiles, chunk, P));
    const int32_t *table = q.table + b * q.table_stride;
    const uint8_t *codes = s.codes + at.code, *scales = s.scales + at.scale;
    pdl_wait();
    const int32_t length = q.lengths[b];
    const int64_t first_row = q.first_rows[b];
    if (block == 0 && threadIdx.x == 0 && (length < 0 || (uint32_t)length > q.max_length)) raise_index_error();
    const uint32_t n = length < 0 ? 0 : min((uint32_t)length, q.max_length);
    uint32_t token = (uint32_t)at.token;
    const uint32_t tile = at.step * P, end = min((uint64_t)n, at.token + (uint64_t)tile * q.tiles);
    for (; token < end; token += tile) {
        uint32_t offset[P];
        int32_t page[P];
#pragma unroll
        for (int u = 0; u < P; ++u) {
            const uint32_t p = token + u * at.step;
            const uint32_t entry = pool.page_tokens32.divmod(p, offset[u]);
            page[u] = p < n ? table[entry] : 0;
        }
        const uint64_t row = (uint64_t)first_row + token;  // a negative first row wraps to where no row is
        Codes<A> c[P];
        unsigned scale[P];
        bool live[P];
#pragma unroll
        for (int u = 0; u < P; ++u) {
            live[u] = at.left > 0 && token + u * at.step < n;
            if (live[u] && ((uint32_t)page[u] >= pool.pages || row + u * at.step >= q.rows)) {
                if (at.first) raise_index_error();
                live[u] = false;
            }
            if (live[u]) {
                c[u].load(codes + ((uint32_t)page[u] * s.page_codes + (uint64_t)offset[u] * s.token_codes), at.left);
                scale[u] = scales[(uint32_t)page[u] * s.page_scales + (uint64_t)offset[u] * s.token_scales];
            }
        }
        T *to = s.wide + (row * s.token_stride + at.wide);  // no access before the row is checked
#pragma unroll
        for (int u = 0; u < P; ++u) {
            if (!live[u]) continue;
            const Pair by(scale_value(scale[u]));
            Unit<T, A> y;
#pragma unroll
            for (int j = 0; j < Form<A>::kValues; j += 2) y.template set_pair<true>(j, c[u].pair(j, by));
            y.store(to + u * (at.step * s.token_stride), at.left, nullptr);
        }
    }
}

Pool pool_of(const lcbCacheQ8 &c) {
    const uint64_t slots = (uint64_t)c.pages * c.page_tokens;
    return {slots, c.pages, FastDiv::of(c.page_tokens), FastDiv32::of((uint32_t)c.page_tokens), c.order == LCB_CACHE_HEADS_FIRST,
            slots <= 0xffffffffu};
}

struct Wide {  // the wide tensor of a side, as given
    const void *p;
    size_t token_stride, head_stride, dim;
    void *codes, *scales;
    // The widest accesses that are aligned in every row (see q8_rows.cu).
    int access(const lcbCacheQ8 &c, size_t tokens, size_t e) const {
        const uint64_t w = reinterpret_cast<uintptr_t>(p) | (tokens > 1 ? token_stride * e : 0) | (c.heads > 1 ? head_stride * e : 0);
        const uint64_t q = reinterpret_cast<uintptr_t>(codes);
        if (dim % 16 == 0 && w % 32 == 0 && q % 16 == 0) return 32;
        if (dim % 8 == 0 && w % 16 == 0 && q % 8 == 0) return 16;
        return 0;
    }
};

// Keys and values go to one launch where their accesses are the same, else to one each.
// launch(access, passes, k side, v side): either side may have no blocks.  passes(access): at most.
template <int LOOSE, typename T, typename Passes, typename Launch>
int by_sides(const lcbCacheQ8 &c, const Wide &k, const Wide &v, size_t tokens, size_t rows, size_t sequences, Passes passes,
             Launch launch) {
    const int ka = k.access(c, rows, sizeof(T)), va = c.v_dim != 0 ? v.access(c, rows, sizeof(T)) : ka;
    auto both = [&](int access, bool with_k, bool with_v) {
        return with_access<LOOSE, false>(access, [&](auto a) {
            auto side = [&](const Wide &w, bool on) {
                Side<T> s{};
                if (!on || w.dim == 0) return s;
                const uint64_t groups = groups_of(w.dim), per_row = groups * Form<a()>::kLanes;
                const bool heads_first = c.order == LCB_CACHE_HEADS_FIRST;
                const uint64_t token_rows = heads_first ? 1 : c.heads, page_rows = (uint64_t)c.page_tokens * c.heads;
                s.wide = static_cast<T *>(const_cast<void *>(w.p));
                s.token_stride = w.token_stride, s.head_stride = w.head_stride;
                s.codes = static_cast<uint8_t *>(w.codes), s.scales = static_cast<uint8_t *>(w.scales);
                s.dim = (uint32_t)w.dim, s.groups = (uint32_t)groups;
                s.head_rows = heads_first ? c.page_tokens : 1;
                s.page_codes = page_rows * w.dim, s.page_scales = page_rows * groups;
                s.token_codes = (uint32_t)(token_rows * w.dim), s.token_scales = (uint32_t)(token_rows * groups);
                s.per_row = FastDiv32::of((uint32_t)per_row);
                s.tiling = Tiling::of(tokens, c.heads * per_row, passes(a), 2 * sequences);
                return s;
            };
            Side<T> ks = side(k, with_k), vs = side(v, with_v);
            const uint32_t p = std::max(ks.tiling.passes, vs.tiling.passes);  // the same for both: they share a kernel
            for (Side<T> *s : {&ks, &vs}) {
                if (s->dim == 0) continue;
                s->tiling.passes = p;
            }
            return with_passes<passes(a)>(p, [&](auto pp) { return launch(a, pp, ks, vs); });
        });
    };
    if (ka == va) return both(ka, true, true);
    const int rc = both(ka, true, false);
    return rc != 0 ? rc : both(va, false, true);
}

template <typename T>
int load_cache_kernels() {
    using C = const T;
    constexpr int loose = kWriteForm<C>;
    return first_error({load_kernel(cache_write_kernel<T, 32, 1>), load_kernel(cache_write_kernel<T, 32, kPassesWrite<32>>),
                        load_kernel(cache_write_kernel<T, 16, 1>), load_kernel(cache_write_kernel<T, 16, kPassesWrite<16>>),
                        load_kernel(cache_write_kernel<T, loose, 1>), load_kernel(cache_write_kernel<T, loose, kPassesWrite<loose>>),
                        load_kernel(cache_read_kernel<T, 32, 1>), load_kernel(cache_read_kernel<T, 32, kPassesRead>),
                        load_kernel(cache_read_kernel<T, 16, 1>), load_kernel(cache_read_kernel<T, 16, kPassesRead>),
                        load_kernel(cache_read_kernel<T, kLooseShort, 1>), load_kernel(cache_read_kernel<T, kLooseShort, kPassesRead>)});
}

}  // namespace

int index_error_mirror(unsigned int *mirror) { return (int)cudaMemcpyToSymbol(g_index_mirror, &mirror, sizeof(mirror)); }
int index_error_take(unsigned int *bits) {
    cudaError_t err = cudaMemcpyFromSymbol(bits, g_index_word, sizeof(*bits));
    const unsigned int zero = 0;
    if (err == cudaSuccess && *bits != 0) err = cudaMemcpyToSymbol(g_index_word, &zero, sizeof(zero));
    return (int)err;
}

int preload_q8_cache_kernels() {
    return first_error({load_cache_kernels<float>(), load_cache_kernels<__half>(), load_cache_kernels<__nv_bfloat16>()});
}
}  // namespace lcb

using namespace lcb;

extern "C" int lcb_cache_write_q8(const lcbCacheQ8 *cache, const void *k, size_t k_token_stride, size_t k_head_stride, const void *v,
                                  size_t v_token_stride, size_t v_head_stride, int type, const int64_t *slots, size_t tokens,
                                  lcbStream stream) {
    if (!cache_write_ok(cache, k, k_token_stride, k_head_stride, v, v_token_stride, v_head_stride, type, slots, tokens)) return 1;
    if (tokens == 0) return 0;
    const Wide kw{k, k_token_stride, k_head_stride, cache->k_dim, cache->k_codes, cache->k_scales};
    const Wide vw{v, v_token_stride, v_head_stride, cache->v_dim, cache->v_codes, cache->v_scales};
    return with_type(type, [&](auto *t) {
        using T = const std::remove_pointer_t<decltype(t)>;
        auto passes = [](auto a) { return kPassesWrite<decltype(a)::value>; };
        return by_sides<kWriteForm<T>, T>(*cache, kw, vw, tokens, tokens, 1, passes,
                                          [&](auto a, auto p, const Side<T> &ks, const Side<T> &vs) {
            const uint64_t kb = ks.all_blocks(), vb = vs.all_blocks();
            if (kb + vb > kMostBlocks) return 1;
            Side<T> kg = ks, vg = vs;
            kg.blocks = (uint32_t)kb, vg.blocks = (uint32_t)vb;
            const unsigned threads = std::max(ks.tiling.threads, vs.tiling.threads);
            return launch_kernel(cache_write_kernel<std::remove_const_t<T>, a(), p()>, (unsigned)(kb + vb), threads, 0,
                                 static_cast<cudaStream_t>(stream), kg, vg, pool_of(*cache), slots, (uint64_t)tokens);
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
    const Wide kw{k, k_token_stride, k_head_stride, cache->k_dim, cache->k_codes, cache->k_scales};
    const Wide vw{v, v_token_stride, v_head_stride, cache->v_dim, cache->v_codes, cache->v_scales};
    return with_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        auto passes = [](auto) { return kPassesRead; };
        return by_sides<kLooseShort, T>(*cache, kw, vw, max_length, rows, sequences, passes,
                                        [&](auto a, auto p, const Side<T> &ks, const Side<T> &vs) {
            // Up to kRunTiles tiles to a CTA while that leaves the GPU kRunWaves grids of resident CTAs, and more of
            // them where the grid would have more than kMostWaves: max_length may be far above the lengths.
            const uint64_t kb = ks.all_blocks(), vb = vs.all_blocks(), all = (kb + vb) * sequences, wave = Tiling::resident_ctas();
            const uint32_t tiles = (uint32_t)std::max<uint64_t>(std::min<uint64_t>(std::max<uint64_t>(all / (wave * kRunWaves), 1), kRunTiles),
                                                                std::min<uint64_t>(all / (wave * kMostWaves), 0x7fffffffu));
            auto runs = [&](const Side<T> &s, uint64_t blocks) {  // of one sequence
                return blocks == 0 ? 0 : (blocks / s.tiling.by_chunks.d + tiles - 1) / tiles * s.tiling.by_chunks.d;
            };
            const uint64_t k_runs = runs(ks, kb), v_runs = runs(vs, vb), each = k_runs + v_runs;
            if (each > kMostBlocks || sequences > kMostBlocks / each) return 1;
            Side<T> kr = ks, vr = vs;
            kr.blocks = (uint32_t)k_runs, vr.blocks = (uint32_t)v_runs;
            const Sequences q{page_table, lengths, first_rows, table_stride, rows, (uint32_t)max_length, tiles, FastDiv32::of((uint32_t)each)};
            const unsigned threads = std::max(ks.tiling.threads, vs.tiling.threads);
            return launch_kernel(cache_read_kernel<T, a(), p()>, (unsigned)(each * sequences), threads, 0,
                                 static_cast<cudaStream_t>(stream), kr, vr, pool_of(*cache), q);
        });
    });
}
