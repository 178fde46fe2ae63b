// Index arithmetic of the 8-bit operators that the host can run too: division by a launch constant, which lane works on
// which values, and which access form a matrix of rows at any address takes.
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __CUDACC__
#define LCB_HOST_DEVICE __host__ __device__ __forceinline__
#else
#define LCB_HOST_DEVICE inline
#endif

namespace lcb {

// ---- division by a launch constant ----------------------------------------------------------------------------
// magic = floor((2^bits - 1) / d): the high half of n * magic is the quotient or one less, for every n of `bits` bits.
LCB_HOST_DEVICE uint64_t high_half(uint64_t a, uint64_t b) {
#ifdef __CUDA_ARCH__
    return __umul64hi(a, b);
#else
    return (uint64_t)((unsigned __int128)a * b >> 64);
#endif
}
LCB_HOST_DEVICE uint32_t high_half(uint32_t a, uint32_t b) {
#ifdef __CUDA_ARCH__
    return __umulhi(a, b);
#else
    return (uint32_t)((uint64_t)a * b >> 32);
#endif
}

template <typename U>
struct FastDivide {
    U magic, d;
    static FastDivide of(U d) { return {(U)(~(U)0 / d), d}; }
    LCB_HOST_DEVICE U divmod(U n, U &rest) const {
        U q = high_half(n, magic);
        rest = n - q * d;
        if (rest >= d) {
            rest -= d;
            ++q;
        }
        return q;
    }
};
using FastDiv = FastDivide<uint64_t>;
using FastDiv32 = FastDivide<uint32_t>;

constexpr int kGroup = 32;  // values per scale byte
int sm_count();             // of the current device

// ---- units --------------------------------------------------------------------------------------------------------
// A unit is kValues consecutive values of a row, held by one lane; kLanes neighbouring lanes hold a group.  Its accesses come
// in forms A.
//   32, 16        bytes of an access to the wide type (the codes then in 16 or 8 bytes); a row ends with a whole unit, or with
//                 8 or 16 values of one
//   kWarp         rows at any address, ending anywhere, a warp inside one row: as kLoose, but the warp loads and stores its 512
//                 wide values as a run of words side by side, handed over through shared memory
//   kLoose, kLooseShort, kLooseTiny
//                 rows at any address too short to give a warp to each: a lane fetches its 16, 8 or 4 values in the words that
//                 the address allows.  A warp then touches many sectors at once; loads find them again in L1, stores do
//                 not, so what a kernel moves decides how many values serve it best.
constexpr int kWarp = 1, kLooseShort = 2, kLooseTiny = 3, kLoose = 4;
template <int A>
struct Form {
    static constexpr int kValues = A == kLooseTiny ? 4 : A == kLooseShort ? 8 : 16;
    static constexpr int kLanes = kGroup / kValues;
};

// ---- which units a lane works on --------------------------------------------------------------------------------
// The data is `lines` lines (rows of a matrix, tokens of a cache) of `width` units each, a row padded to whole
// groups.  A CTA takes `passes` units per lane, at the same place of as many lines, so a lane knows its column once
// and only steps its pointers from line to line.  Lines of up to kMaxThreads units: several lie side by side in a
// CTA.  Longer ones: `chunks` CTAs share a line in even parts.  Parts start at multiples of 32 lanes, lines at
// multiples of a group's lanes, so the lanes of a group are neighbours in one warp.  A grid that would not fill half
// of the GPU that way takes one pass (pack 3000x4096 bf16: 5.7 us with the border at half of the resident CTAs, 7.1
// at all of them; 1000x4096: 2.3, and 2.7 at a sixteenth).  128 threads: with 256 the gated unit takes 113 us instead
// of 101, a cache write 64 instead of 61.
constexpr int kMaxThreads = 128;
struct Tiling {
    uint64_t width, lines;
    FastDiv32 by_chunks, by_width;  // by_width: of lines that lie side by side, else 0 / 1
    uint32_t threads, side_by_side, passes;
    // `times`: how often the launch repeats the tiling
    static Tiling of(uint64_t lines, uint64_t width, uint32_t passes, uint64_t times = 1) {
        Tiling t{width, lines, FastDiv32::of(1), FastDiv32::of(1), 0, 1, passes};
        if (width <= kMaxThreads) {
            t.by_width = FastDiv32::of((uint32_t)width);
            t.side_by_side = (uint32_t)(kMaxThreads / width);
            if (t.side_by_side > lines) t.side_by_side = (uint32_t)lines;
            t.threads = (uint32_t)((t.side_by_side * width + 31) / 32 * 32);
        } else {
            const uint64_t chunks = (width + kMaxThreads - 1) / kMaxThreads;
            t.by_chunks = FastDiv32::of(chunks < 0xffffffffu ? (uint32_t)chunks : 0xffffffffu);  // so many: no launch takes the grid
            t.threads = (uint32_t)(((width + chunks - 1) / chunks + 31) / 32 * 32);
        }
        if (passes > 1 && t.blocks() * times < resident_ctas() / 2) t.passes = 1;
        return t;
    }
    static uint64_t resident_ctas() { return (uint64_t)sm_count() * (2048 / kMaxThreads); }
    uint64_t blocks() const {
        const uint64_t tile = (uint64_t)side_by_side * passes;
        return (lines + tile - 1) / tile * by_chunks.d;
    }
};

// ---- rows at any address: a warp inside one row, or lanes side by side ---------------------------------------------
// Either form costs by the places for values in the lanes it launches, and kWarp launches whole warps per row (of parts, where
// a row takes several CTAs): 513 columns fill half of them.  Operators that pack 16-bit values are bound by instructions, so
// there kWarp is taken where it has at most 10 % more places than the other form, which also ends its rows with whole
// warps now and then (1025 columns).  The others move sectors, which kWarp does better at any row and the lanes behind its
// end do worse: there it is taken where the values fill at least a share of its places.
// Both forms measured at 24 M values, us (other form / kWarp; in brackets the values' share of kWarp's places):
//   bf16         513 columns (50 %)   701 (68 %)   1025 (67 %)    777 (76 %)
//   pack              26.5 / 30.8    23.9 / 25.1   24.7 / 23.6   25.7 / 23.1
//   unpack            26.1 / 28.5    24.3 / 22.5   26.1 / 26.3   24.4 / 20.8
//   gated unit        72.0 / 85.0    61.9 / 67.9   67.2 / 64.8   67.6 / 62.0
//   gradient          58.2 / 75.3    56.7 / 57.5   53.0 / 58.7   56.4 / 53.1
//   f32          225 columns (44 %)    513          701          1201 (78 %)
//   pack              33.5 / 48.7    33.0 / 38.2   31.8 / 32.3   31.5 / 29.1
//   unpack            29.6 / 33.5    48.4 / 30.6   36.7 / 26.1   32.7 / 24.6
//   gated unit        66.8 / 108.6   75.3 / 91.4   69.3 / 81.6   74.9 / 75.0
//   gradient          64.7 / 95.7   101.8 / 83.4   70.9 / 67.4   67.0 / 65.1
// At 27 widths from 225 to 2561 the slower form is taken nowhere by more than 5 %.
enum class RowOp { Pack, Unpack, Unit, Gradient };
// The other form.  Loads of 32-bit values share sectors less, so fewer to a lane; stores still fewer (100 columns of f32:
// pack 35 us with 8, 45 with 16, 40 with 4; unpack 48 with 4, 74 with 8; the 16-bit types the other way round).
constexpr int loose_form(RowOp op, bool f32) {
    return op == RowOp::Pack ? (f32 ? kLooseShort : kLoose) : (f32 ? kLooseTiny : kLooseShort);
}
template <int A>
uint64_t units_of(uint64_t cols) {  // of a row, padded to whole groups, or to whole warps
    const uint64_t units = (cols + kGroup - 1) / kGroup * Form<A>::kLanes;
    return A == kWarp ? (units + 31) / 32 * 32 : units;
}
template <int A>
uint64_t places_of_rows(uint64_t cols, uint64_t rows) {  // for values in the lanes of that many rows side by side
    const Tiling t = Tiling::of(rows, units_of<A>(cols), 1);
    return t.threads * t.blocks() * Form<A>::kValues;
}
inline bool warp_form_pays(RowOp op, bool f32, uint64_t cols) {
    const uint64_t rows = 2 * 3 * 5 * 7 * 8;  // enough for full CTAs, whatever lies side by side
    const uint64_t places = places_of_rows<kWarp>(cols, rows);
    if (!f32 && op == RowOp::Pack) return places / 11 * 10 <= places_of_rows<kLoose>(cols, rows);
    if (!f32 && op == RowOp::Unit) return places / 11 * 10 <= places_of_rows<kLooseShort>(cols, rows);
    const unsigned percent = f32 ? (op == RowOp::Pack ? 66 : op == RowOp::Unit ? 78 : 48) : (op == RowOp::Unpack ? 64 : 74);
    return cols >= places / rows * percent / 100;
}

}  // namespace lcb
