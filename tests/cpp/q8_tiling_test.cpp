// The index arithmetic that the 8-bit kernels share with the host, checked without a GPU.  Prints "8-bit tiling ok".
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <random>
#include <vector>

#include "q8_tiling.h"

#define EXPECT(cond)                                                               \
    do {                                                                           \
        if (!(cond)) {                                                             \
            std::fprintf(stderr, "%s:%d: expected %s\n", __FILE__, __LINE__, #cond); \
            std::exit(1);                                                          \
        }                                                                          \
    } while (0)

static std::mt19937_64 rng(7);

template <typename U>
static U random_of_any_size() {
    return (U)(rng() >> (64 - std::numeric_limits<U>::digits + rng() % std::numeric_limits<U>::digits));
}

template <typename U>
static void divides() {
    const U most = std::numeric_limits<U>::max();
    std::vector<U> ds = {1, 2, 3, 5, 7, 31, 32, 33, 96, 1001, (U)(most / 2), (U)(most / 2 + 1), (U)(most / 2 + 2), (U)(most - 1), most};
    for (int bit = 0; bit < std::numeric_limits<U>::digits; ++bit)
        for (int off = -1; off <= 1; ++off)
            if ((U)((U)1 << bit) + off != 0) ds.push_back((U)(((U)1 << bit) + off));
    for (int i = 0; i < 2000; ++i) {
        const U d = random_of_any_size<U>();
        if (d != 0) ds.push_back(d);
    }
    for (U d : ds) {
        const auto by = lcb::FastDivide<U>::of(d);
        std::vector<U> ns = {0, 1, (U)(d - 1), d, (U)(d + 1), (U)(2 * d - 1), (U)(2 * d), (U)(most / d * d), (U)(most / d * d - 1), (U)(most - 1), most};
        for (int i = 0; i < 50; ++i) ns.push_back(random_of_any_size<U>());
        for (U n : ns) {
            U rest;
            const U q = by.divmod(n, rest);
            EXPECT(q == n / d);
            EXPECT(rest == n % d);
        }
    }
}

// Which access form rows at any address take: where both were measured and differ by 4 % or more, the faster one.
static void form_rule() {
    using lcb::RowOp;
    struct {
        size_t cols;
        bool f32, pack, unpack, unit, gradient;
    } const faster[] = {
        {225, false, false, false, false, false}, {513, false, false, false, false, false}, {521, false, false, false, false, false},
        {561, false, false, false, false, false}, {601, false, false, false, false, false}, {385, false, true, true, true, true},
        {481, false, true, true, true, true},     {511, false, true, true, true, true},     {777, false, true, true, true, true},
        {901, false, true, true, true, true},     {1023, false, true, true, true, true},    {1301, false, true, true, true, true},
        {1401, false, true, true, true, true},    {2561, false, true, true, true, true},    {225, true, false, false, false, false},
        {513, true, false, true, false, true},    {561, true, false, true, false, true},    {601, true, false, true, false, true},
        {651, true, false, true, false, true},     {701, false, false, true, false, false},
    };
    for (const auto &f : faster) {
        EXPECT(lcb::warp_form_pays(RowOp::Pack, f.f32, f.cols) == f.pack);
        EXPECT(lcb::warp_form_pays(RowOp::Unpack, f.f32, f.cols) == f.unpack);
        EXPECT(lcb::warp_form_pays(RowOp::Unit, f.f32, f.cols) == f.unit);
        EXPECT(lcb::warp_form_pays(RowOp::Gradient, f.f32, f.cols) == f.gradient);
    }
    EXPECT(lcb::warp_form_pays(RowOp::Pack, false, 1025) && lcb::warp_form_pays(RowOp::Unit, false, 1025) && !lcb::warp_form_pays(RowOp::Gradient, false, 1025));
    EXPECT(!lcb::warp_form_pays(RowOp::Unit, false, 2049) && !lcb::warp_form_pays(RowOp::Gradient, false, 2049) && lcb::warp_form_pays(RowOp::Unpack, false, 333) && !lcb::warp_form_pays(RowOp::Unit, true, 2049));
    for (RowOp op : {RowOp::Pack, RowOp::Unpack, RowOp::Unit, RowOp::Gradient})
        for (bool f32 : {false, true}) {
            EXPECT(!lcb::warp_form_pays(op, f32, 1) && !lcb::warp_form_pays(op, f32, 65) && !lcb::warp_form_pays(op, f32, 200));
            for (size_t cols : {(size_t)8191, (size_t)10241, (size_t)1 << 40}) EXPECT(lcb::warp_form_pays(op, f32, cols));
        }
}

// Every unit of every line has exactly one lane, whatever the width, the lines and the passes.
static void tilings() {
    for (uint64_t width : {1, 2, 6, 12, 31, 32, 64, 65, 96, 127, 128, 129, 160, 200, 256, 257, 500, 1000})
        for (uint64_t lines : {1, 2, 3, 100, 50001})
            for (uint32_t passes : {1, 2, 4}) {
                const auto t = lcb::Tiling::of(lines, width, passes, 1000);
                EXPECT(t.threads >= 1 && t.threads <= lcb::kMaxThreads && t.threads % 32 == 0);
                EXPECT((uint64_t)t.side_by_side * width <= t.threads || t.by_chunks.d > 1);
                EXPECT(t.by_chunks.d == 1 || ((uint64_t)t.by_chunks.d * t.threads >= width && (uint64_t)(t.by_chunks.d - 1) * t.threads < width));
                EXPECT(t.blocks() / t.by_chunks.d * t.side_by_side * t.passes >= lines);
                EXPECT((t.blocks() / t.by_chunks.d - 1) * t.side_by_side * t.passes < lines);
            }
}

int lcb::sm_count() { return 148; }

int main() {
    divides<uint32_t>();
    divides<uint64_t>();
    form_rule();
    tilings();
    std::puts("8-bit tiling ok");
    return 0;
}
