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

int main() {
    divides<uint32_t>();
    divides<uint64_t>();
    std::puts("8-bit tiling ok");
    return 0;
}
