// A C++ consumer of the 8-bit operators, written as a program that uses the library would be: <librecuda.h>, link `driverapi`, check
// every status.  Values are chosen so that every code is exact (small integers times a power of two) and the whole way,
// through a page that is moved in between, gives them back unchanged.  Prints "8-bit operators ok".  Needs one GPU.
#include <librecuda.h>

#include <cstdio>
#include <cstdlib>
#include <vector>

#define CHECK(expr)                                                                                   \
    do {                                                                                              \
        libreCudaStatus_t status_ = (expr);                                                           \
        if (status_ != LIBRECUDA_SUCCESS) {                                                           \
            const char *name_ = nullptr;                                                              \
            libreCuGetErrorString(status_, &name_);                                                   \
            std::fprintf(stderr, "%s:%d: %s -> %s\n", __FILE__, __LINE__, #expr, name_ ? name_ : "?"); \
            std::exit(1);                                                                             \
        }                                                                                             \
    } while (0)
#define EXPECT(cond)                                                               \
    do {                                                                           \
        if (!(cond)) {                                                             \
            std::fprintf(stderr, "%s:%d: expected %s\n", __FILE__, __LINE__, #cond); \
            std::exit(1);                                                          \
        }                                                                          \
    } while (0)

static void *device(size_t bytes) {
    void *p = nullptr;
    CHECK(libreCuMemAlloc(&p, bytes));
    return p;
}
static void upload(LibreCUstream s, void *d, const void *h, size_t n) { CHECK(libreCuMemcpyHtoD(d, h, n, s)); }

int main() {
    CHECK(libreCuInit(0));
    LibreCUdevice gpu{};
    CHECK(libreCuDeviceGet(&gpu, 0));
    LibreCUcontext ctx{};
    CHECK(libreCuCtxCreate_v2(&ctx, CU_CTX_SCHED_YIELD, gpu));
    LibreCUstream s{};
    CHECK(libreCuStreamCreate(&s, 0));

    // a matrix of multiples of 1/4 below 4 in magnitude: packed and read back
    const size_t rows = 37, cols = 70;
    std::vector<float> x(rows * cols), y(rows * cols);
    for (size_t i = 0; i < x.size(); ++i) x[i] = 0.25f * (float)((int)(i * 7 % 15) - 7);
    void *dx = device(4 * x.size()), *dy = device(4 * x.size()), *codes = device(x.size()), *scales = device(rows * 3);
    upload(s, dx, x.data(), 4 * x.size());
    CHECK(libreCuPackQ8(codes, scales, dx, cols, LCB_F32, rows, cols, s));
    CHECK(libreCuUnpackQ8(dy, cols, LCB_F32, codes, scales, rows, cols, s));
    CHECK(libreCuMemcpyDtoH(y.data(), dy, 4 * y.size(), s));
    CHECK(libreCuStreamCommence(s));
    CHECK(libreCuStreamAwait(s));
    EXPECT(x == y);

    // the gated unit at gate = 0: h = 0, dgate = dh * up / 2, dup = 0, all exact
    void *h = device(4 * x.size()), *dg = device(4 * x.size()), *du = device(4 * x.size());
    void *gc = device(x.size()), *gs = device(rows * 3);
    CHECK(libreCuMemsetD32(dy, 0, x.size(), s));
    CHECK(libreCuSiluMulPackQ8(h, cols, gc, gs, codes, scales, dy, cols, dx, cols, LCB_F32, rows, cols, s));
    CHECK(libreCuSiluMulGradQ8(dg, cols, du, cols, nullptr, 0, dx, cols, gc, gs, codes, scales, LCB_F32, rows, cols, s));
    std::vector<float> a(x.size()), b(x.size()), c(x.size());
    CHECK(libreCuMemcpyDtoH(a.data(), h, 4 * a.size(), s));
    CHECK(libreCuMemcpyDtoH(b.data(), dg, 4 * b.size(), s));
    CHECK(libreCuMemcpyDtoH(c.data(), du, 4 * c.size(), s));
    CHECK(libreCuStreamCommence(s));
    CHECK(libreCuStreamAwait(s));
    for (size_t i = 0; i < x.size(); ++i) EXPECT(a[i] == 0.0f && c[i] == 0.0f && b[i] == x[i] * x[i] / 2);

    // a cache of one tensor: 20 tokens into pages 3 and 1, page 1 moved to 0, read through another table
    const size_t pages = 4, page = 16, heads = 2, dim = 64, tokens = 20;
    lcbCacheQ8 cache = {};
    cache.k_codes = device(pages * page * heads * dim);
    cache.k_scales = device(pages * page * heads * 2);
    cache.pages = pages, cache.page_tokens = page, cache.heads = heads, cache.k_dim = dim, cache.order = LCB_CACHE_HEADS_FIRST;
    std::vector<float> k(tokens * heads * dim), back(tokens * heads * dim, -1.0f);
    for (size_t i = 0; i < k.size(); ++i) k[i] = (float)((int)(i * 11 % 31) - 15);
    std::vector<int64_t> slots(tokens);
    for (size_t t = 0; t < tokens; ++t) slots[t] = t < page ? (int64_t)(3 * page + t) : (int64_t)(1 * page + t - page);
    const int32_t table[2] = {3, 0}, length = (int32_t)tokens;
    const int64_t first = 0;
    void *dk = device(4 * k.size()), *dslots = device(8 * tokens), *dtable = device(8), *dlength = device(4), *dfirst = device(8);
    upload(s, dk, k.data(), 4 * k.size());
    upload(s, dslots, slots.data(), 8 * tokens);
    upload(s, dtable, table, 8);
    upload(s, dlength, &length, 4);
    upload(s, dfirst, &first, 8);
    CHECK(libreCuCacheWriteQ8(&cache, dk, heads * dim, dim, nullptr, 0, 0, LCB_F32, (const int64_t *)dslots, tokens, s));
    char *kc = (char *)cache.k_codes, *ks = (char *)cache.k_scales;
    CHECK(libreCuMemCpy(kc, kc + page * heads * dim, page * heads * dim, s));
    CHECK(libreCuMemCpy(ks, ks + page * heads * 2, page * heads * 2, s));
    CHECK(libreCuMemsetD32(dk, 0, k.size(), s));
    CHECK(libreCuCacheReadQ8(&cache, dk, heads * dim, dim, nullptr, 0, 0, LCB_F32, (const int32_t *)dtable, 2, (const int32_t *)dlength,
                             (const int64_t *)dfirst, 1, 32, tokens, s));
    CHECK(libreCuMemcpyDtoH(back.data(), dk, 4 * back.size(), s));
    CHECK(libreCuStreamCommence(s));
    CHECK(libreCuStreamAwait(s));
    EXPECT(k == back);

    // refusals, and a page that is not there: reported once, and the stream goes on
    EXPECT(libreCuPackQ8(codes, scales, dx, cols, 9, rows, cols, s) == LIBRECUDA_ERROR_INVALID_VALUE);
    EXPECT(libreCuPackQ8(codes, scales, x.data(), cols, LCB_F32, rows, cols, s) == LIBRECUDA_ERROR_INVALID_VALUE);
    const int32_t bad[2] = {3, 4};
    upload(s, dtable, bad, 8);
    CHECK(libreCuCacheReadQ8(&cache, dk, heads * dim, dim, nullptr, 0, 0, LCB_F32, (const int32_t *)dtable, 2, (const int32_t *)dlength,
                             (const int64_t *)dfirst, 1, 32, tokens, s));
    CHECK(libreCuStreamCommence(s));
    EXPECT(libreCuStreamAwait(s) == LIBRECUDA_ERROR_UNKNOWN);
    CHECK(libreCuPackQ8(codes, scales, dx, cols, LCB_F32, rows, cols, s, true));
    CHECK(libreCuStreamCommence(s));
    CHECK(libreCuStreamAwait(s));

    CHECK(libreCuStreamDestroy(s));
    CHECK(libreCuCtxDestroy(ctx));
    std::puts("8-bit operators ok");
    return 0;
}
