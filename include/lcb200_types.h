/* lcb200_types.h -- types shared by the kernel layer (lcb200_kernels.h) and the stream API (librecuda.h). */
#ifndef LCB200_TYPES_H
#define LCB200_TYPES_H

#include <stddef.h>
#include <stdint.h>

/* Element types of the wide side of the 8-bit operators. */
enum lcbType {
    LCB_F32 = 0,  /* IEEE binary32 */
    LCB_F16 = 1,  /* IEEE binary16 */
    LCB_BF16 = 2  /* bfloat16      */
};

/* Order of the two middle dimensions of a paged cache. */
enum lcbCacheOrder {
    LCB_CACHE_TOKENS_FIRST = 0, /* [pages][page_tokens][heads][...] */
    LCB_CACHE_HEADS_FIRST = 1   /* [pages][heads][page_tokens][...] */
};

/* A paged cache in the 8-bit row format (see lcb200_kernels.h): per tensor one array of codes, innermost
 * dimension `dim`, and one of scale bytes, innermost dimension (dim + 31) / 32, both dense in the order above.
 * Slot s of the cache is token s % page_tokens of page s / page_tokens.  A cache of one tensor only (keys and
 * values in one latent vector) has v_codes = v_scales = NULL and v_dim = 0. */
typedef struct lcbCacheQ8 {
    void *k_codes, *k_scales;
    void *v_codes, *v_scales;
    size_t pages;
    size_t page_tokens;
    size_t heads;
    size_t k_dim, v_dim;
    int order; /* enum lcbCacheOrder */
} lcbCacheQ8;

#endif /* LCB200_TYPES_H */
