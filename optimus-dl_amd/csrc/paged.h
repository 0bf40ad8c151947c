// What the kernels over a paged cache share: the cache and the batch as the kernels read them, and the host's checks of both.
#pragma once

#include "common.h"

namespace odl {

struct Paged {
    uint8_t *keys, *values;
    const float *key_scale, *value_scale;
    int64_t k_page, k_head, k_tok, v_page, v_head, v_tok;      // strides in bytes
    const int32_t *table, *offsets, *lengths;
    int64_t table_stride;
    int seqs, rows, pages, kv_heads, dim, shift, e4m3;
    int reach;                                                 // positions that the table can name
};

// Answers an error where the two do not fit what the header says.
int take_paged(const char *who, const odl_fp8_paged_cache *cache, const odl_fp8_paged_batch *batch, Paged &to);

// Strides [row, head] of new queries, keys or values.
int check_strides(const char *who, const char *name, const void *p, const int64_t *strides, int64_t rows);

// New tokens of a sequence: rows first to first + n, n = 0 where the offsets say nothing sensible.
struct Run {
    int first, n;
};
__device__ __forceinline__ Run run_of(const Paged &p, int s) {
    const int a = min(max(p.offsets[s], 0), p.rows), b = min(p.offsets[s + 1], p.rows);
    return {a, max(b - a, 0)};
}

}  // namespace odl
