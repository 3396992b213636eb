// paged_cache.cuh -- the layout of a paged key-value cache (include/cfi_serve.h) as the kernels that
// write and read it see it, and the host checks of its description.
#pragma once
#include "../../include/cfi_serve.h"
#include "cfi_common.cuh"

// Bytes of one (page, kv head) region: f16 rows, or int8 rows and behind them their f16 scales.
// A multiple of 16 for every page size (16 positions of 64 values: 1024 + 64 bytes).
template <int D, bool Q8> CFI_DEV long long paged_region_bytes(int page_size) {
    return Q8 ? (long long)page_size * (D + D / 16) : (long long)page_size * D * 2;
}

inline bool cfi_paged_shape_ok(const CfiPagedCache* c) {
    return (c->type == 1 || c->type == 8) && (c->head_dim == 64 || c->head_dim == 128) && c->page_size >= 16 &&
           c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0 && c->n_pages > 0 && c->n_kv_head > 0 &&
           c->n_kv_head <= 1024;
}
inline bool cfi_paged_ok(const CfiPagedCache* c) {
    return c && cfi_paged_shape_ok(c) && c->k && c->v && !(((uintptr_t)c->k | (uintptr_t)c->v) & 15);
}
