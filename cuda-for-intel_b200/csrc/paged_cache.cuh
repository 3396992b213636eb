// paged_cache.cuh -- the layout of a paged key-value cache (include/cfi_serve.h) as the kernels that
// write and read it see it, and the host checks of its description.
#pragma once
#include "../../include/cfi_serve.h"
#include "cfi_common.cuh"

enum CacheType { CACHE_F16 = 1, CACHE_Q4_1 = 3, CACHE_Q8_0 = 8 };

// Bytes of one (page, kv head) region: f16 rows; int8 rows and behind them their f16 scales; or tiles of Q4_1.
// A multiple of 16 for every page size (16 positions of 64 values: 1024 + 64 bytes).
template <int D, int TY> CFI_DEV long long paged_region_bytes(int page_size) {
    return TY == CACHE_Q8_0 ? (long long)page_size * (D + D / 16)
           : TY == CACHE_Q4_1 ? (long long)page_size * (D / 2 + D / 8)
                              : (long long)page_size * D * 2;
}

// A Q4_1 tile: 16 rows of nibbles, then 16 rows of scales and minima.
constexpr int Q41_TILE = 16;
template <int D> struct Q41 {
    static constexpr int ROW = D / 2, NIBBLES = Q41_TILE * ROW, PARAM_ROW = D / 8, TILE = NIBBLES + Q41_TILE * PARAM_ROW;
    static CFI_DEV int tile_at(int off) { return off / Q41_TILE * TILE; }
    // of the four bytes of K, dims 32 b + 8 c .. + 7
    static CFI_DEV int k_at(int row, int b, int c) { return row * ROW + c * (D / 8) + b * 4; }
    // of the two bytes of V, dims 32 b + 4 g .. + 3; rows of 64 bytes change places so that a warp's reads meet no bank twice
    static CFI_DEV int v_group(int row, int g) { return D == 128 ? g ^ (row & 2) << 1 : g; }
    static CFI_DEV int v_at(int row, int b, int g) { return row * ROW + v_group(row, g) * (D / 16) + b * 2; }
    static CFI_DEV int scale_at(int row, int b) { return NIBBLES + row * PARAM_ROW + b * 2; }
    static CFI_DEV int min_at(int row, int b) { return scale_at(row, b) + D / 16; }
};

CFI_DEV __half2 abs_h2(uint32_t w) {
    w &= 0x7fff7fffu;
    return *reinterpret_cast<const __half2*>(&w);
}

inline bool cfi_paged_shape_ok(const CfiPagedCache* c) {
    return (c->type == CACHE_F16 || c->type == CACHE_Q4_1 || c->type == CACHE_Q8_0) && (c->head_dim == 64 || c->head_dim == 128) &&
           c->page_size >= 16 && c->page_size <= 256 && (c->page_size & (c->page_size - 1)) == 0 && c->n_pages > 0 &&
           c->n_kv_head > 0 && c->n_kv_head <= 1024;
}
inline bool cfi_paged_ok(const CfiPagedCache* c) {
    return c && cfi_paged_shape_ok(c) && c->k && c->v && !(((uintptr_t)c->k | (uintptr_t)c->v) & 15);
}
