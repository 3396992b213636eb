// k_paged_cache.cu -- writing rows of K and V into the pages of a serving cache (quantised to Q8_0 or
// Q4_1 where the cache is, paged_row.cuh) and reading them back as f16.  include/cfi_serve.h gives the layout.
// Four neighbouring threads, 8 values each, make a block of 32.
#include "paged_row.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <stdlib.h>
#include <string.h>

namespace {

// Items of a thread.  Measured with 1, 2 and 4 (f16 rows of 8 x 128, Q8_0 pages): reading back 65537 rows 78, 65.9
// (6.2 TB/s of reads and writes) and 80 us; storing 8192 rows 12.7, 12.7 and 13.8 us (10.3, 5 TB/s, since the maximum of f16
// rows is taken in f16 and the bytes come from one conversion: it is bound by issue), a step's 48 rows 1.2, 1.5 and 1.9.
constexpr int PC_THREADS = 256, PC_STORE_ITEMS = 1, PC_LOAD_ITEMS = 2;
// Q4_1: reading back 65537 rows 52 us (6.7 TB/s of reads and writes), storing 8192 f16 rows 21 (17 from L2): bound by issue, 390 instructions of a
// warp for 8 values of K and of V a lane; of f16 values one of a warp is nearly always near a border, so that
// both ways of paged_row.cuh are gone.  With two items a thread 73.3 us become 72.4, and a step's 48 rows 3.6 become 4.3.
constexpr int PC_Q4_ITEMS = 1;

struct PcArgs {
    uint8_t *k, *v;          // pools
    const int64_t* slots;
    const uint8_t *src_k, *src_v;  // store: rows in
    uint8_t *dst_k, *dst_v;        // load: rows out
    long long k_stride, v_stride;  // values
    long long n_slots;
    uint32_t n_items;        // tokens x kv heads x D / 8
    int page_shift, n_kv_head;
};

CFI_DEV uint4 ldg_stream(const void* p) {  // read once: do not keep it in L1
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

CFI_DEV uint2 ldg_stream2(const void* p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// An item is 8 values of a (token, kv head) row, of K and of V.  A thread has one or two of them, and all their
// loads are issued before the first is used: first the slots, then the rows.
template <int D> struct PcPlace {
    uint32_t t, h, g;
    bool in;
    long long slot;
    CFI_DEV void at(const PcArgs& a, uint32_t i) {
        in = i < a.n_items;
        const uint32_t row = (in ? i : a.n_items - 1) / (D / 8);
        g = i % (D / 8);
        t = row / a.n_kv_head;
        h = row - t * a.n_kv_head;
        slot = a.slots[t];
    }
    CFI_DEV bool ok(const PcArgs& a) const { return in && slot >= 0 && slot < a.n_slots; }
    template <int TY> CFI_DEV long long region(const PcArgs& a) const {
        return ((slot >> a.page_shift) * a.n_kv_head + h) * paged_region_bytes<D, TY>(1 << a.page_shift);
    }
    CFI_DEV int off(const PcArgs& a) const { return (int)(slot & ((1 << a.page_shift) - 1)); }
    CFI_DEV long long value(long long stride) const { return (long long)t * stride + h * D + g * 8; }
};

template <int D, int TY, bool SRC_F16>
__global__ void __launch_bounds__(PC_THREADS) paged_kv_store(const PcArgs a) {
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    const uint32_t base = blockIdx.x * (PC_THREADS * PC_STORE_ITEMS) + threadIdx.x;
    PcPlace<D> p[PC_STORE_ITEMS];
#pragma unroll
    for (int e = 0; e < PC_STORE_ITEMS; e++) p[e].at(a, base + e * PC_THREADS);
    uint4 in[PC_STORE_ITEMS][2][SRC_F16 ? 1 : 2];
#pragma unroll
    for (int e = 0; e < PC_STORE_ITEMS; e++)
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            const uint8_t* src = (kv ? a.src_v : a.src_k) + p[e].value(kv ? a.v_stride : a.k_stride) * (SRC_F16 ? 2 : 4);
#pragma unroll
            for (int j = 0; j < (SRC_F16 ? 1 : 2); j++) in[e][kv][j] = ldg_stream(src + 16 * j);
        }
#pragma unroll
    for (int e = 0; e < PC_STORE_ITEMS; e++)
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            uint8_t* region = (kv ? a.v : a.k) + p[e].template region<TY>(a);
            Row8 r;
            r.h = in[e][kv][0];
            if (SRC_F16) {
                const __half2* h = reinterpret_cast<const __half2*>(&r.h);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = __half22float2(h[j]);
                    r.x[2 * j] = f.x;
                    r.x[2 * j + 1] = f.y;
                }
            } else {
                const uint4 hi = in[e][kv][SRC_F16 ? 0 : 1];
                const uint32_t w[8] = {r.h.x, r.h.y, r.h.z, r.h.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int j = 0; j < 8; j++) r.x[j] = __uint_as_float(w[j]);
                __half2* h = reinterpret_cast<__half2*>(&r.h);
#pragma unroll
                for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(r.x[2 * j], r.x[2 * j + 1]);
            }
            put_row8<D, TY, SRC_F16>(r, region, a.page_shift, p[e].off(a), p[e].g, kv == 1, p[e].ok(a));
        }
}

template <int D, int TY>
__global__ void __launch_bounds__(PC_THREADS) paged_kv_load(const PcArgs a) {
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    const uint32_t base = blockIdx.x * (PC_THREADS * PC_LOAD_ITEMS) + threadIdx.x;
    PcPlace<D> p[PC_LOAD_ITEMS];
#pragma unroll
    for (int e = 0; e < PC_LOAD_ITEMS; e++) p[e].at(a, base + e * PC_THREADS);
    uint4 in[PC_LOAD_ITEMS][2];
    uint32_t scale[PC_LOAD_ITEMS][2];
#pragma unroll
    for (int e = 0; e < PC_LOAD_ITEMS; e++)
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            in[e][kv] = make_uint4(0, 0, 0, 0);
            scale[e][kv] = 0;
            if (!p[e].ok(a)) continue;
            const uint8_t* region = (kv ? a.v : a.k) + p[e].template region<TY>(a);
            const int off = p[e].off(a);
            if (TY == CACHE_Q8_0) {
                const uint2 q = ldg_stream2(region + (size_t)off * D + p[e].g * 8);
                in[e][kv].x = q.x;
                in[e][kv].y = q.y;
                scale[e][kv] = *reinterpret_cast<const uint16_t*>(region + (size_t)(D << a.page_shift) +
                                                                  ((size_t)off * (D / 32) + p[e].g / 4) * 2);
            } else {
                in[e][kv] = ldg_stream(region + ((size_t)off * D + p[e].g * 8) * 2);
            }
        }
#pragma unroll
    for (int e = 0; e < PC_LOAD_ITEMS; e++)
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            uint4 out = in[e][kv];
            if (TY == CACHE_Q8_0) {
                const float d = h2f_bits((uint16_t)scale[e][kv]);
                __half2* o = reinterpret_cast<__half2*>(&out);
                const uint32_t w[2] = {in[e][kv].x, in[e][kv].y};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t b = w[j >> 1] >> (16 * (j & 1));
                    o[j] = __floats2half2_rn(d * (float)(int8_t)(b & 0xff), d * (float)(int8_t)((b >> 8) & 0xff));
                }
            }
            if (p[e].in) *reinterpret_cast<uint4*>((kv ? a.dst_v : a.dst_k) + p[e].value(kv ? a.v_stride : a.k_stride) * 2) = out;
        }
}

// Q4_1: an item is what lies together in a row, dims 8 c .. 8 c + 7 of all its blocks, of K and of V.
template <int D> __global__ void __launch_bounds__(PC_THREADS) paged_kv_load_q4_1(const PcArgs a) {
    using L = Q41<D>;
    constexpr int NB = D / 32, WORDS = D / 32;  // words of nibbles: block b's dims (V: its first four, then its last four in the upper halves)
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    const uint32_t base = blockIdx.x * (PC_THREADS * PC_Q4_ITEMS) + threadIdx.x;
    uint32_t w[PC_Q4_ITEMS][2][WORDS], m[PC_Q4_ITEMS][2][NB];  // nibbles; scales, then minima
    long long slot[PC_Q4_ITEMS];
    uint32_t t[PC_Q4_ITEMS], h[PC_Q4_ITEMS];
    const int c = threadIdx.x & 3;
#pragma unroll
    for (int e = 0; e < PC_Q4_ITEMS; e++) {
        const uint32_t i = base + e * PC_THREADS, row = (i < a.n_items ? i : a.n_items - 1) / 4;
        t[e] = row / a.n_kv_head;
        h[e] = row - t[e] * a.n_kv_head;
        slot[e] = a.slots[t[e]];
    }
#pragma unroll
    for (int e = 0; e < PC_Q4_ITEMS; e++) {
        const bool ok = slot[e] >= 0 && slot[e] < a.n_slots;
        const int off = (int)(slot[e] & ((1 << a.page_shift) - 1)), row = off % Q41_TILE;
        const long long tile = ((slot[e] >> a.page_shift) * a.n_kv_head + h[e]) * paged_region_bytes<D, CACHE_Q4_1>(1 << a.page_shift) + L::tile_at(off);
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            const uint8_t* p = (kv ? a.v : a.k) + tile;
            const uint8_t *q = p + (kv ? L::v_at(row, 0, 2 * c) : L::k_at(row, 0, c)), *r = p + L::scale_at(row, 0);
            if (D == 128) {
                const uint4 x = ok ? ldg_stream(q) : make_uint4(0, 0, 0, 0), y = ok ? *reinterpret_cast<const uint4*>(r) : make_uint4(0, 0, 0, 0);
                w[e][kv][0] = x.x, w[e][kv][1] = x.y, w[e][kv][WORDS - 2] = x.z, w[e][kv][WORDS - 1] = x.w;
                m[e][kv][0] = y.x, m[e][kv][1] = y.y, m[e][kv][NB - 2] = y.z, m[e][kv][NB - 1] = y.w;
            } else {
                const uint2 x = ok ? ldg_stream2(q) : make_uint2(0, 0), y = ok ? *reinterpret_cast<const uint2*>(r) : make_uint2(0, 0);
                w[e][kv][0] = x.x, w[e][kv][1] = x.y;
                m[e][kv][0] = y.x, m[e][kv][1] = y.y;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < PC_Q4_ITEMS; e++) {
        if (base + e * PC_THREADS >= a.n_items) continue;
#pragma unroll
        for (int kv = 0; kv < 2; kv++) {
            uint8_t* to = (kv ? a.dst_v : a.dst_k) + ((long long)t[e] * (kv ? a.v_stride : a.k_stride) + h[e] * D + 8 * c) * 2;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const float d = h2f_bits((uint16_t)(m[e][kv][b >> 1] >> (16 * (b & 1)))), low = h2f_bits((uint16_t)(m[e][kv][(NB + b) >> 1] >> (16 * (b & 1))));
                // V: the lane's two groups of four dims, NB half-words each
                const uint32_t x = kv ? __byte_perm(w[e][kv][b >> 1], w[e][kv][WORDS / 2 + (b >> 1)], b & 1 ? 0x7632 : 0x5410) : w[e][kv][b];
                uint4 out;
                __half2* o = reinterpret_cast<__half2*>(&out);
#pragma unroll
                for (int j = 0; j < 4; j++)
                    o[j] = __floats2half2_rn(fmaf(d, (float)(x >> (8 * j) & 15), low), fmaf(d, (float)(x >> (8 * j + 4) & 15), low));
                *reinterpret_cast<uint4*>(to + 64 * b) = out;
            }
        }
    }
}

int go(const void* fn, const PcArgs& a, int items, cudaStream_t stream) {
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((a.n_items + PC_THREADS * items - 1) / (PC_THREADS * items), 1, 1);
    c.blockDim = dim3(PC_THREADS, 1, 1);
    c.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    void* args[1] = {const_cast<PcArgs*>(&a)};
    return (int)cudaLaunchKernelExC(&c, fn, args);
}

bool rows_ok(const void* k, const void* v, long long ks, long long vs, long long width, const void* slots, int n) {
    return n >= 0 && k && v && slots && !(((uintptr_t)k | (uintptr_t)v) & 15) && !((uintptr_t)slots & 7) && ks % 8 == 0 &&
           vs % 8 == 0 && ks >= width && vs >= width;
}

bool args_of(const CfiPagedCache* c, long long ks, long long vs, const int64_t* slots, int n, PcArgs* a) {
    const long long items = (long long)n * c->n_kv_head * (c->head_dim / 8);
    if (items > 0x7fffffffLL) return false;
    a->k = static_cast<uint8_t*>(c->k);
    a->v = static_cast<uint8_t*>(c->v);
    a->slots = slots;
    a->k_stride = ks;
    a->v_stride = vs;
    a->n_slots = (long long)c->n_pages * c->page_size;
    a->n_items = (uint32_t)items;
    a->page_shift = __builtin_ctz((unsigned)c->page_size);
    a->n_kv_head = c->n_kv_head;
    return true;
}

int type_at(const CfiPagedCache* c) { return c->type == CACHE_F16 ? 0 : c->type == CACHE_Q8_0 ? 1 : 2; }

}  // namespace

extern "C" size_t cfi_paged_page_bytes(const CfiPagedCache* c) {
    if (!c || !cfi_paged_shape_ok(c)) return 0;
    const size_t row = c->type == CACHE_F16 ? (size_t)c->head_dim * 2 : (size_t)c->head_dim / 32 * (c->type == CACHE_Q8_0 ? 34 : 20);
    return (size_t)c->n_kv_head * c->page_size * row;
}

extern "C" int cfi_paged_kv_store(const CfiPagedCache* c, const void* k, const void* v, int src_type, long long k_stride,
                                  long long v_stride, const int64_t* slots, int n_tokens, void* stream) {
    PcArgs a = {};
    if (!cfi_paged_ok(c) || (src_type != 0 && src_type != 1) ||
        !rows_ok(k, v, k_stride, v_stride, (long long)c->n_kv_head * c->head_dim, slots, n_tokens) ||
        !args_of(c, k_stride, v_stride, slots, n_tokens, &a))
        return (int)cudaErrorInvalidValue;
    if (n_tokens == 0) return 0;
    a.src_k = static_cast<const uint8_t*>(k);
    a.src_v = static_cast<const uint8_t*>(v);
    static const void* const fns[12] = {
        (const void*)paged_kv_store<64, CACHE_F16, false>,   (const void*)paged_kv_store<64, CACHE_F16, true>,
        (const void*)paged_kv_store<64, CACHE_Q8_0, false>,  (const void*)paged_kv_store<64, CACHE_Q8_0, true>,
        (const void*)paged_kv_store<64, CACHE_Q4_1, false>,  (const void*)paged_kv_store<64, CACHE_Q4_1, true>,
        (const void*)paged_kv_store<128, CACHE_F16, false>,  (const void*)paged_kv_store<128, CACHE_F16, true>,
        (const void*)paged_kv_store<128, CACHE_Q8_0, false>, (const void*)paged_kv_store<128, CACHE_Q8_0, true>,
        (const void*)paged_kv_store<128, CACHE_Q4_1, false>, (const void*)paged_kv_store<128, CACHE_Q4_1, true>};
    return go(fns[(c->head_dim == 128) * 6 + type_at(c) * 2 + src_type], a, PC_STORE_ITEMS, static_cast<cudaStream_t>(stream));
}

extern "C" int cfi_paged_kv_load(const CfiPagedCache* c, const int64_t* slots, void* k, void* v, long long k_stride,
                                 long long v_stride, int n_tokens, void* stream) {
    PcArgs a = {};
    if (!cfi_paged_ok(c) || !rows_ok(k, v, k_stride, v_stride, (long long)c->n_kv_head * c->head_dim, slots, n_tokens) ||
        !args_of(c, k_stride, v_stride, slots, n_tokens, &a))
        return (int)cudaErrorInvalidValue;
    if (n_tokens == 0) return 0;
    a.dst_k = static_cast<uint8_t*>(k);
    a.dst_v = static_cast<uint8_t*>(v);
    if (c->type == CACHE_Q4_1) {
        a.n_items = a.n_items / (c->head_dim / 8) * 4;
        return go(c->head_dim == 128 ? (const void*)paged_kv_load_q4_1<128> : (const void*)paged_kv_load_q4_1<64>, a, PC_Q4_ITEMS,
                  static_cast<cudaStream_t>(stream));
    }
    static const void* const fns[4] = {(const void*)paged_kv_load<64, CACHE_F16>, (const void*)paged_kv_load<64, CACHE_Q8_0>,
                                       (const void*)paged_kv_load<128, CACHE_F16>, (const void*)paged_kv_load<128, CACHE_Q8_0>};
    return go(fns[(c->head_dim == 128) * 2 + type_at(c)], a, PC_LOAD_ITEMS, static_cast<cudaStream_t>(stream));
}
