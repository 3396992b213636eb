// k_paged_cache.cu -- writing rows of K and V into the pages of a serving cache (quantised to Q8_0
// where the cache is) and reading them back as f16.  include/cfi_serve.h gives the layout.
//
// Per block of 32 values x: d = max|x| / 127, q = rn(x * (1/d)), stored scale f16(d); read back as
// f16(q * scale).  Four neighbouring threads, 8 values each, make a block.
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <stdlib.h>
#include <string.h>

namespace {

// Items of a thread.  Measured with 1, 2 and 4 (f16 rows of 8 x 128, Q8_0 pages): reading back 65537 rows 78, 65.9
// (6.2 TB/s of reads and writes) and 80 us; storing 8192 rows 12.7, 12.7 and 13.8 us (10.3, 5 TB/s, since the maximum of f16
// rows is taken in f16 and the bytes come from one conversion: it is bound by issue), a step's 48 rows 1.2, 1.5 and 1.9.
constexpr int PC_THREADS = 256, PC_STORE_ITEMS = 1, PC_LOAD_ITEMS = 2;

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
    template <bool Q8> CFI_DEV long long region(const PcArgs& a) const {
        return ((slot >> a.page_shift) * a.n_kv_head + h) * paged_region_bytes<D, Q8>(1 << a.page_shift);
    }
    CFI_DEV int off(const PcArgs& a) const { return (int)(slot & ((1 << a.page_shift) - 1)); }
    CFI_DEV long long value(long long stride) const { return (long long)t * stride + h * D + g * 8; }
};

CFI_DEV __half2 abs_h2(uint32_t w) {
    w &= 0x7fff7fffu;
    return *reinterpret_cast<const __half2*>(&w);
}
CFI_DEV int to_s8(float x) {  // to the nearest, ties to even; the ends at +-128, a NaN 0
    int q;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(q) : "f"(x));
    return q;
}
CFI_DEV uint32_t bytes_of(int a, int b, int c, int d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <int D, bool Q8, bool SRC_F16>
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
            const bool ok = p[e].ok(a);
            uint8_t* region = (kv ? a.v : a.k) + p[e].template region<Q8>(a);
            const int off = p[e].off(a);
            float x[8];
            uint4 raw = in[e][kv][0];
            if (SRC_F16) {
                const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float2 f = __half22float2(h[j]);
                    x[2 * j] = f.x;
                    x[2 * j + 1] = f.y;
                }
            } else {
                const uint4 hi = in[e][kv][SRC_F16 ? 0 : 1];
                const uint32_t w[8] = {raw.x, raw.y, raw.z, raw.w, hi.x, hi.y, hi.z, hi.w};
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = __uint_as_float(w[j]);
                __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
                for (int j = 0; j < 4; j++) h[j] = __floats2half2_rn(x[2 * j], x[2 * j + 1]);
            }
            if (!Q8) {
                if (ok) *reinterpret_cast<uint4*>(region + ((size_t)off * D + p[e].g * 8) * 2) = raw;
                continue;
            }
            float m;  // of a block that has a NaN: NaN, and so its scale
            if (SRC_F16) {
                __half2 h = abs_h2(raw.x);
                h = __hmax2_nan(__hmax2_nan(h, abs_h2(raw.y)), __hmax2_nan(abs_h2(raw.z), abs_h2(raw.w)));
                h = __hmax2_nan(h, __lowhigh2highlow(h));
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) h = __hmax2_nan(h, __shfl_xor_sync(0xffffffffu, h, o));
                m = __low2float(h);
            } else {
                m = 0.0f;
                uint32_t nan = 0;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    m = fmaxf(m, fabsf(x[j]));  // drops a NaN
                    nan |= (uint32_t)(x[j] != x[j]);
                }
                if (nan) m = __uint_as_float(0x7fffffffu);
#pragma unroll
                for (int o = 1; o < 4; o <<= 1) {
                    const float other = __shfl_xor_sync(0xffffffffu, m, o);
                    m = other != other ? other : m != m ? m : fmaxf(m, other);
                }
            }
            const float d = m / 127.0f, id = d > 0.0f ? 1.0f / d : 0.0f;
            int q[8];
#pragma unroll
            for (int j = 0; j < 8; j++) q[j] = to_s8(x[j] * id);
            const uint32_t w[2] = {bytes_of(q[0], q[1], q[2], q[3]), bytes_of(q[4], q[5], q[6], q[7])};
            if (!ok) continue;
            *reinterpret_cast<uint2*>(region + (size_t)off * D + p[e].g * 8) = make_uint2(w[0], w[1]);
            if ((p[e].g & 3) == 0)
                *reinterpret_cast<uint16_t*>(region + (size_t)(D << a.page_shift) + ((size_t)off * (D / 32) + p[e].g / 4) * 2) =
                    d != d ? (uint16_t)0x7fff : f2h_bits(d);
        }
}

template <int D, bool Q8>
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
            const uint8_t* region = (kv ? a.v : a.k) + p[e].template region<Q8>(a);
            const int off = p[e].off(a);
            if (Q8) {
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
            if (Q8) {
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

}  // namespace

extern "C" size_t cfi_paged_page_bytes(const CfiPagedCache* c) {
    if (!c || !cfi_paged_shape_ok(c)) return 0;
    return (size_t)c->n_kv_head * c->page_size * (c->type == 1 ? (size_t)c->head_dim * 2 : (size_t)c->head_dim / 32 * 34);
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
    static const void* const fns[8] = {
        (const void*)paged_kv_store<64, false, false>,  (const void*)paged_kv_store<64, false, true>,
        (const void*)paged_kv_store<64, true, false>,   (const void*)paged_kv_store<64, true, true>,
        (const void*)paged_kv_store<128, false, false>, (const void*)paged_kv_store<128, false, true>,
        (const void*)paged_kv_store<128, true, false>,  (const void*)paged_kv_store<128, true, true>};
    return go(fns[(c->head_dim == 128) * 4 + (c->type == 8) * 2 + src_type], a, PC_STORE_ITEMS, static_cast<cudaStream_t>(stream));
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
    static const void* const fns[4] = {(const void*)paged_kv_load<64, false>, (const void*)paged_kv_load<64, true>,
                                       (const void*)paged_kv_load<128, false>, (const void*)paged_kv_load<128, true>};
    return go(fns[(c->head_dim == 128) * 2 + (c->type == 8)], a, PC_LOAD_ITEMS, static_cast<cudaStream_t>(stream));
}
