// k_paged_attn.cu -- attention of one new token per sequence over a paged key-value cache
// (include/cfi_serve.h): out = sum_j softmax_j(scale q.K_j) V_j over the sequence's positions.
//
// One warp walks every fourth position of a (sequence, head) with a running maximum and sum; the four
// meet in shared memory.
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <stdlib.h>
#include <string.h>

namespace {

constexpr int PA_WARPS = 4;

struct PaArgs {
    const uint8_t *k, *v, *q;
    uint8_t* out;
    const int32_t *table, *lens;
    long long q_stride, out_stride;
    int n_pages, page_shift, n_kv_head, group, max_pages, q_f16, out_f16;
    float scale;
};

template <int D, bool Q8> CFI_DEV float cached(const uint8_t* region, int page_size, int off, int d) {
    if (!Q8) return h2f_bits(*reinterpret_cast<const uint16_t*>(region + ((size_t)off * D + d) * 2));
    const float s = h2f_bits(*reinterpret_cast<const uint16_t*>(region + (size_t)D * page_size + ((size_t)off * (D / 32) + d / 32) * 2));
    return s * (float)*reinterpret_cast<const int8_t*>(region + (size_t)off * D + d);
}

template <int D, bool Q8>
__global__ void __launch_bounds__(PA_WARPS * 32) paged_attn(const PaArgs a) {
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    constexpr int E = D / 32;
    __shared__ float sm[PA_WARPS], sl[PA_WARPS], so[PA_WARPS][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = blockIdx.x, seq = blockIdx.y, kvh = head / a.group;
    const int page_size = 1 << a.page_shift;
    const int len = min(a.lens[seq], (int)min((long long)a.max_pages << a.page_shift, 0x7fffffffLL));
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const long long at = seq * a.q_stride + head * D + e * 32 + lane;
        q[e] = a.q_f16 ? h2f_bits(reinterpret_cast<const uint16_t*>(a.q)[at]) : reinterpret_cast<const float*>(a.q)[at];
        o[e] = 0.0f;
    }
    for (int j = warp; j < len; j += PA_WARPS) {
        const int page = min(max(a.table[(long long)seq * a.max_pages + (j >> a.page_shift)], 0), a.n_pages - 1);
        const long long region = ((long long)page * a.n_kv_head + kvh) * paged_region_bytes<D, Q8>(page_size);
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) s += q[e] * cached<D, Q8>(a.k + region, page_size, j & (page_size - 1), e * 32 + lane);
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : expf(m - mn), p = s == -INFINITY ? 0.0f : expf(s - mn);
        l = l * c + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * c + p * cached<D, Q8>(a.v + region, page_size, j & (page_size - 1), e * 32 + lane);
        m = mn;
    }
    if (lane == 0) {
        sm[warp] = m;
        sl[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < E; e++) so[warp][e * 32 + lane] = o[e];
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += PA_WARPS * 32) {
        float mm = -INFINITY, ll = 0.0f, oo = 0.0f;
        for (int w = 0; w < PA_WARPS; w++) mm = fmaxf(mm, sm[w]);
        for (int w = 0; w < PA_WARPS; w++) {
            const float c = sm[w] == -INFINITY ? 0.0f : expf(sm[w] - mm);
            ll += c * sl[w];
            oo += c * so[w][d];
        }
        const float r = ll > 0.0f ? oo / ll : oo;
        const long long at = seq * a.out_stride + head * D + d;
        if (a.out_f16)
            reinterpret_cast<uint16_t*>(a.out)[at] = f2h_bits(r);
        else
            reinterpret_cast<float*>(a.out)[at] = r;
    }
}

}  // namespace

extern "C" int cfi_paged_attention(const CfiPagedCache* c, const void* q, int q_type, long long q_stride, void* out,
                                   int out_type, long long out_stride, const int32_t* table, int max_pages,
                                   const int32_t* lens, int n_seq, int n_head, float scale, void* stream) {
    if (!cfi_paged_ok(c) || !q || !out || !table || !lens || (q_type != 0 && q_type != 1) || (out_type != 0 && out_type != 1) ||
        n_seq < 0 || n_seq > 65535 || max_pages <= 0 || n_head <= 0 || n_head % c->n_kv_head ||
        (((uintptr_t)q | (uintptr_t)out) & 15) || (((uintptr_t)table | (uintptr_t)lens) & 3) || q_stride % 8 || out_stride % 8 ||
        q_stride < (long long)n_head * c->head_dim || out_stride < (long long)n_head * c->head_dim)
        return (int)cudaErrorInvalidValue;
    if (n_seq == 0) return 0;
    PaArgs a;
    a.k = static_cast<const uint8_t*>(c->k);
    a.v = static_cast<const uint8_t*>(c->v);
    a.q = static_cast<const uint8_t*>(q);
    a.out = static_cast<uint8_t*>(out);
    a.table = table;
    a.lens = lens;
    a.q_stride = q_stride;
    a.out_stride = out_stride;
    a.n_pages = c->n_pages;
    a.page_shift = __builtin_ctz((unsigned)c->page_size);
    a.n_kv_head = c->n_kv_head;
    a.group = n_head / c->n_kv_head;
    a.max_pages = max_pages;
    a.q_f16 = q_type;
    a.out_f16 = out_type;
    a.scale = scale;
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(n_head, n_seq, 1);
    lc.blockDim = dim3(PA_WARPS * 32, 1, 1);
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    const void* fn = c->head_dim == 64 ? (c->type == 1 ? (const void*)paged_attn<64, false> : (const void*)paged_attn<64, true>)
                                       : (c->type == 1 ? (const void*)paged_attn<128, false> : (const void*)paged_attn<128, true>);
    void* args[1] = {&a};
    return (int)cudaLaunchKernelExC(&lc, fn, args);
}
