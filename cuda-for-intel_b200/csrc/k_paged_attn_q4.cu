// k_paged_attn_q4.cu -- attention of one new token per sequence over a Q4_1 cache (include/cfi_serve.h):
// out = sum_j softmax_j(scale q.K_j) V_j with K_j = d n + m in each block of 32 dims, so that
//   q.K_j = sum_b d_jb (sum_i q_i n_ji) + m_jb (sum_i q_i),  o = sum_j p_j d_jb n_ji + p_j m_jb.
//
// A CTA has a (sequence, kv head, chunk of 8 query heads); its warps take every fourth position.
#include "paged_attn.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

namespace {

template <int D> __global__ void __launch_bounds__(PA_WARPS * 32) paged_attn_q4(const PaArgs a) {
    constexpr int E = D / 32;  // dims of a lane
    __shared__ float meet[PA_WARPS][PA_HEADS][D + 2];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, hc = a.n_kv_head * a.chunks;
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    const int seq = blockIdx.x / hc, pair = blockIdx.x % hc;
    const int kvh = pair / a.chunks, h0 = (pair - kvh * a.chunks) * PA_HEADS, nh = min(PA_HEADS, a.group - h0);
    const int head0 = kvh * a.group + h0, page_size = 1 << a.page_shift;
    const int len = (int)min((long long)max(a.lens[seq], 0), (long long)a.max_pages << a.page_shift);
    const int dim = lane * E, b = dim / 32;
    float q[PA_HEADS][E], o[PA_HEADS][E], m[PA_HEADS], l[PA_HEADS];
#pragma unroll
    for (int h = 0; h < PA_HEADS; h++) {
        m[h] = -INFINITY;
        l[h] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) {
            const long long at = seq * a.q_stride + (long long)(head0 + h) * D + dim + e;
            o[h][e] = 0.0f;
            q[h][e] = h >= nh ? 0.0f
                      : (a.q_f16 ? __half2float(reinterpret_cast<const __half*>(a.q)[at]) : reinterpret_cast<const float*>(a.q)[at]) * a.scale_log2;
        }
    }
    for (int j = warp; j < len; j += PA_WARPS) {
        const int page = min(max(a.table[(long long)seq * a.max_pages + (j >> a.page_shift)], 0), a.n_pages - 1), off = j & (page_size - 1);
        const long long region = ((long long)page * a.n_kv_head + kvh) * paged_region_bytes<D, CACHE_Q4_1>(page_size) + Q41<D>::tile_at(off);
        const int row = off % Q41_TILE;
        const uint8_t *tk = a.k + region, *tv = a.v + region;
        const float dk = __half2float(*reinterpret_cast<const __half*>(tk + Q41<D>::scale_at(row, b))),
                    mk = __half2float(*reinterpret_cast<const __half*>(tk + Q41<D>::min_at(row, b))),
                    dv = __half2float(*reinterpret_cast<const __half*>(tv + Q41<D>::scale_at(row, b))),
                    mv = __half2float(*reinterpret_cast<const __half*>(tv + Q41<D>::min_at(row, b)));
        float k[E], v[E];
#pragma unroll
        for (int e = 0; e < E; e++) {
            const int i = (dim + e) % 32;
            k[e] = fmaf(dk, (float)(tk[Q41<D>::k_at(row, b, i / 8) + i % 8 / 2] >> 4 * (i & 1) & 15), mk);
            v[e] = fmaf(dv, (float)(tv[Q41<D>::v_at(row, b, i / 4) + i % 4 / 2] >> 4 * (i & 1) & 15), mv);
        }
#pragma unroll
        for (int h = 0; h < PA_HEADS; h++) {
            float s = 0.0f;
#pragma unroll
            for (int e = 0; e < E; e++) s = fmaf(q[h][e], k[e], s);
            s = warp_sum(s);
            const float mn = fmaxf(m[h], s), f = m[h] == -INFINITY ? 0.0f : ex2(m[h] - mn), p = ex2(s - (mn == -INFINITY ? 0.0f : mn));
            m[h] = mn;
            l[h] = fmaf(l[h], f, p);
#pragma unroll
            for (int e = 0; e < E; e++) o[h][e] = fmaf(o[h][e], f, p * v[e]);
        }
    }
#pragma unroll
    for (int h = 0; h < PA_HEADS; h++) {
#pragma unroll
        for (int e = 0; e < E; e++) meet[warp][h][dim + e] = o[h][e];
        if (lane == 0) {
            meet[warp][h][D] = m[h];
            meet[warp][h][D + 1] = l[h];
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < nh * (D / 4); i += PA_WARPS * 32) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float mm = -INFINITY, ll = 0.0f;
        float4 oo = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < PA_WARPS; w++) mm = fmaxf(mm, meet[w][h][D]);
#pragma unroll
        for (int w = 0; w < PA_WARPS; w++) {
            const float* p = meet[w][h];
            const float f = p[D] == -INFINITY ? (p[D + 1] != p[D + 1] ? p[D + 1] : 0.0f) : ex2(p[D] - mm);
            ll = fmaf(f, p[D + 1], ll);
            add_to(oo, f, make_float4(p[d], p[d + 1], p[d + 2], p[d + 3]));
        }
        write_out(a, seq, head0 + h, D, d, oo, ll);
    }
}

}  // namespace

int cfi_paged_attention_q4_1(PaArgs& a, int head_dim, long long pairs, cudaStream_t stream) {
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)pairs, 1, 1);
    lc.blockDim = dim3(PA_WARPS * 32, 1, 1);
    lc.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    return (int)(head_dim == 64 ? cudaLaunchKernelEx(&lc, paged_attn_q4<64>, (const PaArgs)a) : cudaLaunchKernelEx(&lc, paged_attn_q4<128>, (const PaArgs)a));
}
