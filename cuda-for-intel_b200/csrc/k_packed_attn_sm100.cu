// k_packed_attn_sm100.cu -- causal attention of packed sequences (include/cfi_serve.h).
//
// One warp per (query, head) walks the keys it sees with a running maximum and sum.
#include "../../include/cfi_serve.h"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <stdlib.h>
#include <string.h>

namespace {

constexpr int KA_WARPS = 4;

template <int D>
__global__ void __launch_bounds__(KA_WARPS * 32) packed_attn(const CfiPackedAttention a) {
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    constexpr int E = D / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x * KA_WARPS + warp, head = blockIdx.y, kvh = head / (a.n_head / a.n_kv_head);
    if (t >= min(a.n_q, a.cu_q[a.n_seq])) return;
    int lo = 0, hi = a.n_seq;  // the sequence: cu_q[lo] <= t < cu_q[lo + 1]
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (a.cu_q[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    const int q0 = a.cu_q[lo], nq = min(a.cu_q[lo + 1], a.n_q) - q0;
    const int k0 = max(a.cu_kv[lo], 0), k1 = min(a.cu_kv[lo + 1], a.n_kv), nk = k1 - k0;
    const int seen = a.causal ? min(nk, t - q0 + nk - nq + 1) : nk;
    const __half* qp = static_cast<const __half*>(a.q) + t * a.q_stride + head * D;
    float q[E], o[E], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int e = 0; e < E; e++) {
        q[e] = __half2float(qp[e * 32 + lane]);
        o[e] = 0.0f;
    }
    for (int j = 0; j < seen; j++) {
        const __half* kp = static_cast<const __half*>(a.k) + (k0 + j) * a.k_stride + kvh * D;
        const __half* vp = static_cast<const __half*>(a.v) + (k0 + j) * a.v_stride + kvh * D;
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < E; e++) s += q[e] * __half2float(kp[e * 32 + lane]);
        s = warp_sum(s) * a.scale;
        const float mn = fmaxf(m, s), c = m == -INFINITY ? 0.0f : expf(m - mn), p = s == -INFINITY ? 0.0f : expf(s - mn);
        l = l * c + p;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] = o[e] * c + p * __half2float(vp[e * 32 + lane]);
        m = mn;
    }
#pragma unroll
    for (int e = 0; e < E; e++) {
        const float r = l > 0.0f ? o[e] / l : o[e];
        const long long at = t * a.out_stride + head * D + e * 32 + lane;
        if (a.out_type == 1)
            static_cast<__half*>(a.out)[at] = __float2half_rn(r);
        else
            static_cast<float*>(a.out)[at] = r;
    }
}

}  // namespace

extern "C" int cfi_packed_attention(const CfiPackedAttention* a, void* stream) {
    if (!a || !a->q || !a->k || !a->v || !a->out || !a->cu_q || !a->cu_kv || a->n_seq < 0 || a->n_seq > 65535 || a->n_q < 0 ||
        a->n_kv < 0 || a->n_head <= 0 || a->n_kv_head <= 0 || a->n_head % a->n_kv_head || a->n_head / a->n_kv_head > 128 ||
        a->n_head > 65535 || (a->head_dim != 64 && a->head_dim != 128) || (a->out_type != 0 && a->out_type != 1))
        return (int)cudaErrorInvalidValue;
    const long long wq = (long long)a->n_head * a->head_dim, wk = (long long)a->n_kv_head * a->head_dim;
    if ((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) & 15) ||
        (((uintptr_t)a->cu_q | (uintptr_t)a->cu_kv) & 3) || (a->q_stride | a->k_stride | a->v_stride | a->out_stride) % 8 ||
        a->q_stride < wq || a->out_stride < wq || a->k_stride < wk || a->v_stride < wk)
        return (int)cudaErrorInvalidValue;
    if (a->n_seq == 0 || a->n_q == 0) return 0;
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((a->n_q + KA_WARPS - 1) / KA_WARPS, a->n_head, 1);
    lc.blockDim = dim3(KA_WARPS * 32, 1, 1);
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    void* args[1] = {const_cast<CfiPackedAttention*>(a)};
    return (int)cudaLaunchKernelExC(&lc, a->head_dim == 64 ? (const void*)packed_attn<64> : (const void*)packed_attn<128>, args);
}
