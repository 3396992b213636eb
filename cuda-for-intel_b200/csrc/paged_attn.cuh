// paged_attn.cuh -- what the kernels of the single-token attention over a paged cache share (k_paged_attn.cu for f16 and
// Q8_0, k_paged_attn_q4.cu for Q4_1): arguments, the cut of the list into runs, the join of partial results.
#pragma once
#include "paged_cache.cuh"
#include "paged_cut.h"
#include "mma_sync.cuh"

constexpr int PA_WARPS = 4;  // of a CTA; twice as many where a CTA has a pair and an SM to itself
constexpr int PA_HEADS = 8;  // query heads of a chunk

struct PaArgs {
    const uint8_t *k, *v, *q;
    uint8_t* out;
    const int32_t *table, *lens;
    float* parts;            // [2 x CTAs][PART]
    unsigned int* counters;  // [sequence][pair]: zero between calls
    long long q_stride, out_stride;
    int n_pages, page_shift, n_kv_head, group, chunks, max_pages, n_seq, q_f16, out_f16;
    int whole;  // a CTA to a pair
    float scale_log2;
};

CFI_DEV float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
CFI_DEV void cp16z(uint32_t dst, const void* src, bool take) {  // 16 bytes, or 16 zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
CFI_DEV void cp8z(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(src), "r"(take ? 8 : 0) : "memory");
}
CFI_DEV void cp4z(uint32_t dst, const void* src, bool take) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(take ? 4 : 0) : "memory");
}
CFI_DEV void ldsm_x4_trans(uint32_t a, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(a));
}
CFI_DEV void mma_f16f32(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
CFI_DEV uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
// (x, y) as f16 and what the rounding left, as f16: 22 bits together
CFI_DEV void split(float x, float y, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    *hi = h2_bits(h);
    *lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}
CFI_DEV void add_to(float4& x, float f, const float4& y) {
    x.x = fmaf(f, y.x, x.x);
    x.y = fmaf(f, y.y, x.y);
    x.z = fmaf(f, y.z, x.z);
    x.w = fmaf(f, y.w, x.w);
}
// Four values of a head's row, over the sum of its weights.
CFI_DEV void write_out(const PaArgs& a, int seq, int head, int dim, int d, float4 v, float sum) {
    const float r = sum == 0.0f ? 0.0f : 1.0f / sum;
    if (sum == 0.0f) v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const long long w = seq * a.out_stride + (long long)head * dim + d;
    if (a.out_f16)
        *reinterpret_cast<uint2*>(a.out + w * 2) =
            make_uint2(h2_bits(__floats2half2_rn(v.x * r, v.y * r)), h2_bits(__floats2half2_rn(v.z * r, v.w * r)));
    else
        *reinterpret_cast<float4*>(a.out + w * 4) = make_float4(v.x * r, v.y * r, v.z * r, v.w * r);
}

// How the work is cut: a pair (kv head, chunk) of a sequence is FIXED units (what beginning and ending it costs, in tiles, so that
// CTAs with many short sequences get fewer tiles) and then one for each tile of TILE positions, the pairs of all sequences follow
// one another, and CTA b has the units b * quota .. (b + 1) * quota.  There are less than 2^31.
constexpr int PA_KEPT = 4;
template <int TILE, int FIXED> struct PaCut {
    const int32_t* lens;
    int most, total, quota;
    int units[PA_KEPT];  // of the sequences that are this lane's, of the first 32 PA_KEPT, all loaded together
    CFI_DEV int length(int s) const { return max(0, min(lens[s], most)); }
    // an empty sequence still has its zeros to write
    static CFI_DEV int tiles_of(int len) { return max(1, (len + TILE - 1) / TILE); }
    CFI_DEV int units_of(int s) const { return FIXED + tiles_of(length(s)); }
    CFI_DEV explicit PaCut(const PaArgs& a)
        : lens(a.lens), most((int)min((long long)a.max_pages << a.page_shift, 0x7fffff00LL)) {}
    // Called by whole warps.
    CFI_DEV void read(const PaArgs& a, int ctas) {
        const int lane = threadIdx.x & 31, hc = a.n_kv_head * a.chunks;
        int n = 0;
#pragma unroll
        for (int e = 0; e < PA_KEPT; e++) units[e] = lane + 32 * e < a.n_seq ? units_of(lane + 32 * e) * hc : 0;
#pragma unroll
        for (int e = 0; e < PA_KEPT; e++) n += units[e];
        for (int s = lane + 32 * PA_KEPT; s < a.n_seq; s += 32) n += units_of(s) * hc;
        total = __reduce_add_sync(0xffffffffu, n);
        quota = paged_quota(total, ctas, FIXED + PA_WARPS);
    }
    // This CTA's run [*begin, *end) and the sequence that it begins in, whose first unit is *seq_start; false where it has none.
    // Called by whole warps.
    CFI_DEV bool find(const PaArgs& a, int* begin, int* end, int* seq, int* seq_start) {
        const int lane = threadIdx.x & 31, hc = a.n_kv_head * a.chunks;
        read(a, gridDim.x);
        if ((int)blockIdx.x >= paged_runs(total, quota)) return false;
        const int at = blockIdx.x * quota;
        *begin = at;
        *end = paged_run_end(at, quota, total);
        auto among = [&](int base, int n) {  // is it one of the 32 sequences from `base` on, this lane's with n units?
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, *seq_start + incl > at);
            const int l = hit ? __ffs(hit) - 1 : 31;
            *seq = base + l;
            *seq_start += __shfl_sync(0xffffffffu, hit ? incl - n : incl, l);
            return hit != 0;
        };
        bool found = false;
#pragma unroll
        for (int e = 0; e < PA_KEPT; e++)
            if (!found) found = among(32 * e, units[e]);
        for (int base = 32 * PA_KEPT; !found && base < a.n_seq; base += 32)
            found = among(base, base + lane < a.n_seq ? units_of(base + lane) * hc : 0);
        return true;
    }
};

// A pair that this CTA has a part of, and what it takes to join all of them.
struct PaShared {
    int id = -1, seq, head0, nh, b0, n;  // place of its counter; CTAs b0 .. b0 + n - 1 have its tiles
};

// Joins the results of a pair's CTAs in their order.  A thread takes four dims of a head; a round's loads are
// in flight together.
template <class S, int D, int THREADS> CFI_DEV void join_parts(const PaArgs& a, const PaShared& p) {
    constexpr int ROUND = 16;
    const float* parts = a.parts + 2LL * p.b0 * S::PART;
    for (int i = threadIdx.x; i < p.nh * (D / 4); i += THREADS) {
        const int h = i / (D / 4), d = i % (D / 4) * 4;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int x0 = 0; x0 < p.n; x0 += ROUND) {
            float4 v[ROUND];
            float2 ml[ROUND];
#pragma unroll
            for (int e = 0; e < ROUND; e++) {
                const int x = x0 + e;
                // the first CTA's result is in its second place: it leaves the pair unfinished
                const float* q = parts + (2LL * x + (x == 0 ? 1 : 0)) * S::PART;
                ml[e] = x < p.n ? __ldcg(reinterpret_cast<const float2*>(q + PA_HEADS * D) + h) : make_float2(-INFINITY, 0.0f);
                v[e] = x < p.n ? __ldcg(reinterpret_cast<const float4*>(q + h * D + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            }
            float mm = m;
#pragma unroll
            for (int e = 0; e < ROUND; e++) mm = fmaxf(mm, ml[e].x);
            const float keep = m == -INFINITY ? 0.0f : ex2(m - mm);
            l *= keep;
            o = make_float4(o.x * keep, o.y * keep, o.z * keep, o.w * keep);
            m = mm;
#pragma unroll
            for (int e = 0; e < ROUND; e++) {
                const float f = ml[e].x == -INFINITY ? 0.0f : ex2(ml[e].x - mm);
                l = fmaf(f, ml[e].y, l);
                add_to(o, f, v[e]);
            }
        }
        write_out(a, p.seq, p.head0 + h, D, d, o, l);
    }
}

// Behind a CTA's run: the results that are parts are joined by the last of their pair's CTAs to come here.
template <class S, int D, int THREADS> CFI_DEV void join_shared(const PaArgs& a, const PaShared (&shared)[2], int (&s_last)[2]) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (shared[0].id < 0 && shared[1].id < 0) return;
    if (lane == 0 && warp < 2) {  // one thread for each
        const PaShared p = warp == 0 ? shared[0] : shared[1];
        bool last = false;
        if (p.id >= 0) {
            // after a barrier: releases the stores of the whole CTA, and acquires those of the others
            unsigned int before;
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(a.counters + p.id) : "memory");
            last = before == (unsigned)(p.n - 1);
            if (last) a.counters[p.id] = 0u;
        }
        s_last[warp] = last;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2; x++)
        if (s_last[x]) join_parts<S, D, THREADS>(a, shared[x]);
}

// The Q4_1 kernel's launch (k_paged_attn_q4.cu), for a checked call.
int cfi_paged_attention_q4_1(PaArgs& a, int head_dim, long long pairs, cudaStream_t stream);
