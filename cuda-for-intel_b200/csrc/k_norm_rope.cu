// k_norm_rope.cu -- bias, norm of each head and rotation of a product's rows of q and k, bias of v, in one pass, the
// rows of k and v into the slots of a paged cache (include/cfi_serve.h).
//
// Bound by HBM: every row is read once and written once.  D / 8 lanes take a head: lane l the four dims 4 l .. and their four
// partners n_rot / 2 behind, so that a rotation needs no other lane (the lanes behind n_rot / 8 take eight dims that are not turned).
//
// Angles.  A pair's rate in turns, freq_scale freq_base^(-2 i / n_rot) / 2 pi, is a fraction of 2^64; times the position it wraps by
// whole turns, exactly, and the upper 32 bits are the angle: off by 2^-32 of a turn and, as f32, by 2^-25 of half a turn, 9.5e-8 rad, beside
// what the rate is off by times the position.  (A position of 100000 times a rate in f32 would be off by 4e-3 rad.)
#include "paged_row.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <algorithm>
#include <math.h>
#include <stdlib.h>
#include <string.h>

namespace {

constexpr int NR_RATES = 64;
// Few rows: a head to a group of lanes.  Many: a run of up to NR_HEADS heads of one token to a group, which reads its angles once; from
// nr_many() heads a group of all SMs' CTAs on.  Measured (us), a head to a group against runs, at 5, 7, 9 and 12 such heads:
//   12/2 heads of 128, f16 6.0 to 6.1, 7.1 to 7.0, 9.1 to 7.5, 11.7 to 7.6; Q8_0 6.3 to 4.6, 8.2 to 6.0, 9.7 to 6.0, 12.5 to 8.8; Q4_1 7.7 to
//      5.5, 9.9 to 5.6, 12.1 to 8.7, 15.4 to 9.4;
//   32/8 of 128, f16 6.0 to 5.4, 7.8 to 6.3, 9.4 to 7.7, 11.9 to 8.4; Q8_0 6.3 to 7.4, 8.1 to 8.4, 9.8 to 8.6, 12.6 to 9.0; Q4_1 6.8 to 8.1, 9.0
//      to 8.7, 11.3 to 9.1, 14.7 to 9.3;
//   14/2 of 64, f16 5.0 to 7.0, 6.3 to 7.9, 7.6 to 5.7, 9.4 to 8.5; Q8_0 6.0 to 6.8, 7.9 to 7.0, 9.0 to 7.0, 11.7 to 11.2; Q4_1 7.3 to 6.4, 9.6 to
//      6.5, 11.9 to 6.7, 15.0 to 11.7;
//   16/16 of 64, f16 4.5 to 5.4, 5.4 to 6.2, 6.5 to 7.6, 8.0 to 8.4; Q8_0 5.2 to 8.5, 6.5 to 9.1, 7.8 to 9.4, 9.8 to 9.7; Q4_1 6.4 to 8.7, 8.2 to
//      9.1, 10.1 to 9.4, 12.9 to 9.5.
// Where they cross is a matter of how full the last wave of CTAs is: no limit is right for all, and these cost 3.2 us at most.
constexpr int nr_many(int head_dim) { return head_dim == 128 ? 7 : 8; }
// Measured, 8191 rows of 32/8 heads of 128 normed, turned and put into f16 pages, 61 us (5.0 TB/s): runs of 4, 8, 12, 16 heads 66, 63, 68, 73
// (before the last step); 1, 2, 4 heads' loads together 87, 65, 73; blocks of 256, 128, 64, 32 threads 65, 64, 63, 63; 64 and 72 registers
// (16 and 14 blocks of 64 an SM) 60.7 and 62.2, but 1000 rows 10.0 and 9.4.  Norm weights read for each head and angles
// turned into sines after all are formed leave the 64 registers nearly unspilled: 63 to 61 us, 631 rows of 12/2 6.1 to 5.3.  The loads' latency
// and 190 instructions for two heads of a warp share the time.
constexpr int NR_HEADS = 8, NR_AT_ONCE = 2;
constexpr int nr_threads(bool many) { return many ? 64 : 256; }
constexpr int nr_ctas(int ty, bool many) { return (ty == CACHE_F16 ? 1024 : 512) / nr_threads(many); }

struct NrArgs {
    CfiNormRope r;
    uint8_t *k_pool, *v_pool;
    long long n_slots;
    int page_shift;
    uint32_t runs;           // of a token's heads: those of q begin at 0, of k and v at begin[1] and begin[2]
    int begin[3], heads[3];  // heads of a run
    int most;                // the largest of them
    union {
        unsigned long long turn[NR_RATES];  // of 2^64
        float2 rate[NR_RATES];              // in turns, the sum of two, where freq_factors divide them
    };
};

CFI_DEV float4 f4(uint4 w) { return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)); }
CFI_DEV uint4 ldg128_stream(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
CFI_DEV uint2 ldg64_stream(const void* p) {
    uint2 v;
    asm volatile("ld.global.L1::no_allocate.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
template <bool IN_F16> CFI_DEV float4 load4(const void* rows, long long at) {
    if (!IN_F16) return f4(ldg128_stream(static_cast<const float*>(rows) + at));
    const uint2 w = ldg64_stream(static_cast<const __half*>(rows) + at);
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
CFI_DEV uint2 halves(float4 x) {
    const __half2 a = __floats2half2_rn(x.x, x.y), b = __floats2half2_rn(x.z, x.w);
    return make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
CFI_DEV void store4(void* rows, int f16, long long at, float4 x) {
    if (f16)
        *reinterpret_cast<uint2*>(static_cast<__half*>(rows) + at) = halves(x);
    else
        *reinterpret_cast<float4*>(static_cast<float*>(rows) + at) = x;
}
CFI_DEV float4 add4(float4 a, float4 b) { return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w); }
CFI_DEV float4 mul4(float4 a, float s, float4 b) { return make_float4(a.x * s * b.x, a.y * s * b.y, a.z * s * b.z, a.w * s * b.w); }
CFI_DEV float dot4(float4 a) { return fmaf(a.x, a.x, fmaf(a.y, a.y, fmaf(a.z, a.z, a.w * a.w))); }
// (x, y) turned, the products rounded as they are
CFI_DEV void turn1(float& x, float& y, float c, float s) {
    const float t = fmaf(x, c, -(y * s));
    y = fmaf(x, s, y * c);
    x = t;
}

// A rate in turns over f, as a fraction of 2^64: the quotient digit by digit, 24 bits each.  The first remainder, up to 2^-23 of the rate, is
// rounded to 24 bits, and so is its sum with the rate's second part: the quotient is off by less than 2^-45 of itself.  (The remainders kept
// whole, with three parts of a rate, are off by 2^-64 of a turn, but the kernel without factors took 1 to 10 % longer beside them.)
CFI_DEV unsigned long long divided(float2 rate, float f) {
    const float inv = 1.0f / f, q0 = rate.x * inv;
    const float r0 = fmaf(-q0, f, rate.x) + rate.y, q1 = r0 * inv, q2 = fmaf(-q1, f, r0) * inv;
    const float two64 = 18446744073709551616.0f;
    return (unsigned long long)(__float2ll_rn((q0 - rintf(q0)) * two64) + __float2ll_rn(q1 * two64) + __float2ll_rn(q2 * two64));
}

// TY: of the cache; F16 also where there is none.
template <int D, bool IN_F16, int TY, bool MANY>
__global__ void __launch_bounds__(nr_threads(MANY), nr_ctas(TY, MANY)) norm_rope(const __grid_constant__ NrArgs a) {
    constexpr int G = D / 8, THREADS = nr_threads(MANY), AT_ONCE = MANY ? NR_AT_ONCE : 1;  // G: lanes of a head
    __shared__ float4 s_row[TY == CACHE_F16 ? 1 : THREADS / G][2 * G];  // a row of k or v, where the cache wants eight dims in a lane
    const CfiNormRope& r = a.r;
    const int lane = threadIdx.x % G, group = threadIdx.x / G;
    const int eighth = r.n_rot / 8;  // lanes that turn
    const int d0 = lane < eighth ? 4 * lane : 8 * lane, d1 = lane < eighth ? 4 * (lane + eighth) : 8 * lane + 4;
    // this group's token and run of heads, of q (kind 0), k or v
    const uint32_t id = blockIdx.x * (THREADS / G) + group;
    const bool live = id < (uint32_t)r.n_tokens * a.runs;
    const int t = live ? (int)(id / a.runs) : r.n_tokens - 1, run = live ? (int)(id % a.runs) : 0;
    const int kind = run < a.begin[1] ? 0 : run < a.begin[2] ? 1 : 2;
    const int h0 = (run - a.begin[kind]) * a.heads[kind], n = live ? min(a.heads[kind], (kind ? r.n_kv_head : r.n_head) - h0) : 0;
    const bool turns = lane < eighth && kind != 2;
    const long long from = (long long)t * (kind == 0 ? r.q_stride : kind == 1 ? r.k_stride : r.v_stride) + h0 * D;
    const uint8_t* in = static_cast<const uint8_t*>(kind == 0 ? r.q : kind == 1 ? r.k : r.v) + from * (IN_F16 ? 2 : 4);
    const float* bias = kind == 0 ? r.q_bias : kind == 1 ? r.k_bias : r.v_bias;
    if (bias) bias += h0 * D;
    const float* norm = kind == 0 ? r.q_norm : kind == 1 ? r.k_norm : nullptr;
    const int out_f16 = kind == 0 ? r.q_out_type : r.kv_out_type;
    uint8_t* out = static_cast<uint8_t*>(kind == 0 ? r.q_out : kind == 1 ? r.k_out : r.v_out);
    if (out) out += ((long long)t * (kind == 0 ? r.q_out_stride : kind == 1 ? r.k_out_stride : r.v_out_stride) + h0 * D) * (out_f16 ? 2 : 4);
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    const long long slot = a.k_pool && kind != 0 ? r.slots[t] : -1;
    const bool put = live && slot >= 0 && slot < a.n_slots;
    const int off = (int)(slot & ((1 << a.page_shift) - 1));
    const long long region_bytes = paged_region_bytes<D, TY>(1 << a.page_shift);
    uint8_t* region = (kind == 2 ? a.v_pool : a.k_pool) + ((slot >> a.page_shift) * r.n_kv_head + h0) * region_bytes;
    float cs[4], sn[4];
    for (int i0 = 0; i0 < a.most; i0 += AT_ONCE) {
        // all loads first
        float4 x[AT_ONCE][2];
#pragma unroll
        for (int e = 0; e < AT_ONCE; e++) {
            x[e][0] = x[e][1] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i0 + e < n) {
                x[e][0] = load4<IN_F16>(in, (i0 + e) * D + d0);
                x[e][1] = load4<IN_F16>(in, (i0 + e) * D + d1);
            }
        }
        if (i0 == 0 && turns) {
            const int pos = r.pos[t];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const unsigned long long f = r.freq_factors ? divided(a.rate[4 * lane + e], r.freq_factors[4 * lane + e]) : a.turn[4 * lane + e];
                cs[e] = (float)(int)((f * (unsigned long long)(long long)pos) >> 32) * 0x1p-31f;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) sincospif(cs[e], &sn[e], &cs[e]);
        }
#pragma unroll
        for (int e = 0; e < AT_ONCE; e++) {
            const int h = i0 + e;
            const bool on = h < n;
            float4 x0 = x[e][0], x1 = x[e][1];
            if (bias && on) {
                x0 = add4(x0, *reinterpret_cast<const float4*>(bias + h * D + d0));
                x1 = add4(x1, *reinterpret_cast<const float4*>(bias + h * D + d1));
            }
            if (r.q_norm || r.k_norm) {
                float ss = dot4(x0) + dot4(x1);
#pragma unroll
                for (int o = 1; o < G; o <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                if (norm && on) {
                    const float s = rsqrtf(ss / (float)D + r.eps);
                    x0 = mul4(x0, s, *reinterpret_cast<const float4*>(norm + d0));
                    x1 = mul4(x1, s, *reinterpret_cast<const float4*>(norm + d1));
                }
            }
            if (turns) {
                turn1(x0.x, x1.x, cs[0], sn[0]);
                turn1(x0.y, x1.y, cs[1], sn[1]);
                turn1(x0.z, x1.z, cs[2], sn[2]);
                turn1(x0.w, x1.w, cs[3], sn[3]);
            }
            if (out && on) {
                store4(out, out_f16, h * D + d0, x0);
                store4(out, out_f16, h * D + d1, x1);
            }
            if (!a.k_pool) continue;
            uint8_t* to = region + h * region_bytes;
            if (TY == CACHE_F16) {
                if (put && on) {
                    *reinterpret_cast<uint2*>(to + (off * D + d0) * 2) = halves(x0);
                    *reinterpret_cast<uint2*>(to + (off * D + d1) * 2) = halves(x1);
                }
            } else if (__any_sync(0xffffffffu, put && on)) {
                // eight neighbouring dims in a lane
                __syncwarp();
                s_row[group][d0 / 4] = x0;
                s_row[group][d1 / 4] = x1;
                __syncwarp();
                const float4 y0 = s_row[group][2 * lane], y1 = s_row[group][2 * lane + 1];
                const Row8 y = {{y0.x, y0.y, y0.z, y0.w, y1.x, y1.y, y1.z, y1.w}, {}};
                if (TY == CACHE_Q8_0)
                    put_q8_0<D, false>(y, to, a.page_shift, off, lane, put && on);
                else
                    put_q4_1<D, false>(y, to, off, lane, kind == 2, put && on);
            }
        }
    }
}

bool rows_ok(const void* p, long long stride, long long width) { return p && !((uintptr_t)p & 15) && stride % 8 == 0 && stride >= width; }
bool type_ok(int t) { return t == 0 || t == 1; }

template <int D, bool IN_F16, int TY> const void* kernel(bool many) {
    return many ? (const void*)norm_rope<D, IN_F16, TY, true> : (const void*)norm_rope<D, IN_F16, TY, false>;
}
template <int D, bool IN_F16> const void* kernel(int ty, bool many) {
    return ty == CACHE_Q8_0   ? kernel<D, IN_F16, CACHE_Q8_0>(many)
           : ty == CACHE_Q4_1 ? kernel<D, IN_F16, CACHE_Q4_1>(many)
                              : kernel<D, IN_F16, CACHE_F16>(many);
}
const void* kernel_of(int head_dim, int in_type, int ty, bool many) {
    if (head_dim == 64) return in_type ? kernel<64, true>(ty, many) : kernel<64, false>(ty, many);
    return in_type ? kernel<128, true>(ty, many) : kernel<128, false>(ty, many);
}

// The pairs' rates in turns.
void rates(const CfiNormRope* r, NrArgs* a) {
    const long double step = powl((long double)r->freq_base, -2.0L / r->n_rot), two64 = 18446744073709551616.0L;
    long double rate = (long double)r->freq_scale / 6.283185307179586476925287L;
    if (!r->freq_factors && step < 1.0L && rate >= 0.0L && rate < 1.0L) {  // as is usual: whole numbers all the way
        unsigned long long turn = (unsigned long long)(rate * two64);
        const unsigned long long by = (unsigned long long)(step * two64);
        for (int i = 0; i < r->n_rot / 2; i++) {
            a->turn[i] = turn;
            turn = (unsigned long long)(((unsigned __int128)turn * by) >> 64);
        }
        return;
    }
    for (int i = 0; i < r->n_rot / 2; i++, rate *= step) {
        const long double part = (rate - floorl(rate)) * two64;
        if (r->freq_factors)
            a->rate[i] = make_float2((float)rate, (float)(rate - (float)rate));
        else
            a->turn[i] = part < two64 ? (unsigned long long)part : 0;
    }
}

}  // namespace

extern "C" int cfi_norm_rope(const CfiNormRope* r, const CfiPagedCache* c, void* stream) {
    if (!r || (r->head_dim != 64 && r->head_dim != 128) || r->n_tokens < 0 || r->n_head <= 0 || r->n_head > 65535 || r->n_kv_head < 0 ||
        r->n_kv_head > 65535 || !type_ok(r->in_type) || !type_ok(r->q_out_type) || !type_ok(r->kv_out_type) || r->n_rot < 0 ||
        r->n_rot > r->head_dim || r->n_rot % 8 || !(r->eps >= 0.0f) || isinf(r->eps))
        return (int)cudaErrorInvalidValue;
    const long long wq = (long long)r->n_head * r->head_dim, wk = (long long)r->n_kv_head * r->head_dim;
    if (!rows_ok(r->q, r->q_stride, wq) || !rows_ok(r->q_out, r->q_out_stride, wq) || (r->k && !rows_ok(r->k, r->k_stride, wk)) ||
        (r->v && !rows_ok(r->v, r->v_stride, wk)) || (r->k_out && !rows_ok(r->k_out, r->k_out_stride, wk)) ||
        (r->v_out && !rows_ok(r->v_out, r->v_out_stride, wk)) || ((r->k || r->v) && r->n_kv_head == 0) || (r->k && !r->k_out && !c) ||
        (r->v && !r->v_out && !c) || (r->k_out && !r->k) || (r->v_out && !r->v))
        return (int)cudaErrorInvalidValue;
    if ((((uintptr_t)r->q_bias | (uintptr_t)r->k_bias | (uintptr_t)r->v_bias | (uintptr_t)r->q_norm | (uintptr_t)r->k_norm) & 15) ||
        ((uintptr_t)r->freq_factors & 3))
        return (int)cudaErrorInvalidValue;
    if (r->n_rot && (!r->pos || ((uintptr_t)r->pos & 3) || !(r->freq_base > 0.0f) || isinf(r->freq_base) || !isfinite(r->freq_scale)))
        return (int)cudaErrorInvalidValue;
    if (c && (!cfi_paged_ok(c) || !r->k || !r->v || !r->slots || ((uintptr_t)r->slots & 7) || c->head_dim != r->head_dim ||
              c->n_kv_head != r->n_kv_head))
        return (int)cudaErrorInvalidValue;
    if (r->n_tokens == 0) return 0;
    NrArgs a = {};
    a.r = *r;
    if (c) {
        a.k_pool = static_cast<uint8_t*>(c->k);
        a.v_pool = static_cast<uint8_t*>(c->v);
        a.n_slots = (long long)c->n_pages * c->page_size;
        a.page_shift = __builtin_ctz((unsigned)c->page_size);
    }
    if (r->n_rot) {
        rates(r, &a);
    }
    const int heads = r->n_head + (r->k ? r->n_kv_head : 0) + (r->v ? r->n_kv_head : 0), lanes = r->head_dim / 8;
    if ((long long)r->n_tokens * heads > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    const bool many = (long long)r->n_tokens * heads >= nr_many(r->head_dim) * (long long)cfi_sm_count() * (nr_threads(false) / lanes);
    const int groups = nr_threads(many) / lanes;
    const int count[3] = {r->n_head, r->k ? r->n_kv_head : 0, r->v ? r->n_kv_head : 0};
    for (int i = 0; i < 3; i++) {
        a.begin[i] = (int)a.runs;
        const int runs = many ? (count[i] + NR_HEADS - 1) / NR_HEADS : count[i];
        a.heads[i] = runs ? (count[i] + runs - 1) / runs : 0;
        a.runs += runs;
        a.most = std::max(a.most, a.heads[i]);
    }
    const uint32_t ctas = ((uint32_t)r->n_tokens * a.runs + groups - 1) / groups;
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3(ctas, 1, 1);
    lc.blockDim = dim3((unsigned)nr_threads(many), 1, 1);
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    void* args[1] = {&a};
    return (int)cudaLaunchKernelExC(&lc, kernel_of(r->head_dim, r->in_type, c ? c->type : CACHE_F16, many), args);
}
