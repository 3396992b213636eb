// k_paged_attn_q4.cu -- attention of one new token per sequence over a Q4_1 cache (include/cfi_serve.h):
// out = sum_j softmax_j(scale q.K_j) V_j with K_j = d n + m in each block of 32 dims, so that
//   q.K_j = sum_b d_jb (sum_i q_i n_ji) + m_jb (sum_i q_i),  o = sum_j p_j d_jb n_ji + p_j m_jb.
//
// The list of all sequences' tiles is cut into equal runs and partial results are joined as in k_paged_attn.cu, and as there
// an MMA has up to 8 query heads: rows 0-7 of A are f16 values, rows 8-15 what f16 left of them.  A tile is 32 positions here, two tiles
// of the cache: what a tile costs beside its products (maximum, vote, copies) is shared by twice as many.
//
// A position and kv head are 160 bytes with heads of 128, which at the memory's rate leaves a warp some 28 instructions: what has to
// be cheap is making operands of nibbles.  A nibble needs no conversion: the bits 0x000n are the f16 number n 2^-24, and
// 0x00n0 is 16 n 2^-24, exact subnormals that the MMA multiplies like any others.  One AND (with one shift for every second pair)
// makes two operands; the powers of two go into q (divided by 16 where the upper nibbles meet it) and into the result.
//   K: a word of the cache is 8 dims of one position for one lane; dims i and i + 4 of it share a register.
//   V: two positions meet in a register, so half-words of two rows are first put together by one byte permutation.
// Which position is which column of the scores is free, as long as the weights go back to the same: column 2 c + e of the n-th eight
// is position 8 n + 4 e + (c ^ 3 e), so that no two lanes read the same bank of K or of V.
// The minima of K meet the sums of q over each block in one MMA for 8 positions, those of V the weights in one for 16.
#include "paged_attn.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <algorithm>
#include <math.h>
#include <stdlib.h>
#include <string.h>

namespace {

using namespace sm100;

constexpr int P4_TILE = 32;         // positions
constexpr int P4_FIXED = 3;         // what beginning and ending a pair costs, in tiles
constexpr float P4_TOP = 15.0f;     // log2 of the largest weight as it is split: f16 ends at 65504
constexpr float P4_LEAST_V = -23.0f, P4_MOST_V = 16.0f;  // f16 scales are below 2^these
constexpr float P4_N = 16777216.0f;  // 2^24: nibbles are whole numbers times its inverse
using Cut = PaCut<P4_TILE, P4_FIXED>;

template <int D, int W = PA_WARPS> struct P4Shape {
    static constexpr int TILE = Q41<D>::TILE;
    static constexpr int STAGE = 4 * TILE;  // two tiles of K, two of V
    static constexpr int STAGES = D == 64 ? 5 : 3;
    static constexpr int CTAS = W > PA_WARPS ? 1 : 3;  // per SM
    static constexpr int RING = STAGES * STAGE;        // a warp's
    static constexpr int SMEM = W * RING;
    static constexpr int PART = PA_HEADS * (D + 2);    // floats of a partial result: values, then maximum and sum of each head
    static constexpr int MEET_ROW = D + 4, MEET = PA_HEADS * MEET_ROW;  // where the warps meet
    static_assert(SMEM >= W * MEET * 4, "the warps meet in the stages' memory");
};

CFI_DEV void cp16n(uint32_t dst, const void* src, int bytes) {  // the first `bytes` of 16, zeros behind
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
// two floats at once
using f2 = unsigned long long;
CFI_DEV f2 pair2(float x, float y) {
    f2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
CFI_DEV float2 both(f2 a) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
    return r;
}
CFI_DEV f2 add2(f2 a, f2 b) {
    f2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
CFI_DEV f2 mul2(f2 a, f2 b) {
    f2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
CFI_DEV f2 fma2(f2 a, f2 b, f2 c) {
    f2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
CFI_DEV float half_of(uint32_t w, int i) {
    const __half2 h = *reinterpret_cast<const __half2*>(&w);
    return i ? __high2float(h) : __low2float(h);
}
CFI_DEV void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // the sum begins with it
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
CFI_DEV void ldsm_x2_trans(uint32_t a, uint32_t& r0, uint32_t& r1) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(a));
}
// the even and odd nibbles of each half's lower byte as f16 numbers, n 2^-24 and 16 n 2^-24
CFI_DEV uint32_t low_nibbles(uint32_t w) { return w & 0x000f000fu; }
CFI_DEV uint32_t high_nibbles(uint32_t w) { return w & 0x00f000f0u; }
// column 2 c + e of the n-th eight scores
CFI_DEV int position_of(int c, int e, int n) { return 8 * n + 4 * e + (c ^ (3 * e)); }

template <int D, int W>
__global__ void __launch_bounds__(W * 32, (P4Shape<D, W>::CTAS)) paged_attn_q4(const PaArgs a) {
    using S = P4Shape<D, W>;
    using L = Q41<D>;
    constexpr int NB = D / 32, NT = D / 8, KK = D / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_last[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int page_size = 1 << a.page_shift, hc = a.n_kv_head * a.chunks;
    pdl_launch_dependents();
    pdl_wait();

    Cut cut(a);
    int begin = 0, end = 1, at = 0, seq = 0, seq_start = 0, pair = 0;  // seq_start: the sequence's first unit
    if (a.whole) {
        seq = blockIdx.x / hc;
        pair = blockIdx.x - seq * hc;
    } else if (!cut.find(a, &begin, &end, &seq, &seq_start)) {
        return;
    }
    at = begin;

    const uint32_t ring = smem_u32(smem) + warp * S::RING;
    const int row_k = position_of(g >> 1, g & 1, 0);  // this lane's row of K among eight
    PaShared shared[2];  // of the pairs that it goes on with, and leaves unfinished
    while (at < end) {
        // ---- one (sequence, kv head, chunk): its tiles [t0, t1) of n_tiles ----
        const int len = cut.length(seq), n_tiles = Cut::tiles_of(len);
        int t0 = 0, t1 = n_tiles;
        if (!a.whole) {
            const int units = P4_FIXED + n_tiles;
            pair = (at - seq_start) / units;
            const int first = seq_start + pair * units + P4_FIXED;
            t0 = max(0, at - first);
            t1 = min(n_tiles, end - first);
            at = first + n_tiles;
            if (t1 <= 0) break;  // the run ends before the pair's first tile
        } else {
            at = end;
        }
        const int kvh = pair / a.chunks, h0 = (pair - kvh * a.chunks) * PA_HEADS, nh = min(PA_HEADS, a.group - h0);
        const int head0 = kvh * a.group + h0;

        // page ids of this warp's next 32 tiles, one a lane, of both halves
        const int32_t* trow = a.table + (long long)seq * a.max_pages;
        const int mine = t1 - t0 > warp ? (t1 - t0 - warp + W - 1) / W : 0;  // tiles of this warp
        auto load_id = [&](int i, int half) {
            const int t = t0 + warp + (i + lane) * W, p = t * P4_TILE + half * Q41_TILE;
            return t < t1 && p < len ? min(max(trow[p >> a.page_shift], 0), a.n_pages - 1) : 0;
        };
        int id0 = load_id(0, 0), id1 = load_id(0, 1);

        // the queries: loaded here, converted when the first tiles are on their way.  Dims 32 b + 8 c .. + 7
        float qv[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int e = 0; e < 8; e++) qv[b][e] = 0.0f;
            if (g < nh) {
                const long long o = seq * a.q_stride + (long long)(head0 + g) * D + 32 * b + 8 * c;
                if (a.q_f16) {
                    const uint4 w = *reinterpret_cast<const uint4*>(a.q + o * 2);
                    qv[b][0] = __uint_as_float(w.x), qv[b][1] = __uint_as_float(w.y), qv[b][2] = __uint_as_float(w.z), qv[b][3] = __uint_as_float(w.w);
                } else {
                    const float4 x = *reinterpret_cast<const float4*>(a.q + o * 4), y = *reinterpret_cast<const float4*>(a.q + o * 4 + 16);
                    qv[b][0] = x.x, qv[b][1] = x.y, qv[b][2] = x.z, qv[b][3] = x.w;
                    qv[b][4] = y.x, qv[b][5] = y.y, qv[b][6] = y.z, qv[b][7] = y.w;
                }
            }
        }

        auto fetch = [&](int i) {  // tile i of this warp into its stage
            if (i < mine) {
                const int p0 = (t0 + warp + i * W) * P4_TILE, left = len - p0;
                const int page0 = __shfl_sync(0xffffffffu, id0, i & 31), page1 = __shfl_sync(0xffffffffu, id1, i & 31);
                const uint32_t st = ring + (i % S::STAGES) * S::STAGE;
                auto tile_at = [&](int page, int p) {
                    return ((long long)page * a.n_kv_head + kvh) * paged_region_bytes<D, CACHE_Q4_1>(page_size) + L::tile_at(p & (page_size - 1));
                };
                const long long src0 = tile_at(page0, p0), src1 = tile_at(page1, p0 + Q41_TILE);
                const int two = left > Q41_TILE ? 16 : 0;  // is there a second half?
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    const uint8_t* pool = kv ? a.v : a.k;
                    const uint32_t dst = st + kv * 2 * S::TILE;
#pragma unroll
                    for (int e = 0; e < L::NIBBLES / 512; e++) {
                        const int o = (e * 32 + lane) * 16;
                        cp16n(dst + o, pool + src0 + o, 16);
                        cp16n(dst + S::TILE + o, pool + src1 + o, two);
                    }
                }
                // scales and minima, a chunk a lane; rows past the length get zeros, so that what a page holds there never matters
                constexpr int CH = Q41_TILE * L::PARAM_ROW / 16, ROWS = Q41_TILE / CH;  // chunks of a tile, rows of a chunk
#pragma unroll
                for (int x = 0; x < 4 * CH / 32; x++) {
                    const int n = (x * 32 + lane) / CH, ch = lane % CH, half = n & 1, kv = n >> 1;  // n: tiles as they lie in the stage
                    const int bytes = min(max((left - half * Q41_TILE - ch * ROWS) * L::PARAM_ROW, 0), 16);
                    cp16n(st + n * S::TILE + L::NIBBLES + ch * 16, (kv ? a.v : a.k) + (half ? src1 : src0) + L::NIBBLES + ch * 16, bytes);
                }
            }
            cp_async_commit();
        };

        // V's scales have been below 2^top_v; o has 2^-top_v in it, and 2^-24 (odd dims 2^-20)
        float o[NT][4], mins[4], m = -INFINITY, top_v = P4_LEAST_V, per_top = ex2(-P4_LEAST_V);
        f2 l = 0;
        __half2 limit_v = __float2half2_rn(ex2(top_v));
#pragma unroll
        for (int e = 0; e < 4; e++) mins[e] = 0.0f;
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[j][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < S::STAGES - 1; i++) fetch(i);
        if (a.q_f16) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 3; e >= 0; e--) {
                    const uint32_t raw = __float_as_uint(qv[b][e]);
                    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&raw));
                    qv[b][2 * e] = f.x;
                    qv[b][2 * e + 1] = f.y;
                }
        }
        float largest = 0.0f;  // a NaN is passed over
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                qv[b][e] *= a.scale_log2;
                largest = fmaxf(largest, fabsf(qv[b][e]));
            }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // 2^(its exponent - 14) and the other way round, both normal: below 2^-111 the largest stays below 2^14
        const uint32_t exponent = max(__float_as_uint(largest) >> 23, 15u);
        const float unit = __uint_as_float((exponent - 14) << 23), per_unit = __uint_as_float((268 - exponent) << 23);
        uint32_t qf[KK][4], qs[2];  // in log2 units over `unit`, split; the sums of the blocks, over 2^6
        float sums[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            sums[b] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                qv[b][e] *= per_unit;
                sums[b] += qv[b][e];
            }
            sums[b] += __shfl_xor_sync(0xffffffffu, sums[b], 1);
            sums[b] += __shfl_xor_sync(0xffffffffu, sums[b], 2);
#pragma unroll
            for (int k = 0; k < 2; k++) {
                split(qv[b][2 * k], qv[b][2 * k + 4], &qf[2 * b + k][0], &qf[2 * b + k][1]);
                split(qv[b][2 * k + 1] * 0.0625f, qv[b][2 * k + 5] * 0.0625f, &qf[2 * b + k][2], &qf[2 * b + k][3]);
            }
        }
        {
            // a row of scales and minima is 2 NB f16 numbers: the lane's pair of those are minima of blocks x and x + 1
            const int x = 2 * c - NB;
            const float s0 = x == 0 ? sums[0] : NB == 4 && x == 2 ? sums[NB - 2] : 0.0f, s1 = x == 0 ? sums[1] : NB == 4 && x == 2 ? sums[NB - 1] : 0.0f;
            split(s0 * 0.015625f, s1 * 0.015625f, &qs[0], &qs[1]);
        }
        for (int i = 0; i < mine; i++) {
            if ((i + S::STAGES - 1) % 32 == 0) {
                id0 = load_id(i + S::STAGES - 1, 0);
                id1 = load_id(i + S::STAGES - 1, 1);
            }
            fetch(i + S::STAGES - 1);
            cp_async_wait<S::STAGES - 1>();
            __syncwarp();
            const uint32_t sk = ring + (i % S::STAGES) * S::STAGE, sv = sk + 2 * S::TILE;
            // ---- scores, over 2^24 `unit`, of head g: columns 2c, 2c+1 of four eights ----
            f2 s[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const uint32_t tile = sk + (n >> 1) * S::TILE;
                const int row = row_k + 8 * (n & 1);
                {
                    float acc[4];
                    const uint32_t sums2[4] = {qs[0], qs[1], 0, 0};
                    mma_first(acc, sums2, lds32(tile + L::NIBBLES + row * L::PARAM_ROW + 4 * (c & (NB - 1))), 0);
                    s[n] = mul2(add2(pair2(acc[0], acc[1]), pair2(acc[2], acc[3])), pair2(64.0f / P4_N, 64.0f / P4_N));
                }
                uint32_t w[NB], d[2][NB / 2];  // eight dims of each block of the lane's row; scales of columns 2c and 2c+1
                if (D == 128) {
                    const uint4 x = lds128(tile + row * L::ROW + c * 16);
                    w[0] = x.x, w[1] = x.y, w[NB - 2] = x.z, w[NB - 1] = x.w;
                } else {
                    const uint2 x = lds64(tile + row * L::ROW + c * 8);
                    w[0] = x.x, w[1] = x.y;
                }
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const uint32_t p = tile + L::NIBBLES + position_of(c, e, n & 1) * L::PARAM_ROW;
                    if (D == 128) {
                        const uint2 x = lds64(p);
                        d[e][0] = x.x, d[e][NB / 2 - 1] = x.y;
                    } else {
                        d[e][0] = lds32(p);
                    }
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    float acc[4];
                    mma_first(acc, qf[2 * b], low_nibbles(w[b]), high_nibbles(w[b]));
                    mma_f16f32(acc, qf[2 * b + 1], low_nibbles(w[b] >> 8), high_nibbles(w[b] >> 8));
                    s[n] = fma2(add2(pair2(acc[0], acc[1]), pair2(acc[2], acc[3])),
                                pair2(half_of(d[0][b >> 1], b & 1), half_of(d[1][b >> 1], b & 1)), s[n]);
                }
            }
            const int left = len - (t0 + warp + i * W) * P4_TILE;
            if (left < P4_TILE) {
#pragma unroll
                for (int n = 0; n < 4; n++) {
                    float2 x = both(s[n]);
                    if (16 * (n >> 1) + position_of(c, 0, n & 1) >= left) x.x = -INFINITY;
                    if (16 * (n >> 1) + position_of(c, 1, n & 1) >= left) x.y = -INFINITY;
                    s[n] = pair2(x.x, x.y);
                }
            }
            float mx = -INFINITY;
#pragma unroll
            for (int n = 0; n < 4; n++) mx = fmaxf(mx, fmaxf(both(s[n]).x, both(s[n]).y));
            if (__any_sync(0xffffffffu, mx > m)) {
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
                const float mn = fmaxf(m, mx), alpha = m == -INFINITY ? 0.0f : ex2((m - mn) * P4_N * unit);
                const f2 alpha2 = pair2(alpha, alpha);
                l = mul2(l, alpha2);
#pragma unroll
                for (int e = 0; e < 4; e++) mins[e] *= alpha;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[j][e] *= alpha;
                m = mn;
            }
            const float sub = m == -INFINITY ? 0.0f : -m * P4_N, rise = P4_TOP;  // added last: a large score would swallow it
            f2 p[4];
#pragma unroll
            for (int n = 0; n < 4; n++) {
                const float2 x = both(fma2(fma2(s[n], pair2(P4_N, P4_N), pair2(sub, sub)), pair2(unit, unit), pair2(rise, rise)));
                p[n] = pair2(ex2(x.x), ex2(x.y));
                l = add2(l, p[n]);
            }
            // ---- weighted values ----
            {
                // a lane looks at some of the tile's scales
                __half2 d = __float2half2_rn(0.0f);
#pragma unroll
                for (int x = 0; x < NB / 2; x++) {
                    const uint32_t row = sv + (lane >> 4) * S::TILE + L::NIBBLES + (lane & 15) * L::PARAM_ROW;
                    d = __hmax2_nan(d, abs_h2(lds32(row + 4 * x)));
                }
                if (__any_sync(0xffffffffu, !__hblt2(d, limit_v))) {
                    // the exponent of the largest, cut where that is an infinity or a NaN
                    const uint32_t ex = __float_as_uint(fmaxf(__low2float(d), __high2float(d))) >> 23;
                    const float grown = fmaxf(top_v, fminf((float)__reduce_max_sync(0xffffffffu, ex) - 126.0f, P4_MOST_V));
                    const float f = ex2(top_v - grown);
#pragma unroll
                    for (int j = 0; j < NT; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[j][e] *= f;
                    per_top = ex2(-grown);
                    top_v = grown;
                    limit_v = __float2half2_rn(ex2(grown));
                }
            }
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const uint32_t tile = sv + t * S::TILE;
                {  // minima: column x of a row's scales and minima, of which those from NB on count
                    uint32_t pf[4], b0, b1;
#pragma unroll
                    for (int n = 0; n < 2; n++) split(both(p[2 * t + n]).x, both(p[2 * t + n]).y, &pf[2 * n], &pf[2 * n + 1]);
                    if (D == 128) {
                        ldsm_x2_trans(tile + L::NIBBLES + position_of(lane >> 1 & 3, lane & 1, lane >> 3 & 1) * L::PARAM_ROW, b0, b1);
                    } else {  // rows of four numbers: column g & 3 of the lane's four positions
                        uint32_t x[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = lds16(tile + L::NIBBLES + position_of(c, e & 1, e >> 1) * L::PARAM_ROW + 2 * (g & 3));
                        b0 = x[0] | x[1] << 16;
                        b1 = x[2] | x[3] << 16;
                    }
                    mma_f16f32(mins, pf, b0, b1);
                }
                uint32_t w[2][2][NB / 2], d[2][2][NB / 2];  // of column e of eight n: the lane's dims; scales
#pragma unroll
                for (int n = 0; n < 2; n++)
#pragma unroll
                    for (int e = 0; e < 2; e++) {
                        const int row = position_of(c, e, n);
                        const uint32_t q = tile + row * L::ROW + L::v_group(row, g) * (D / 16), r = tile + L::NIBBLES + row * L::PARAM_ROW;
                        if (D == 128) {
                            const uint2 x = lds64(q), y = lds64(r);
                            w[n][e][0] = x.x, w[n][e][NB / 2 - 1] = x.y;
                            d[n][e][0] = y.x, d[n][e][NB / 2 - 1] = y.y;
                        } else {
                            w[n][e][0] = lds32(q);
                            d[n][e][0] = lds32(r);
                        }
                    }
                f2 pv[2];
#pragma unroll
                for (int n = 0; n < 2; n++) pv[n] = mul2(p[2 * t + n], pair2(per_top, per_top));
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t pf[4], bw[2][4];
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const float2 x = both(mul2(pv[n], pair2(half_of(d[n][0][b >> 1], b & 1), half_of(d[n][1][b >> 1], b & 1))));
                        split(x.x, x.y, &pf[2 * n], &pf[2 * n + 1]);
                        // dims 32 b + 4 g .. + 3 of two positions: column g of MMA e is dim 32 b + 4 g + e
                        const uint32_t z = __byte_perm(w[n][0][b >> 1], w[n][1][b >> 1], b & 1 ? 0x7632 : 0x5410);
                        bw[n][0] = low_nibbles(z);
                        bw[n][1] = high_nibbles(z);
                        bw[n][2] = low_nibbles(z >> 8);
                        bw[n][3] = high_nibbles(z >> 8);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) mma_f16f32(o[4 * b + e], pf, bw[0][e], bw[1][e]);
                }
            }
            __syncwarp();  // the stage is free
        }
        // ---- the warps meet: [warp][head]: D values, maximum, sum ----
        cp_async_wait<0>();
        const float back = ex2(top_v) * P4_N;  // each warp has had scales of its own
        float sum = both(l).x + both(l).y, low[NB];
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int b = 0; b < NB; b++)  // columns 2 c and 2 c + 1 of the minima are this lane's
            low[b] = __shfl_sync(0xffffffffu, mins[b & 1] + mins[2 + (b & 1)], (lane & ~3) + (NB + b) / 2);
        __syncthreads();  // every warp is done with its stages
        float* meet = reinterpret_cast<float*>(smem);
        float* mine_o = meet + warp * S::MEET + g * S::MEET_ROW;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                float f[4];
#pragma unroll
                for (int x = 0; x < 4; x++)
                    f[x] = fmaf(o[4 * b + x][e] + o[4 * b + x][e + 2], x & 1 ? back / 16.0f : back, low[b]);
                *reinterpret_cast<float4*>(mine_o + 32 * b + 8 * c + 4 * e) = make_float4(f[0], f[1], f[2], f[3]);
            }
        if (c == 0) *reinterpret_cast<float2*>(mine_o + D) = make_float2(m * P4_N * unit, sum);
        __syncthreads();
        const bool done = t0 == 0 && t1 == n_tiles;
        if (!done) {
            const int start = at - n_tiles, b0 = start / cut.quota, n = (at - 1) / cut.quota - b0 + 1;
            const PaShared p = {seq * hc + pair, seq, head0, nh, b0, n};
            if (t0 == 0) shared[1] = p; else shared[0] = p;
        }
        float* part = a.parts + (2LL * blockIdx.x + (t0 == 0 ? 1 : 0)) * S::PART;
        for (int i = tid; i < nh * (D / 4); i += W * 32) {
            const int h = i / (D / 4), d = i % (D / 4) * 4;
            const float* p = meet + h * S::MEET_ROW;
            float mm = -INFINITY, ll = 0.0f;
            float4 oo = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < W; w++) mm = fmaxf(mm, p[w * S::MEET + D]);
#pragma unroll
            for (int w = 0; w < W; w++) {
                const float2 ml = *reinterpret_cast<const float2*>(p + w * S::MEET + D);
                const float f = ml.x == -INFINITY ? 0.0f : ex2(ml.x - mm);
                ll = fmaf(f, ml.y, ll);
                add_to(oo, f, *reinterpret_cast<const float4*>(p + w * S::MEET + d));
            }
            if (done) {
                write_out(a, seq, head0 + h, D, d, oo, ll);
            } else {
                __stcg(reinterpret_cast<float4*>(part + h * D + d), oo);
                if (d == 0) __stcg(reinterpret_cast<float2*>(part + PA_HEADS * D + 2 * h), make_float2(mm, ll));
            }
        }
        __syncthreads();  // the meeting place is free for the next pair's stages
        if (pair == hc - 1) {
            seq_start = at;
            seq++;
        }
    }
    if (!a.whole) join_shared<S, D, W * 32>(a, shared, s_last);
}

template <int D, int W> int launch(PaArgs& a, long long pairs, long long most_units, cudaStream_t stream) {
    using S = P4Shape<D, W>;
    static CfiPerDeviceOnce once;
    cfi_once_per_device(once, [] { cudaFuncSetAttribute(paged_attn_q4<D, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
    long long grid = pairs;
    if (!a.whole) {
        // no CTA has fewer units than this
        const long long ctas = (long long)cfi_sm_count() * S::CTAS;
        grid = std::min(ctas, most_units / (P4_FIXED + PA_WARPS) + 1);
        int err = 0;
        a.parts = static_cast<float*>(cfi_stream_buffer(CFI_BUF_PAGED_PARTS, (size_t)ctas * 2 * S::PART * 4, stream, &err));
        if (!a.parts) return err;
        a.counters = static_cast<unsigned int*>(cfi_stream_buffer(CFI_BUF_COUNTERS, (size_t)pairs * 4, stream, &err));
        if (!a.counters) return err;
    }
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)grid, 1, 1);
    lc.blockDim = dim3(W * 32, 1, 1);
    lc.dynamicSmemBytes = S::SMEM;
    lc.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    return (int)cudaLaunchKernelEx(&lc, paged_attn_q4<D, W>, (const PaArgs)a);
}

}  // namespace

int cfi_paged_attention_q4_1(PaArgs& a, int head_dim, long long pairs, cudaStream_t stream) {
    const long long positions = (long long)a.max_pages << a.page_shift;
    const long long most_units = pairs * (P4_FIXED + (positions + P4_TILE - 1) / P4_TILE);
    const int sms = cfi_sm_count();
    const int w = pairs <= sms ? (positions <= (2 * pairs > sms ? 1536 : 768) ? 8 : 0) : positions <= 768 ? 4 : 0;
    a.whole = w > 0;
    if (w == 8) return head_dim == 64 ? launch<64, 8>(a, pairs, most_units, stream) : launch<128, 8>(a, pairs, most_units, stream);
    return head_dim == 64 ? launch<64, PA_WARPS>(a, pairs, most_units, stream) : launch<128, PA_WARPS>(a, pairs, most_units, stream);
}
