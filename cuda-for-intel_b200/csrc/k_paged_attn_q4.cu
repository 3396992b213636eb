// k_paged_attn_q4.cu -- attention of one new token per sequence over a Q4_1 cache (include/cfi_serve.h):
// out = sum_j softmax_j(scale q.K_j) V_j with K_j = d n + m in each block of 32 dims, so that
//   q.K_j = sum_b d_jb (sum_i q_i n_ji) + m_jb (sum_i q_i),  o = sum_j p_j d_jb n_ji + p_j m_jb.
//
// The list of all sequences' tiles is cut into equal runs and partial results are joined as in k_paged_attn.cu, and as there
// an MMA has up to 8 query heads: rows 0-7 of A are f16 values, rows 8-15 what f16 left of them.  A tile is 32 positions here, two tiles
// of the cache: what a tile costs beside its products (maximum, vote, copies) is shared by twice as many.
//
// A position and kv head are 160 bytes with heads of 128, which at the memory's rate leaves a warp some 28 instructions: what has to
// be cheap is making operands of nibbles.  A byte 16 h + l with 0x64 above it is the f16 number 1024 + 16 h + l; without its upper
// nibble it is 1024 + l, and one subtraction for two of them takes the 1024 away.  So both go in, where
//   x l + y h = (x - y/16) l + (y/16) (16 h + l),
// and V's sums are taken apart at the end.  (The bits 0x00hl alone are 16 h + l times 2^-24, with no instruction more: but an MMA lines
// its products up by their exponents' fields, cuts them at 24 bits, and subnormal operands lose up to ten of those.)
//   K, five to eight heads: A is q, B is K: a word of the cache is 8 dims of one position for one lane; dims i and i + 4 of it share a
//      register.  Rows 0-7 of the result and rows 8-15 are added.
//   K, up to four heads: whole numbers.  q is four digits of 8 bits, four heads times four digits are the 16 rows of A, and one MMA
//      of bytes takes a block of 32 dims where f16 needs two; its sums begin at the bits of 1.5 2^23, so that they are read as floats.
//   V: two positions meet in a register, so half-words of two rows are first put together by one byte permutation.  A is V with
//      dims as rows, B the weights, which lie as the scores came out; f16 values and what these leave go one after the other, or, with up to
//      four heads, in columns 0-3 and 4-7 of the same MMA.
// Which position is which column of the scores is free, as long as the weights go back to the same: column 2 c + e of the n-th eight
// is position 8 n + 4 e + (c ^ 3 e), so that no two lanes read the same bank of K or of V.
// The minima of K meet the sums of q over each block in one MMA for 8 positions, those of V the weights in one for 16.
//
// Bound by instruction issue and by chains that two warps a scheduler do not cover.  An MMA of 16 x 8 x 16 holds its part of the SM for 8 cycles in
// which nothing else is issued (measured: 8 + N cycles for one beside N other instructions), and a tile of 32 positions is 38 (five to eight heads:
// 70) of them and 720 other instructions of a warp, 1020 cycles where the memory's rate allows 880: of the 71 us below, that is 50.  The others are
// idle, a fifth to a quarter of the cycles, between an MMA, its sums, the maximum, the weights and the next MMA.  Two CTAs an SM with up to 255
// registers a thread: with three, 8 to 12 % more instructions, and no faster.  Measured: 8 sequences of 9000 to 65000 positions, 32/8 heads of 128, 71 us, 4.0 TB/s; 8 of 64000
// 151 us, 4.3 TB/s (64/8 heads 175); 64 of 16 to 4096, 12/2 heads of 128, 15.0 us; one of 672, 14/2 heads of 64, 5.4 us.
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
// What beginning and ending a pair costs, in tiles: lengths, table, first tiles and the meeting are memory round trips after one
// another.  Measured with 3, 6, 9 and 12: 64 sequences of 100 to 4000, 32/8 heads of 128, 52.8, 43.5, 39.3 and 39.2 us; 4 of 30000, 12/2
// heads of 128, 26.1, 23.3, 22.6 and 22.5; 64 of 16 to 4096, 14/2 heads of 64, 12.0, 11.1, 11.1 and 11.5.
constexpr int P4_FIXED = 9;
constexpr float P4_TOP = 15.0f;     // log2 of the largest weight as it is split: f16 ends at 65504
constexpr float P4_LEAST_V = -15.0f;  // f16 has the inverse of 2^this
using Cut = PaCut<P4_TILE, P4_FIXED>;

template <int D, int W = PA_WARPS> struct P4Shape {
    static constexpr int TILE = Q41<D>::TILE;
    static constexpr int STAGE = 4 * TILE;  // two tiles of K, two of V
    static constexpr int STAGES = D == 64 ? 5 : W > PA_WARPS ? 4 : 3;
    static constexpr int CTAS = W > PA_WARPS ? 1 : D == 64 ? 3 : 2;  // per SM
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
// (x, y) as f16 and what the rounding left, as f16: 22 bits together
CFI_DEV void split2(f2 x, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(both(x).x, both(x).y);
    const float2 f = __half22float2(h);
    *hi = h2_bits(h);
    *lo = h2_bits(__floats2half2_rn(both(x).x - f.x, both(x).y - f.y));
}
CFI_DEV void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {  // the sum begins with it
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
// Adds the sums of an MMA, rounded.  (An MMA cuts its own result to 24 bits: where it kept the sums of a whole run, all of positive
// products, they would be short by half a unit for each tile.)
CFI_DEV void add4(float (&d)[4], const float (&x)[4]) {
    const float2 a = both(add2(pair2(d[0], d[1]), pair2(x[0], x[1]))), b = both(add2(pair2(d[2], d[3]), pair2(x[2], x[3])));
    d[0] = a.x, d[1] = a.y, d[2] = b.x, d[3] = b.y;
}
CFI_DEV void mma_k8(float (&d)[4], const uint32_t (&a)[2], uint32_t b) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5}, {%6}, {%7, %7, %7, %7};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(b), "f"(0.0f));
}
// Rows of digits by a block's nibbles; the sums are read as floats, 1.5 2^23 more than they are.
constexpr float P4_MAGIC = 12582912.0f;
CFI_DEV void mma_digits(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    int e[4];
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %10, %10, %10};"
                 : "=r"(e[0]), "=r"(e[1]), "=r"(e[2]), "=r"(e[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "r"(0x4b400000));
#pragma unroll
    for (int i = 0; i < 4; i++) d[i] = __int_as_float(e[i]);
}
CFI_DEV void ldsm_x2_trans(uint32_t a, uint32_t& r0, uint32_t& r1) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];" : "=r"(r0), "=r"(r1) : "r"(a));
}
// The lower byte of each half, without and with its upper nibble, as f16 numbers; then the upper byte.
struct Nibbles {
    uint32_t x0, y0, x1, y1;
    CFI_DEV explicit Nibbles(uint32_t w) {
        const uint32_t a = __byte_perm(w, 0x64646464u, 0x4240), b = __byte_perm(w, 0x64646464u, 0x4341);
        x0 = less(a & 0xff0fff0fu);
        y0 = less(a);
        x1 = less(b & 0xff0fff0fu);
        y1 = less(b);
    }
    static CFI_DEV uint32_t less(uint32_t w) {
        return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&w), __half2half2(__ushort_as_half(0x6400))));
    }
};
// column 2 c + e of the n-th eight scores
CFI_DEV int position_of(int c, int e, int n) { return 8 * n + 4 * e + (c ^ (3 * e)); }

CFI_DEV __half2 as_h2(uint32_t w) { return *reinterpret_cast<const __half2*>(&w); }

// The largest of V's scales so far: they have been below 2^top, and what the weights are multiplied by is divided by it.
struct ScalesTop {
    float top, per;  // per: 2^-top
    __half2 limit, least;  // 2^top; the least scale but 0 that divided by it is a normal f16 number
    CFI_DEV void set(float t) {
        top = t;
        per = ex2(-t);
        limit = __float2half2_rn(ex2(t));
        least = __float2half2_rn(ex2(t - 14.0f));
    }
    // Looks at a tile's scales, some a lane.  Where one passes `top`, raises it: `by` is what the sums so far have to be multiplied by, or
    // 1.  True where a scale is so far below the largest that f16 would not hold it over 2^top.
    template <int D> CFI_DEV bool look(uint32_t sv, float* by) {
        const int lane = threadIdx.x & 31;
        __half2 d[D / 64], most = __float2half2_rn(0.0f);
#pragma unroll
        for (int x = 0; x < D / 64; x++) {
            d[x] = abs_h2(lds32(sv + (lane >> 4) * Q41<D>::TILE + Q41<D>::NIBBLES + (lane & 15) * Q41<D>::PARAM_ROW + 4 * x));
            most = __hmax2_nan(most, d[x]);
        }
        *by = 1.0f;
        if (__any_sync(0xffffffffu, !__hblt2(most, limit))) {
            // the exponent of the largest finite one: an infinity or a NaN spoils its own dims and says nothing of the others
            most = __float2half2_rn(0.0f);
#pragma unroll
            for (int x = 0; x < D / 64; x++)
                most = __hmax2(most, as_h2(h2_bits(d[x]) & __hlt2_mask(d[x], __half2half2(__ushort_as_half(0x7c00)))));
            const uint32_t ex = __float_as_uint(fmaxf(__low2float(most), __high2float(most))) >> 23;
            const float old = top;
            set(fmaxf(top, (float)__reduce_max_sync(0xffffffffu, ex) - 126.0f));
            *by = ex2(old - top);
        }
        uint32_t small = 0;
#pragma unroll
        for (int x = 0; x < D / 64; x++) small |= __hlt2_mask(d[x], least) & __hne2_mask(d[x], __float2half2_rn(0.0f));
        return __any_sync(0xffffffffu, small != 0);
    }
};
// Scales of two rows of blocks 0, 1 and 2, 3
template <int D> CFI_DEV void scales_of(uint32_t tile, int row, uint32_t (&d)[D / 64]) {
    const uint32_t p = tile + Q41<D>::NIBBLES + row * Q41<D>::PARAM_ROW;
    if (D == 128) {
        const uint2 x = lds64(p);
        d[0] = x.x, d[D / 64 - 1] = x.y;
    } else {
        d[0] = lds32(p);
    }
}
// This lane's eight dims of each block of a row of K
template <int D> CFI_DEV void dims_of_k(uint32_t tile, int row, uint32_t (&w)[D / 32]) {
    const int c = threadIdx.x & 3;
    if (D == 128) {
        const uint4 x = lds128(tile + row * Q41<D>::ROW + c * 16);
        w[0] = x.x, w[1] = x.y, w[D / 32 - 2] = x.z, w[D / 32 - 1] = x.w;
    } else {
        const uint2 x = lds64(tile + row * Q41<D>::ROW + c * 8);
        w[0] = x.x, w[1] = x.y;
    }
}
// This lane's four dims of blocks 0, 1 and 2, 3 of a row of V
template <int D> CFI_DEV void dims_of_v(uint32_t tile, int row, uint32_t (&w)[D / 64]) {
    const int g = threadIdx.x >> 2 & 7;
    const uint32_t q = tile + row * Q41<D>::ROW + Q41<D>::v_group(row, g) * (D / 16);
    if (D == 128) {
        const uint2 x = lds64(q);
        w[0] = x.x, w[D / 64 - 1] = x.y;
    } else {
        w[0] = lds32(q);
    }
}
// The tile's scales and minima, turned: of number g of a row, positions of columns 2 c and 2 c + 1 of both eights
template <int D> CFI_DEV void params_turned(uint32_t tile, uint32_t& b0, uint32_t& b1) {
    const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
    if (D == 128) {
        ldsm_x2_trans(tile + Q41<D>::NIBBLES + position_of(lane >> 1 & 3, lane & 1, lane >> 3 & 1) * Q41<D>::PARAM_ROW, b0, b1);
    } else {  // rows of four numbers: g & 3
        uint32_t x[4];
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = lds16(tile + Q41<D>::NIBBLES + position_of(c, e & 1, e >> 1) * Q41<D>::PARAM_ROW + 2 * (g & 3));
        b0 = x[0] | x[1] << 16;
        b1 = x[2] | x[3] << 16;
    }
}

// A lane's query values, dims 32 b + 8 c .. + 7 of head g (FEW: g & 3), as MMA operands over `unit`; and the sums of the blocks over 2^6
// where a row of scales and minima (2 NB numbers, of which a lane has two) has its minima.
template <int D, bool FEW> struct Queries {
    static constexpr int NB = D / 32;
    uint32_t a[FEW ? NB : 2 * NB][4], sums[2];
    float unit;
    CFI_DEV void convert(float (&qv)[NB][8], float scale_log2) {
        const int lane = threadIdx.x & 31, c = lane & 3;
        float largest = 0.0f;  // a NaN is passed over
        bool odd = false;      // NaN or an infinity among them
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 8; e++) {
                qv[b][e] *= scale_log2;
                largest = fmaxf(largest, fabsf(qv[b][e]));
                odd |= !(fabsf(qv[b][e]) < INFINITY);
            }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // 2^(its exponent - 14) and the other way round, both normal: below 2^-111 the largest stays below 2^14
        const uint32_t exponent = max(__float_as_uint(largest) >> 23, 15u);
        unit = __uint_as_float((exponent - 14) << 23);
        const float per_unit = __uint_as_float((268 - exponent) << 23);
        float sum[NB];
#pragma unroll
        for (int b = 0; b < NB; b++) {
            sum[b] = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                qv[b][e] *= per_unit;
                sum[b] += qv[b][e];
            }
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 1);
            sum[b] += __shfl_xor_sync(0xffffffffu, sum[b], 2);
            if (FEW) {
                // digits of q 2^15: rows 0-3 have the first of heads 0-3, rows 4-7 the second, 8-11 the third, 12-15 the last; bytes of a
                // register are dims 0, 2, 4, 6 of the lane's, or 1, 3, 5, 7
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    uint32_t d[4] = {0, 0, 0, 0};  // from the last
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        int v = __float2int_rn(qv[b][2 * e + x] * 32768.0f);
#pragma unroll
                        for (int k = 0; k < 4; k++) {
                            d[k] |= (uint32_t)(v & 0xff) << (8 * e);
                            v = (v - (int)(int8_t)(v & 0xff)) >> 8;
                        }
                    }
                    a[b][2 * x] = lane < 16 ? d[3] : d[2];
                    a[b][2 * x + 1] = lane < 16 ? d[1] : d[0];
                }
            } else {
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const float y0 = qv[b][2 * k + 1] * 0.0625f, y1 = qv[b][2 * k + 5] * 0.0625f;
                    split(qv[b][2 * k] - y0, qv[b][2 * k + 4] - y1, &a[(2 * b + k) % (FEW ? NB : 2 * NB)][0], &a[(2 * b + k) % (FEW ? NB : 2 * NB)][1]);
                    split(y0, y1, &a[(2 * b + k) % (FEW ? NB : 2 * NB)][2], &a[(2 * b + k) % (FEW ? NB : 2 * NB)][3]);
                }
            }
        }
        // a NaN or an infinity has no digits: it reaches the scores by its sum
        const int x = 2 * c - NB;
        float s0 = x == 0 ? sum[0] : NB == 4 && x == 2 ? sum[NB - 2] : 0.0f, s1 = x == 0 ? sum[1] : NB == 4 && x == 2 ? sum[NB - 1] : 0.0f;
        if (FEW && odd) s0 = s1 = NAN;
        split(s0 * 0.015625f, s1 * 0.015625f, &sums[0], &sums[1]);
    }
};

// What a warp keeps of up to eight heads (FEW: four).  A lane has the scores of head g (g & 3, lanes g and g + 4 the same) in columns 2 c
// and 2 c + 1 of a tile's four eights.
template <int D, bool FEW> struct Heads {
    static constexpr int NB = D / 32;
    Queries<D, FEW> q;
    // o has 2^-top in it.  Of columns 2 c and 2 c + 1, dims 32 b + 4 g + 2 x and the next one, which has 16 times itself and the first;
    // a column is a head, or (FEW, from 4 on) what f16 left of a head's weights
    float o[NB][2][4], mins[4], m;
    f2 l;
    ScalesTop v;
    static CFI_DEV int head() { return threadIdx.x >> 2 & (FEW ? 3 : 7); }  // whose queries this lane loads
    CFI_DEV void begin() {
        m = -INFINITY;
        l = 0;
        v.set(P4_LEAST_V);
#pragma unroll
        for (int e = 0; e < 4; e++) mins[e] = 0.0f;
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[b][0][e] = o[b][1][e] = 0.0f;
    }
    CFI_DEV void tile(uint32_t sk, uint32_t sv, int left) {
        using L = Q41<D>;
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        // ---- scores, over `unit` ----
        f2 s[4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const uint32_t tile = sk + (n >> 1) * L::TILE;
            const int row = position_of(g >> 1, g & 1, n & 1);
            float first[4];
            mma_k8(first, q.sums, lds32(tile + L::NIBBLES + row * L::PARAM_ROW + 4 * (c & (NB - 1))));
            const f2 low = add2(pair2(first[0], first[1]), pair2(first[2], first[3]));
            uint32_t w[NB], d0[NB / 2], d1[NB / 2];
            dims_of_k<D>(tile, row, w);
            scales_of<D>(tile, position_of(c, 0, n & 1), d0);
            scales_of<D>(tile, position_of(c, 1, n & 1), d1);
            f2 sum = 0;
#pragma unroll
            for (int b = 0; b < NB; b++) {
                const f2 scale = pair2(half_of(d0[b >> 1], b & 1), half_of(d1[b >> 1], b & 1));
                float acc[4];
                if (FEW) {
                    mma_digits(acc, q.a[b], w[b] & 0x0f0f0f0fu, w[b] >> 4 & 0x0f0f0f0fu);
                    // 2^16 times rows g and rows g + 8
                    const f2 upper = fma2(pair2(acc[0], acc[1]), pair2(65536.0f, 65536.0f), pair2(-65536.0f * P4_MAGIC, -65536.0f * P4_MAGIC)),
                             lower = add2(pair2(acc[2], acc[3]), pair2(-P4_MAGIC, -P4_MAGIC));
                    sum = fma2(add2(upper, lower), scale, sum);
                } else {
                    const Nibbles k(w[b]);
                    mma_first(acc, q.a[(2 * b) % (FEW ? NB : 2 * NB)], k.x0, k.y0);
                    mma_f16f32(acc, q.a[(2 * b + 1) % (FEW ? NB : 2 * NB)], k.x1, k.y1);
                    sum = fma2(add2(pair2(acc[0], acc[1]), pair2(acc[2], acc[3])), scale, sum);
                }
            }
            if (FEW) {  // the first digits are 2^8 the second ones', which lanes g and g + 4 have
                const float by = lane < 16 ? 256.0f / 32768.0f : 1.0f / 32768.0f;
                sum = mul2(sum, pair2(by, by));
                sum = add2(sum, pair2(__shfl_xor_sync(0xffffffffu, both(sum).x, 16), __shfl_xor_sync(0xffffffffu, both(sum).y, 16)));
            }
            s[n] = fma2(low, pair2(64.0f, 64.0f), sum);
        }
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
            const float mn = fmaxf(m, mx), alpha = m == -INFINITY ? 0.0f : ex2((m - mn) * q.unit);
            l = mul2(l, pair2(alpha, alpha));
            const int from = 8 * (FEW ? c & 1 : c);
            const float a0 = __shfl_sync(0xffffffffu, alpha, from), a1 = __shfl_sync(0xffffffffu, alpha, from + 4);
#pragma unroll
            for (int e = 0; e < 4; e++) mins[e] *= alpha;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int x = 0; x < 2; x++) o[b][x][0] *= a0, o[b][x][1] *= a1, o[b][x][2] *= a0, o[b][x][3] *= a1;
            m = mn;
        }
        const float sub = m == -INFINITY ? 0.0f : -m;  // P4_TOP is added last: a large score would swallow it
        f2 p[4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const float2 x = both(fma2(add2(s[n], pair2(sub, sub)), pair2(q.unit, q.unit), pair2(P4_TOP, P4_TOP)));
            p[n] = pair2(ex2(x.x), ex2(x.y));
            l = add2(l, p[n]);
        }
        // ---- weighted values: A is V with dims as rows, B the weights ----
        float by;
        const bool wide = v.template look<D>(sv, &by);
        if (by != 1.0f) {
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 4; e++) o[b][0][e] *= by, o[b][1][e] *= by;
        }
        if (wide)
            values<true>(sv, p);
        else
            values<false>(sv, p);
    }
    // Adds the weighted values of a tile.  The weights p, f16 values and the rest, are multiplied by the scales over 2^top in f16: h = hi d
    // rounded, and what that left (exact in one fused product) with lo d.  WIDE: in 32 bits, where some of these scales are not f16 numbers.
    template <bool WIDE> CFI_DEV void values(uint32_t sv, const f2 (&p)[4]) {
        using L = Q41<D>;
        const int c = threadIdx.x & 3;
        const uint32_t rest = (threadIdx.x & 31) < 16 ? 0u : 0xffffffffu;  // FEW: lanes whose column is what f16 left
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const uint32_t tile = sv + t * L::TILE;
            uint32_t pf[4], b0, b1;
#pragma unroll
            for (int n = 0; n < 2; n++) split2(p[2 * t + n], &pf[2 * n], &pf[2 * n + 1]);
            // minima: column x of a row's scales and minima, of which those from NB on count
            params_turned<D>(tile, b0, b1);
            float sums[4];
            mma_first(sums, pf, b0, b1);
            add4(mins, sums);
            uint32_t w[2][2][NB / 2], d[2][2][NB / 2];  // of column 2 c + e of eight n
            const __half2 per = __float2half2_rn(v.per);
#pragma unroll
            for (int n = 0; n < 2; n++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    dims_of_v<D>(tile, position_of(c, e, n), w[n][e]);
                    scales_of<D>(tile, position_of(c, e, n), d[n][e]);
                    if (!WIDE) {
#pragma unroll
                        for (int x = 0; x < NB / 2; x++) d[n][e][x] = h2_bits(__hmul2(as_h2(d[n][e][x]), per));
                    }
                }
#pragma unroll
            for (int b = 0; b < NB; b++) {
                uint32_t hi[2], lo[2], z[2];
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    if (WIDE) {
                        const f2 scale = pair2(half_of(d[n][0][b >> 1], b & 1) * v.per, half_of(d[n][1][b >> 1], b & 1) * v.per);
                        split2(mul2(p[2 * t + n], scale), &hi[n], &lo[n]);
                        if (FEW) hi[n] = rest ? lo[n] : hi[n];
                    } else {
                        const __half2 scale = as_h2(__byte_perm(d[n][0][b >> 1], d[n][1][b >> 1], b & 1 ? 0x7632 : 0x5410));
                        if (FEW) {  // with the masked ones 0: hi d rounded; with them whole: what that leaves, and lo d
                            const __half2 h = __hmul2(as_h2(pf[2 * n] & rest), scale);
                            hi[n] = h2_bits(__hfma2(as_h2(pf[2 * n + 1] & rest), scale, __hfma2(as_h2(pf[2 * n]), scale, __hneg2(h))));
                        } else {
                            const __half2 h = __hmul2(as_h2(pf[2 * n]), scale);
                            hi[n] = h2_bits(h);
                            lo[n] = h2_bits(__hfma2(as_h2(pf[2 * n + 1]), scale, __hfma2(as_h2(pf[2 * n]), scale, __hneg2(h))));
                        }
                    }
                    z[n] = __byte_perm(w[n][0][b >> 1], w[n][1][b >> 1], b & 1 ? 0x7632 : 0x5410);  // dims 32 b + 4 g .. + 3 of two positions
                }
                const Nibbles v0(z[0]), v1(z[1]);
                const uint32_t r0[4] = {v0.x0, v0.y0, v1.x0, v1.y0}, r1[4] = {v0.x1, v0.y1, v1.x1, v1.y1};
                float s0[4], s1[4];
                if (FEW) {
                    mma_first(s0, r0, hi[0], hi[1]);
                    mma_first(s1, r1, hi[0], hi[1]);
                } else {
                    mma_first(s0, r0, lo[0], lo[1]);
                    mma_first(s1, r1, lo[0], lo[1]);
                    mma_f16f32(s0, r0, hi[0], hi[1]);
                    mma_f16f32(s1, r1, hi[0], hi[1]);
                }
                add4(o[b][0], s0);
                add4(o[b][1], s1);
            }
        }
    }
    // Values, maximum and sum of each head as rows of `row` floats.
    CFI_DEV void finish(float* meet, int row) {
        const int lane = threadIdx.x & 31, g = lane >> 2, c = lane & 3;
        const float back = ex2(v.top);  // each warp has had scales of its own
        float sum = both(l).x + both(l).y;
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
        for (int b = 0; b < NB; b++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const float low = __shfl_sync(0xffffffffu, mins[b & 1] + mins[2 + (b & 1)], 4 * (2 * c + e) + (NB + b) / 2);  // column NB + b
                float f[4];
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    float u = o[b][x][e], w = o[b][x][2 + e];
                    if (FEW) u += __shfl_xor_sync(0xffffffffu, u, 2), w += __shfl_xor_sync(0xffffffffu, w, 2);
                    f[2 * x] = fmaf(u, back, low);
                    f[2 * x + 1] = fmaf(w - u, back / 16.0f, low);
                }
                if (!FEW || c < 2) *reinterpret_cast<float4*>(meet + (2 * c + e) * row + 32 * b + 4 * g) = make_float4(f[0], f[1], f[2], f[3]);
            }
        if (c == 0 && (!FEW || g < 4)) *reinterpret_cast<float2*>(meet + g * row + D) = make_float2(m * q.unit, sum);
    }
};

template <int D, int W, bool FEW>
__global__ void __launch_bounds__(W * 32, (P4Shape<D, W>::CTAS)) paged_attn_q4(const PaArgs a) {
    using S = P4Shape<D, W>;
    using L = Q41<D>;
    constexpr int NB = D / 32;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_last[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, c = lane & 3;
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
        const int h = Heads<D, FEW>::head();
        float qv[NB][8];
#pragma unroll
        for (int b = 0; b < NB; b++) {
#pragma unroll
            for (int e = 0; e < 8; e++) qv[b][e] = 0.0f;
            if (h < nh) {
                const long long o = seq * a.q_stride + (long long)(head0 + h) * D + 32 * b + 8 * c;
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

        const uint32_t page_bytes = a.n_kv_head * (uint32_t)paged_region_bytes<D, CACHE_Q4_1>(page_size);
        const uint8_t *k_lane = a.k + kvh * paged_region_bytes<D, CACHE_Q4_1>(page_size) + lane * 16, *v_lane = k_lane + (a.v - a.k);
        auto fetch = [&](int i) {  // tile i of this warp into its stage
            if (i < mine) {
                const int p0 = (t0 + warp + i * W) * P4_TILE, left = len - p0;
                const uint32_t page0 = __shfl_sync(0xffffffffu, id0, i & 31), page1 = __shfl_sync(0xffffffffu, id1, i & 31);
                const uint32_t st = ring + (i % S::STAGES) * S::STAGE + lane * 16;
                const uint64_t o0 = (uint64_t)page0 * page_bytes + L::tile_at(p0 & (page_size - 1)),
                               o1 = (uint64_t)page1 * page_bytes + L::tile_at((p0 + Q41_TILE) & (page_size - 1));
                // Scales and minima: a chunk a lane, of 4 CH for the four tiles.  Rows past the length get zeros, so that what a page holds
                // there never matters.
                constexpr int CH = Q41_TILE * L::PARAM_ROW / 16, ROWS = Q41_TILE / CH, N = 32 / CH;  // of a tile; rows of a chunk; tiles a warp
                const int n = lane / CH, half = n & 1;
                const uint64_t op = half ? o1 : o0;
                const uint32_t to = st + n * (S::TILE - 16 * CH) + L::NIBBLES;  // st counts all lanes before
                const uint8_t* from = (N == 4 && n >= 2 ? v_lane : k_lane) + op + (L::NIBBLES - 16 * CH * n);
                if (left >= P4_TILE) {
#pragma unroll
                    for (int e = 0; e < L::NIBBLES / 512; e++) {
                        cp_async16_cg(st + e * 512, k_lane + o0 + e * 512);
                        cp_async16_cg(st + S::TILE + e * 512, k_lane + o1 + e * 512);
                        cp_async16_cg(st + 2 * S::TILE + e * 512, v_lane + o0 + e * 512);
                        cp_async16_cg(st + 3 * S::TILE + e * 512, v_lane + o1 + e * 512);
                    }
                    cp_async16_cg(to, from);
                    if (N == 2) cp_async16_cg(to + 2 * S::TILE, from + (a.v - a.k));
                } else {
                    const int two = left > Q41_TILE ? 16 : 0;  // is there a second half?
#pragma unroll
                    for (int e = 0; e < L::NIBBLES / 512; e++) {
                        cp16n(st + e * 512, k_lane + o0 + e * 512, 16);
                        cp16n(st + S::TILE + e * 512, k_lane + o1 + e * 512, two);
                        cp16n(st + 2 * S::TILE + e * 512, v_lane + o0 + e * 512, 16);
                        cp16n(st + 3 * S::TILE + e * 512, v_lane + o1 + e * 512, two);
                    }
                    const int bytes = min(max((left - half * Q41_TILE - lane % CH * ROWS) * L::PARAM_ROW, 0), 16);
                    cp16n(to, from, bytes);
                    if (N == 2) cp16n(to + 2 * S::TILE, from + (a.v - a.k), bytes);
                }
            }
            cp_async_commit();
        };

        Heads<D, FEW> heads;
        heads.begin();
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
        heads.q.convert(qv, a.scale_log2);
        for (int i = 0; i < mine; i++) {
            if ((i + S::STAGES - 1) % 32 == 0) {
                id0 = load_id(i + S::STAGES - 1, 0);
                id1 = load_id(i + S::STAGES - 1, 1);
            }
            fetch(i + S::STAGES - 1);
            cp_async_wait<S::STAGES - 1>();
            __syncwarp();
            const uint32_t st = ring + (i % S::STAGES) * S::STAGE;
            heads.tile(st, st + 2 * S::TILE, len - (t0 + warp + i * W) * P4_TILE);
            __syncwarp();  // the stage is free
        }
        // ---- the warps meet: [warp][head]: D values, maximum, sum ----
        cp_async_wait<0>();
        __syncthreads();  // every warp is done with its stages
        float* meet = reinterpret_cast<float*>(smem);
        heads.finish(meet + warp * S::MEET, S::MEET_ROW);
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

template <int D, int W, bool FEW> int launch(PaArgs& a, long long pairs, long long most_units, cudaStream_t stream) {
    using S = P4Shape<D, W>;
    static CfiPerDeviceOnce once;
    cfi_once_per_device(once, [] { cudaFuncSetAttribute(paged_attn_q4<D, W, FEW>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
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
    return (int)cudaLaunchKernelEx(&lc, paged_attn_q4<D, W, FEW>, (const PaArgs)a);
}

}  // namespace

int cfi_paged_attention_q4_1(PaArgs& a, int head_dim, long long pairs, cudaStream_t stream) {
    const long long positions = (long long)a.max_pages << a.page_shift;
    const long long most_units = pairs * (P4_FIXED + (positions + P4_TILE - 1) / P4_TILE);
    // Short tables: a CTA to a pair, which neither reads all lengths nor joins anything; eight warps where an SM has one pair at most, four
    // otherwise.  Measured against the equal runs (us, lengths from a quarter of the longest; 14/2 heads of 64, 12/2 of 128): one
    // sequence of 768 5.5 to 7.4 and 7.8 to 9.7, of 1280 7.6 to 7.6 and 11.1 to 9.9, of 2048 10.8 to 7.9 and 15.7 to 10.2; 16 of 1024 6.8 to
    // 8.9 and 9.6 to 11.6, of 2048 10.9 to 9.9 and 15.8 to 12.3; 64 of 2048 11.2 to 11.3 and 16.4 to 16.4; four warps, 128 of 512 8.3 to 10.8
    // and 9.7 to 14.5, of 1024 13.6 to 12.5 and 15.8 to 17.8; 64 of 2048 with 32/8 heads of 128 40.7 to 37.8.
    const int sms = cfi_sm_count();
    const int w = pairs <= sms ? (positions <= (2 * pairs > sms ? 2048 : 1024) ? 8 : 0) : positions <= (head_dim == 128 ? 1024 : 768) ? 4 : 0;
    a.whole = w > 0;
    const int variant = (head_dim == 128) * 4 + (w == 8) * 2 + (a.group <= 4);
    switch (variant) {
        case 0: return launch<64, PA_WARPS, false>(a, pairs, most_units, stream);
        case 1: return launch<64, PA_WARPS, true>(a, pairs, most_units, stream);
        case 2: return launch<64, 8, false>(a, pairs, most_units, stream);
        case 3: return launch<64, 8, true>(a, pairs, most_units, stream);
        case 4: return launch<128, PA_WARPS, false>(a, pairs, most_units, stream);
        case 5: return launch<128, PA_WARPS, true>(a, pairs, most_units, stream);
        case 6: return launch<128, 8, false>(a, pairs, most_units, stream);
        default: return launch<128, 8, true>(a, pairs, most_units, stream);
    }
}
