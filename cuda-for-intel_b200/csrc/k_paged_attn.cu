// k_paged_attn.cu -- attention of one new token per sequence over a paged key-value cache
// (include/cfi_serve.h): out = sum_j softmax_j(scale q.K_j) V_j over the sequence's positions.
//
// Bound by HBM: every cached row is read once for the query heads that share it.  The list of all
// 16-position tiles of all (sequence, kv head) pairs is cut into equal runs, one per CTA, whatever the
// lengths: no CTA waits for the longest sequence.  The lengths are read on the device, so every CTA
// works out the same cuts.  A pair whose tiles lie in several CTAs leaves partial sums (row maximum,
// sum, weighted values) in the stream's workspace; the last of its CTAs to finish joins them in CTA order,
// so that the result does not depend on which one that was.
//
// Each of a CTA's four warps walks every fourth tile with its own ring of cp.async stages (rows past the
// length are filled with zeros, so what a page holds there never matters) and a running maximum.
// The products run on mma.sync m16n8k16 with at most 8 query heads: rows 0-7 of A are the heads'
// f16 values and rows 8-15 what f16 rounding left of them, so one MMA multiplies operands of 22 bits
// and the two halves of its result are added.  The same holds for the weights.  A group of more than 8
// heads is cut into chunks that read the rows again (from L2).
//
// A query head is split times the power of two that brings its largest value to 2^14 .. 2^15 (the scores are divided by it again
// in the exponent), and a weight at 2^15 times its size: what f16 leaves of either ends at 2^-39 of the largest, and a long tail
// of small weights stays as large as the sum of them that the result is divided by.
//
// Q8_0: int8 values are exact in f16, so K enters the MMA as whole numbers, one block of 32 dims at
// a time, and each block's sum is multiplied by its scale in 32 bits; V's scales are multiplied into the
// weights before these are split, in units of the power of two above the largest scale so far (the sums are rescaled where
// that grows, as they are where the maximum does).
//
// Measured: 8 sequences of 9000 to 65000 positions, 32/8 heads of 128 in f16, 146 us, 6.2 TB/s; 64 of 16 to 4096, 12/2 heads
// of 128 in Q8_0, 20.9 us (36 MB; the work of a tile, some 600 instructions of a warp, is what it waits for:
// the warps of three CTAs issue in 45 % of the cycles); one of 672, 14/2 heads of 64 in f16, 5.9 us, 5.1 of them on the device:
// launch, table, one round of loads and the join.
#include "paged_cache.cuh"
#include "paged_cut.h"
#include "sm100_ptx.cuh"
#include "mma_sync.cuh"
#include "cfi_kernels.h"

#include <algorithm>
#include <math.h>
#include <stdlib.h>
#include <string.h>

namespace {

using namespace sm100;

constexpr int PA_WARPS = 4;        // of a CTA; twice as many where a CTA has a pair and an SM to itself
constexpr int PA_HEADS = 8;        // query heads of a chunk
constexpr int PA_TILE = 16;        // positions; a page is a multiple of it
constexpr float PA_TOP = 15.0f;    // log2 of the largest weight as it is split: f16 ends at 65504
constexpr float PA_LEAST_V = -23.0f, PA_MOST_V = 16.0f;  // f16 scales are below 2^these
// What beginning and ending a pair costs, in tiles: a run's share of the list counts it, so that CTAs with
// many short sequences get fewer tiles.
constexpr int PA_FIXED = 5;
constexpr int PA_KEPT = 4;

template <int D, bool Q8, int W = PA_WARPS> struct PaShape {
    static constexpr int ROW = Q8 ? D : 2 * D;            // bytes of a row
    static constexpr int ROWS = PA_TILE * ROW;            // of a tile of K or V
    static constexpr int SCALES = Q8 ? PA_TILE * D / 16 : 0;
    static constexpr int STAGE = 2 * (ROWS + SCALES);
    static constexpr int STAGES = Q8 ? (D == 64 ? 6 : 4) : (D == 64 ? 4 : 3);
    static constexpr int CTAS = W > PA_WARPS ? 1 : Q8 ? 3 : (D == 64 ? 3 : 2);  // per SM
    static constexpr int RING = STAGES * STAGE;           // a warp's
    static constexpr int SMEM = W * RING;
    static constexpr int PART = PA_HEADS * (D + 2);       // floats of a partial result: values, then maximum and sum of each head
    // where the warps meet: a row is a head's values, maximum and sum (stores of the fragments meet no bank twice)
    static constexpr int MEET_ROW = D + (Q8 ? 4 : 8), MEET = PA_HEADS * MEET_ROW;
    static_assert(SMEM >= W * MEET * 4, "the warps meet in the stages' memory");
};

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
CFI_DEV __half2 abs_h2(uint32_t w) {
    w &= 0x7fff7fffu;
    return *reinterpret_cast<const __half2*>(&w);
}
// (x, y) as f16 and what the rounding left, as f16: 22 bits together
CFI_DEV void split(float x, float y, uint32_t* hi, uint32_t* lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    *hi = h2_bits(h);
    *lo = h2_bits(__floats2half2_rn(x - f.x, y - f.y));
}
// bytes `sel` of w (int8 with its sign bit flipped) as two f16: 0x6400 + u is 1024 + u, less 1152
CFI_DEV uint32_t s8_to_h2(uint32_t w, uint32_t sel) {
    const uint32_t u = __byte_perm(w, 0x64646464u, sel);
    return h2_bits(__hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480))));
}

// Byte offset of 16-byte chunk c of row r in a tile: chunks are exchanged so that the reads below
// take every bank once.
template <int D, bool Q8, bool V> CFI_DEV uint32_t chunk_at(int r, int c) {
    if (!Q8) return r * (2 * D) + ((c ^ (r & 7)) << 4);                    // ldmatrix: 8 rows, one chunk each
    if (D == 128) return r * 128 + ((c ^ (((V ? r >> 1 : r) & 3) << 1)) << 4);  // 4 rows, two chunks each
    // 64-byte rows, two to a line of banks
    const int half = V ? r >> 2 & 1 : r & 1, line = V ? (r & 3) | (r >> 3) << 2 : r >> 1;
    return line * 128 + half * 64 + ((c ^ ((r >> 1 & 1) << 1)) << 4);
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

// How the work is cut: a pair (kv head, chunk) of a sequence is PA_FIXED units and then one for each tile,
// the pairs of all sequences follow one another, and CTA b has the units b * quota .. (b + 1) * quota.
// There are less than 2^31.
struct PaCut {
    const int32_t* lens;
    int most, total, quota;
    int units[PA_KEPT];  // of the sequences that are this lane's, of the first 32 PA_KEPT, all loaded together
    CFI_DEV int length(int s) const { return max(0, min(lens[s], most)); }
    // an empty sequence still has its zeros to write
    static CFI_DEV int tiles_of(int len) { return max(1, (len + PA_TILE - 1) / PA_TILE); }
    CFI_DEV int units_of(int s) const { return PA_FIXED + tiles_of(length(s)); }
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
        quota = paged_quota(total, ctas, PA_FIXED + PA_WARPS);
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

template <int D, bool Q8, int W>
__global__ void __launch_bounds__(W * 32, (PaShape<D, Q8, W>::CTAS)) paged_attn(const PaArgs a) {
    using S = PaShape<D, Q8, W>;
    constexpr int NB = D / 32, NT = D / 8, KK = D / 16;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int s_last[2];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
    const int page_size = 1 << a.page_shift, hc = a.n_kv_head * a.chunks;
    pdl_launch_dependents();
    pdl_wait();

    PaCut cut(a);
    int begin = 0, end = 1, at = 0, seq = 0, seq_start = 0, pair = 0;  // seq_start: the sequence's first unit
    if (a.whole) {
        seq = blockIdx.x / hc;
        pair = blockIdx.x - seq * hc;
    } else {
        // ---- this CTA's run ----
        cut.read(a, gridDim.x);
        if ((int)blockIdx.x >= paged_runs(cut.total, cut.quota)) return;
        begin = at = blockIdx.x * cut.quota;
        end = paged_run_end(begin, cut.quota, cut.total);
        auto among = [&](int base, int n) {  // is it one of the 32 sequences from `base` on, this lane's with n units?
            int incl = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, seq_start + incl > at);
            const int l = hit ? __ffs(hit) - 1 : 31;
            seq = base + l;
            seq_start += __shfl_sync(0xffffffffu, hit ? incl - n : incl, l);
            return hit != 0;
        };
        bool found = false;
#pragma unroll
        for (int e = 0; e < PA_KEPT; e++)
            if (!found) found = among(32 * e, cut.units[e]);
        for (int base = 32 * PA_KEPT; !found && base < a.n_seq; base += 32)
            found = among(base, base + lane < a.n_seq ? cut.units_of(base + lane) * hc : 0);
    }

    const uint32_t ring = smem_u32(smem) + warp * S::RING;
    PaShared shared[2];  // of the pairs that it goes on with, and leaves unfinished
    while (at < end) {
        // ---- one (sequence, kv head, chunk): its tiles [t0, t1) of n_tiles ----
        const int len = cut.length(seq), n_tiles = PaCut::tiles_of(len);
        int t0 = 0, t1 = n_tiles;
        if (!a.whole) {
            const int units = PA_FIXED + n_tiles;
            pair = (at - seq_start) / units;
            const int first = seq_start + pair * units + PA_FIXED;
            t0 = max(0, at - first);
            t1 = min(n_tiles, end - first);
            at = first + n_tiles;
            if (t1 <= 0) break;  // the run ends before the pair's first tile
        } else {
            at = end;
        }
        const int kvh = pair / a.chunks, h0 = (pair - kvh * a.chunks) * PA_HEADS, nh = min(PA_HEADS, a.group - h0);
        const int head0 = kvh * a.group + h0;

        // page ids of this warp's next 32 tiles, one a lane
        const int32_t* trow = a.table + (long long)seq * a.max_pages;
        const int mine = t1 - t0 > warp ? (t1 - t0 - warp + W - 1) / W : 0;  // tiles of this warp
        auto load_ids = [&](int i) {
            const int t = t0 + warp + (i + lane) * W;
            return t < t1 && t * PA_TILE < len ? min(max(trow[t * PA_TILE >> a.page_shift], 0), a.n_pages - 1) : 0;
        };
        int ids = load_ids(0);

        // the queries: loaded here, converted when the first tiles are on their way.  A's k = 2c, 2c+1
        // (x 0) and 2c+8, 2c+9 (x 1) are dims in the order that K's fragments have
        float2 qv[KK][2];
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const int d = Q8 ? 32 * (kk >> 1) + 8 * c + 4 * (kk & 1) + 2 * x : 16 * kk + 2 * c + 8 * x;
                qv[kk][x] = make_float2(0.0f, 0.0f);
                if (g < nh) {
                    const long long o = seq * a.q_stride + (long long)(head0 + g) * D + d;
                    if (a.q_f16)
                        qv[kk][x].x = __uint_as_float(*reinterpret_cast<const uint32_t*>(a.q + o * 2));
                    else
                        qv[kk][x] = *reinterpret_cast<const float2*>(a.q + o * 4);
                }
            }

        auto fetch = [&](int i) {  // tile i of this warp into its stage
            if (i < mine) {
                const int t = t0 + warp + i * W, p0 = t * PA_TILE;
                const int page = __shfl_sync(0xffffffffu, ids, i & 31), off = p0 & (page_size - 1);
                const long long region = ((long long)page * a.n_kv_head + kvh) * paged_region_bytes<D, Q8>(page_size);
                const uint32_t st = ring + (i % S::STAGES) * S::STAGE;
                const int left = len - p0;
#pragma unroll
                for (int e = 0; e < S::ROWS / 512; e++) {
                    constexpr int CH = S::ROW / 16;
                    const int r = (e * 32 + lane) / CH, ch = (e * 32 + lane) % CH;
                    const long long src = region + (long long)(off + r) * S::ROW + ch * 16;
                    cp16z(st + chunk_at<D, Q8, false>(r, ch), a.k + src, r < left);
                    cp16z(st + S::ROWS + chunk_at<D, Q8, true>(r, ch), a.v + src, r < left);
                }
                if (Q8) {  // lanes 0-15 bring K's scales, 16-31 V's
                    const int r = lane & 15;
                    const uint8_t* src = (lane < 16 ? a.k : a.v) + region + (long long)page_size * D + (off + r) * (D / 16);
                    const uint32_t dst = st + 2 * S::ROWS + (lane < 16 ? 0 : S::SCALES) + r * (D / 16);
                    if (D == 128) cp8z(dst, src, r < left); else cp4z(dst, src, r < left);
                }
            }
            cp_async_commit();
        };

        // Q8_0: V's scales have been below 2^top_v; weights, l and o have 2^-top_v in them
        float o[NT][4], m = -INFINITY, l = 0.0f, top_v = Q8 ? PA_LEAST_V : 0.0f;
        __half2 limit_v = __float2half2_rn(ex2(top_v));
#pragma unroll
        for (int j = 0; j < NT; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) o[j][e] = 0.0f;
#pragma unroll
        for (int i = 0; i < S::STAGES - 1; i++) fetch(i);
        uint32_t qf[KK][4];  // in log2 units over `unit`, split
        float largest = 0.0f;  // a NaN is passed over
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int x = 0; x < 2; x++) {
                const uint32_t raw = __float_as_uint(qv[kk][x].x);
                const float2 f = a.q_f16 ? __half22float2(*reinterpret_cast<const __half2*>(&raw)) : qv[kk][x];
                qv[kk][x] = make_float2(f.x * a.scale_log2, f.y * a.scale_log2);
                largest = fmaxf(largest, fmaxf(fabsf(qv[kk][x].x), fabsf(qv[kk][x].y)));
            }
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
        // 2^(its exponent - 14) and the other way round, both normal: below 2^-111 the largest stays below 2^14
        const uint32_t exponent = max(__float_as_uint(largest) >> 23, 15u);
        const float unit = __uint_as_float((exponent - 14) << 23), per_unit = __uint_as_float((268 - exponent) << 23);
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int x = 0; x < 2; x++) split(qv[kk][x].x * per_unit, qv[kk][x].y * per_unit, &qf[kk][2 * x], &qf[kk][2 * x + 1]);
        for (int i = 0; i < mine; i++) {
            if ((i + S::STAGES - 1) % 32 == 0) ids = load_ids(i + S::STAGES - 1);
            fetch(i + S::STAGES - 1);
            cp_async_wait<S::STAGES - 1>();
            __syncwarp();
            const uint32_t sk = ring + (i % S::STAGES) * S::STAGE, sv = sk + S::ROWS, ss = sk + 2 * S::ROWS;
            // ---- scores, over `unit`, of positions 2c, 2c+1 and 8+2c, 9+2c for head g ----
            float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            if (!Q8) {
                float acc[2][4] = {};
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    uint32_t b[4];
                    ldsm_x4(sk + chunk_at<D, Q8, false>((lane >> 4) * 8 + (lane & 7), 2 * kk + (lane >> 3 & 1)), b);
                    mma_f16f32(acc[0], qf[kk], b[0], b[1]);
                    mma_f16f32(acc[1], qf[kk], b[2], b[3]);
                }
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    s[2 * n] = acc[n][0] + acc[n][2];
                    s[2 * n + 1] = acc[n][1] + acc[n][3];
                }
            } else {
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    uint32_t sc[NB];  // scales of positions 2c and 2c+1
                    if (D == 128) {
                        const uint4 w = lds128(ss + (8 * n + 2 * c) * 8);
                        sc[0] = w.x, sc[1] = w.y, sc[NB - 2] = w.z, sc[NB - 1] = w.w;
                    } else {
                        const uint2 w = lds64(ss + (8 * n + 2 * c) * 4);
                        sc[0] = w.x, sc[1] = w.y;
                    }
#pragma unroll
                    for (int b = 0; b < NB; b++) {
                        const uint2 w = lds64(sk + chunk_at<D, Q8, false>(8 * n + g, 2 * b + (c >> 1)) + 8 * (c & 1));
                        const uint32_t w0 = w.x ^ 0x80808080u, w1 = w.y ^ 0x80808080u;
                        float acc[4] = {};
                        mma_f16f32(acc, qf[2 * b], s8_to_h2(w0, 0x4140), s8_to_h2(w0, 0x4342));
                        mma_f16f32(acc, qf[2 * b + 1], s8_to_h2(w1, 0x4140), s8_to_h2(w1, 0x4342));
                        const float d0 = h2f_bits((uint16_t)(sc[b >> 1] >> (16 * (b & 1)))),
                                    d1 = h2f_bits((uint16_t)(sc[NB / 2 + (b >> 1)] >> (16 * (b & 1))));
                        s[2 * n] = fmaf(acc[0] + acc[2], d0, s[2 * n]);
                        s[2 * n + 1] = fmaf(acc[1] + acc[3], d1, s[2 * n + 1]);
                    }
                }
            }
            const int left = len - (t0 + warp + i * W) * PA_TILE;
            if (left < PA_TILE) {
#pragma unroll
                for (int e = 0; e < 4; e++)
                    if ((e >> 1) * 8 + 2 * c + (e & 1) >= left) s[e] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
            if (__any_sync(0xffffffffu, mx > m)) {
                const float mn = fmaxf(m, mx), alpha = m == -INFINITY ? 0.0f : ex2((m - mn) * unit);
                l *= alpha;
#pragma unroll
                for (int j = 0; j < NT; j++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[j][e] *= alpha;
                m = mn;
            }
            const float sub = m == -INFINITY ? 0.0f : m, rise = PA_TOP - top_v;  // added last: a large score would swallow it
            float p[4];
#pragma unroll
            for (int e = 0; e < 4; e++) p[e] = ex2(fmaf(s[e] - sub, unit, rise));
            l += (p[0] + p[1]) + (p[2] + p[3]);
            // ---- weighted values ----
            if (!Q8) {
                uint32_t pf[4];
                split(p[0], p[1], &pf[0], &pf[1]);
                split(p[2], p[3], &pf[2], &pf[3]);
#pragma unroll
                for (int j = 0; j < NT; j += 2) {
                    uint32_t b[4];
                    ldsm_x4_trans(sv + chunk_at<D, Q8, true>(lane & 15, j + (lane >> 4)), b);
                    mma_f16f32(o[j], pf, b[0], b[1]);
                    mma_f16f32(o[j + 1], pf, b[2], b[3]);
                }
            } else {
                uint32_t sc[2][NB];  // scales of positions 2c, 2c+1 and 8+2c, 9+2c
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    if (D == 128) {
                        const uint4 w = lds128(ss + S::SCALES + (8 * n + 2 * c) * 8);
                        sc[n][0] = w.x, sc[n][1] = w.y, sc[n][NB - 2] = w.z, sc[n][NB - 1] = w.w;
                    } else {
                        const uint2 w = lds64(ss + S::SCALES + (8 * n + 2 * c) * 4);
                        sc[n][0] = w.x, sc[n][1] = w.y;
                    }
                }
                // a lane looks at two of the tile's scales
                const __half2 d = abs_h2(lds32(ss + S::SCALES + (lane * 4 & (D - 1))));
                if (__any_sync(0xffffffffu, !__hblt2(d, limit_v))) {
                    // the exponent of the largest, cut where that is an infinity or a NaN
                    const uint32_t exponent = __float_as_uint(fmaxf(__low2float(d), __high2float(d))) >> 23;
                    const float grown = fmaxf(top_v, fminf((float)__reduce_max_sync(0xffffffffu, exponent) - 126.0f, PA_MOST_V));
                    const float f = ex2(top_v - grown);
                    l *= f;
#pragma unroll
                    for (int e = 0; e < 4; e++) p[e] *= f;
#pragma unroll
                    for (int j = 0; j < NT; j++)
#pragma unroll
                        for (int e = 0; e < 4; e++) o[j][e] *= f;
                    top_v = grown;
                    limit_v = __float2half2_rn(ex2(grown));
                }
#pragma unroll
                for (int b = 0; b < NB; b++) {
                    uint32_t pf[4], bw[2][4];
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const float d0 = h2f_bits((uint16_t)(sc[n][b >> 1] >> (16 * (b & 1)))),
                                    d1 = h2f_bits((uint16_t)(sc[n][NB / 2 + (b >> 1)] >> (16 * (b & 1))));
                        split(p[2 * n] * d0, p[2 * n + 1] * d1, &pf[2 * n], &pf[2 * n + 1]);
                        // dims 32 b + 4 g .. + 3 of two positions, interleaved: column g of MMA e is dim 32 b + 4 g + e
                        const uint32_t wa = lds32(sv + chunk_at<D, Q8, true>(8 * n + 2 * c, 2 * b + (g >> 2)) + 4 * (g & 3)) ^ 0x80808080u;
                        const uint32_t wb = lds32(sv + chunk_at<D, Q8, true>(8 * n + 2 * c + 1, 2 * b + (g >> 2)) + 4 * (g & 3)) ^ 0x80808080u;
                        const uint32_t x = __byte_perm(wa, wb, 0x5140), y = __byte_perm(wa, wb, 0x7362);
                        bw[n][0] = s8_to_h2(x, 0x4140);
                        bw[n][1] = s8_to_h2(x, 0x4342);
                        bw[n][2] = s8_to_h2(y, 0x4140);
                        bw[n][3] = s8_to_h2(y, 0x4342);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) mma_f16f32(o[4 * b + e], pf, bw[0][e], bw[1][e]);
                }
            }
            __syncwarp();  // the stage is free
        }
        // ---- the warps meet: [warp][head]: D values, maximum, sum ----
        cp_async_wait<0>();
        l += __shfl_xor_sync(0xffffffffu, l, 1);
        l += __shfl_xor_sync(0xffffffffu, l, 2);
        __syncthreads();  // every warp is done with its stages
        float* meet = reinterpret_cast<float*>(smem);
        float* mine_o = meet + warp * S::MEET + g * S::MEET_ROW;
        if (Q8) {
            const float back = ex2(top_v);  // each warp has had scales of its own
            l *= back;
#pragma unroll
            for (int b = 0; b < NB; b++)
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    float f[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) f[i] = (o[4 * b + i][e] + o[4 * b + i][e + 2]) * back;
                    *reinterpret_cast<float4*>(mine_o + 32 * b + 8 * c + 4 * e) = make_float4(f[0], f[1], f[2], f[3]);
                }
        } else {
#pragma unroll
            for (int j = 0; j < NT; j++)
                *reinterpret_cast<float2*>(mine_o + 8 * j + 2 * c) = make_float2(o[j][0] + o[j][2], o[j][1] + o[j][3]);
        }
        if (c == 0) *reinterpret_cast<float2*>(mine_o + D) = make_float2(m * unit, l);
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
    // ---- the results that are parts: the last of a pair's CTAs to come here joins them ----
    if (a.whole || (shared[0].id < 0 && shared[1].id < 0)) return;
    if (lane == 0 && warp < 2) {  // one thread for each
        const PaShared p = warp == 0 ? shared[0] : shared[1];
        bool last = false;
        if (p.id >= 0) {
            __threadfence();  // after a barrier: covers the stores of the whole CTA
            last = atomicAdd(&a.counters[p.id], 1u) == (unsigned)(p.n - 1);
            if (last) {
                __threadfence();
                a.counters[p.id] = 0u;
            }
        }
        s_last[warp] = last;
    }
    __syncthreads();
#pragma unroll
    for (int x = 0; x < 2; x++)
        if (s_last[x]) join_parts<S, D, W * 32>(a, shared[x]);
}

template <int D, bool Q8, int W> int launch(PaArgs& a, long long pairs, long long most_units, cudaStream_t stream) {
    using S = PaShape<D, Q8, W>;
    static CfiPerDeviceOnce once;
    cfi_once_per_device(once, [] { cudaFuncSetAttribute(paged_attn<D, Q8, W>, cudaFuncAttributeMaxDynamicSharedMemorySize, S::SMEM); });
    long long grid = pairs;
    if (!a.whole) {
        // no CTA has fewer units than this
        const long long ctas = (long long)cfi_sm_count() * S::CTAS;
        grid = std::min(ctas, most_units / (PA_FIXED + PA_WARPS) + 1);
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
    return (int)cudaLaunchKernelEx(&lc, paged_attn<D, Q8, W>, (const PaArgs)a);
}

}  // namespace

extern "C" int cfi_paged_attention(const CfiPagedCache* c, const void* q, int q_type, long long q_stride, void* out,
                                   int out_type, long long out_stride, const int32_t* table, int max_pages,
                                   const int32_t* lens, int n_seq, int n_head, float scale, void* stream) {
    if (!cfi_paged_ok(c) || !q || !out || !table || !lens || (q_type != 0 && q_type != 1) || (out_type != 0 && out_type != 1) ||
        n_seq < 0 || n_seq > 65535 || max_pages <= 0 || n_head <= 0 || n_head > 65535 || n_head % c->n_kv_head ||
        (((uintptr_t)q | (uintptr_t)out) & 15) || (((uintptr_t)table | (uintptr_t)lens) & 3) || q_stride % 8 || out_stride % 8 ||
        q_stride < (long long)n_head * c->head_dim || out_stride < (long long)n_head * c->head_dim || !(scale > 0.0f) || isinf(scale))
        return (int)cudaErrorInvalidValue;
    if (n_seq == 0) return 0;
    PaArgs a = {};
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
    a.chunks = (a.group + PA_HEADS - 1) / PA_HEADS;
    a.max_pages = max_pages;
    a.n_seq = n_seq;
    a.q_f16 = q_type;
    a.out_f16 = out_type;
    a.scale_log2 = scale * 1.4426950408889634f;
    const long long pairs = (long long)n_seq * c->n_kv_head * a.chunks;
    const long long most_units = pairs * (PA_FIXED + (long long)max_pages * (c->page_size / PA_TILE));
    if (most_units > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const long long positions = (long long)max_pages * c->page_size;
    // Short tables: a CTA to a pair, which neither reads all lengths nor joins anything.  Measured against the equal
    // runs (us, every sequence but one up to four times shorter than the longest; 14/2 heads of 64 in f16, then 12/2 of
    // 128 in Q8_0): eight warps, 1 sequence of 768 5.1 to 6.0 and 9.0 to 8.0, of 2048 9.6 to 6.3 and 19 to 9.6; 64
    // sequences of 1536 8.2 to 11 and 15 to 16, of 2048 10 to 11 and 19 to 19; four warps, three CTAs to an SM, 128
    // sequences of 768 9.1 to 13 and 19 to 18.
    const int sms = cfi_sm_count();
    const int w = pairs <= sms ? (positions <= (2 * pairs > sms ? 1536 : 768) ? 8 : 0) : positions <= 768 ? 4 : 0;
    a.whole = w > 0;
    const int variant = (c->head_dim == 128) * 2 + (c->type == 8);
    if (w == 8)
        return variant == 0   ? launch<64, false, 8>(a, pairs, most_units, s)
               : variant == 1 ? launch<64, true, 8>(a, pairs, most_units, s)
               : variant == 2 ? launch<128, false, 8>(a, pairs, most_units, s)
                              : launch<128, true, 8>(a, pairs, most_units, s);
    return variant == 0   ? launch<64, false, PA_WARPS>(a, pairs, most_units, s)
           : variant == 1 ? launch<64, true, PA_WARPS>(a, pairs, most_units, s)
           : variant == 2 ? launch<128, false, PA_WARPS>(a, pairs, most_units, s)
                          : launch<128, true, PA_WARPS>(a, pairs, most_units, s);
}
