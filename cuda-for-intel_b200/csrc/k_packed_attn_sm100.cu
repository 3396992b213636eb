// k_packed_attn_sm100.cu -- causal attention of packed sequences (include/cfi_serve.h) on the
// 5th-generation tensor cores: O = softmax(scale Q K') V by blocks of 128 keys, with a running row
// maximum and sum, so that no score leaves the SM.
//
// Rows are (token, head) pairs of one kv head's group: a tile is floor(128 / G) tokens times the G query
// heads that share the kv head, one TMA box in token-major order.  That fills the 128 rows of an MMA
// for any group (126 for 7, 126 for 6, 128 for 4), keeps a tile's tokens close together (few keys past
// the diagonal), and reads K and V once for the whole group.
//
// A CTA of 384 threads has two tiles, A and B, of neighbouring tokens, over the same keys:
//   * warps 0-3 run the softmax of tile A, warps 4-7 that of B, a thread for each row (TMEM lane): the
//     128 scores of a block come from tensor memory into registers, the weights go back over them
//     as f16, the A operand of the product with V.  The rows of O are rescaled only when a row's maximum
//     has grown by more than 2^8 since the last time (weights stay far inside f16);
//   * warp 8 issues the MMAs: O_A += P_A V_j, S_A = Q_A K_j+1', then the same for B, so that the tensor
//     pipe works on one tile while the other is in its softmax;
//   * warp 9 brings Q and the ring of K and V blocks by TMA.  V rows past the sequence's end are zeroed
//     in shared memory (the next sequence's rows are there, and 0 x NaN would reach this one).
// A weight of a key that a row does not see is zero, and zero times a NaN or an infinity is a NaN, in every row of the tile: where
// a warp's first row has one, each row is looked at, and what is not finite is summed again over the keys that it
// sees (repair), by its thread, from memory.
// Where there are few tiles a CTA takes one: A and B are then the same rows over every other block of keys, and are joined at
// the end by their maxima and sums, through shared memory.
//
// Tensor memory: S_A, S_B (128 columns each; P over the first 64), O_A, O_B (D columns each).
//
// Bound by the softmax: a block of a tile takes 16384 exponentials, 1024 cycles of an SM's exponential unit, and with
// the maxima, the fp16 packing and two trips through tensor memory about 2000, half of it beside the other
// tile's; its MMAs take 512 (heads of 64) or 1024.  One document of 16384 tokens, 12/2 heads of 128: 0.82 ms under the
// power cap, 1003 TFLOP/s (0.68 ms in short bursts); sixteen prompts of 1 to 2048 tokens 54.6 us, 579 TFLOP/s (the longest
// tile's 16 blocks and the CTAs behind it); four chunks after 7000 tokens, 14/2 heads of 64, 79.5 us, 551 TFLOP/s.
#include "../../include/cfi_serve.h"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <math.h>
#include <stdlib.h>
#include <string.h>

namespace {

using namespace sm100;

constexpr int KA_MMA_WARP = 8, KA_TMA_WARP = 9, KA_THREADS = 384;
// Registers: 384 threads start with 168 each; the softmax warps take 208 (a row's 128 scores stay in
// them) and the other four give up theirs: 256 x 208 + 128 x 88 = 384 x 168.
constexpr int KA_REGS_SOFTMAX = 208, KA_REGS_OTHER = 88;
constexpr int KA_M = 128, KA_N = 128;       // rows of a tile, keys of a block
constexpr uint32_t KA_TMEM_COLS = 512;
constexpr float KA_RESCALE_LOG2 = 8.0f;
template <int D> constexpr int ka_slots() { return D == 64 ? 8 : 5; }  // K and V blocks in flight
template <int D> constexpr uint32_t ka_tile_bytes() { return KA_M * D * 2; }
template <int D> constexpr size_t ka_smem() { return 1024 + (2 + ka_slots<D>()) * (size_t)ka_tile_bytes<D>() + 256; }

struct KaArgs {
    void* out;
    const int32_t *cu_q, *cu_kv;
    long long out_stride;
    int n_seq, n_q, n_kv, n_kv_head, group, tokens, tiles;  // tokens a tile has, tiles a CTA has
    int out_f16, causal;
    float scale_log2;
    unsigned int* err;
    const uint8_t *q, *k, *v;  // f16, for repair()
    long long q_stride, k_stride, v_stride;
};

CFI_DEV float ex2(float x) {  // 2^x (PTX ex2.approx; -inf -> +0)
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

CFI_DEV float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
// ---- packed pairs of f32 ----
CFI_DEV uint64_t pair_of(float lo, float hi) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
    return r;
}
CFI_DEV float2 of_pair(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
CFI_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
CFI_DEV uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
CFI_DEV bool all_finite(const uint4& v) {
    const float x = fmaf(__uint_as_float(v.x), 0.0f, __uint_as_float(v.y) * 0.0f), y = fmaf(__uint_as_float(v.z), 0.0f, __uint_as_float(v.w) * 0.0f);
    return x + y == 0.0f;
}
CFI_DEV bool all_finite_h2(const uint4& v) {
    const __half2 *h = reinterpret_cast<const __half2*>(&v), zero = __float2half2_rn(0.0f);
    const __half2 x = __hfma2(h[0], zero, __hmul2(h[1], zero)), y = __hfma2(h[2], zero, __hmul2(h[3], zero));
    return __hbeq2(__hadd2(x, y), zero);
}
CFI_DEV bool elect_one() {  // true in one lane of a converged warp
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// The `index`-th pair of tiles (of `span` tokens) in the order in which they are begun.  No long one is left for the end: of
// each 32 sequences that with the most keys first, a sequence's last pair, which sees the most, before the others, and the kv
// heads of a pair together (sixteen prompts of 1 to 2048 tokens, 12/2 heads of 128: 58 us by sequences and heads as they
// come, 53 so, 56 by the pairs' own lengths, which take longer to find; one of 2048, 32/8 heads of 128: 61 and 44).
// Called by a warp; out: the pair's number in its sequence, or -1 where there are fewer pairs, and the sequence's
// first query, queries, first key and keys.
CFI_DEV void find_pair(const KaArgs& a, int span, int index, int* out) {
    const int lane = threadIdx.x & 31;
    if (lane == 0) out[0] = -1;
    __syncwarp();
    for (int base = 0, acc = 0; base < a.n_seq && acc <= index; base += 32) {
        const int s = base + lane;
        int q0 = 0, nq = 0, k0 = 0, nk = 0;
        if (s < a.n_seq) {
            q0 = min(max(a.cu_q[s], 0), a.n_q);
            nq = max(min(a.cu_q[s + 1], a.n_q) - q0, 0);
            k0 = min(max(a.cu_kv[s], 0), a.n_kv);
            nk = max(min(a.cu_kv[s + 1], a.n_kv) - k0, 0);
        }
        const int n = (nq + span - 1) / span;
        int before = acc;
        for (int l = 0; l < min(32, a.n_seq - base); l++) {
            const int other = __shfl_sync(0xffffffffu, nk, l), pairs = __shfl_sync(0xffffffffu, n, l);
            if (other > nk || (other == nk && l < lane)) before += pairs;
        }
        if (index >= before && index < before + n)
            out[0] = n - 1 - (index - before), out[1] = q0, out[2] = nq, out[3] = k0, out[4] = nk;
        acc += (int)__reduce_add_sync(0xffffffffu, n);
    }
    __syncwarp();
}

// One row that is in memory: its pieces of 32 dims that are not finite again, over `keys` keys from k0 on; m and inv as
// the row's sums ended.  Looking for such rows costs 0.4 of 54 us of sixteen prompts and nothing of one; a document of 16384 tokens
// takes 24 ms instead of 0.8 with one dim of V all NaN, 65 with the last key's.
template <int D>
__device__ __noinline__ void repair(const KaArgs& a, int head, int kvh, int token, int k0, int keys, float m, float inv) {
    const uint4* q = reinterpret_cast<const uint4*>(a.q + (token * a.q_stride + (long long)head * D) * 2);
    for (int c = 0; c < D / 32; c++) {
        const long long at = token * a.out_stride + (long long)head * D + 32 * c;
        float none = 0.0f;  // but of a NaN or an infinity a NaN
        for (int i = 0; i < 32; i++)
            none = fmaf(a.out_f16 ? __half2float(static_cast<const __half*>(a.out)[at + i]) : static_cast<const float*>(a.out)[at + i], 0.0f, none);
        if (none == 0.0f) continue;
        float o[32];
#pragma unroll
        for (int i = 0; i < 32; i++) o[i] = 0.0f;
        for (int j = 0; j < keys; j++) {
            const uint4* k = reinterpret_cast<const uint4*>(a.k + ((k0 + j) * a.k_stride + (long long)kvh * D) * 2);
            const uint4* v = reinterpret_cast<const uint4*>(a.v + ((k0 + j) * a.v_stride + (long long)kvh * D + 32 * c) * 2);
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < D / 8; i++) {
                const uint4 x = __ldg(q + i), y = __ldg(k + i);
                const __half2 *xh = reinterpret_cast<const __half2*>(&x), *yh = reinterpret_cast<const __half2*>(&y);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 f = __half22float2(xh[e]), g = __half22float2(yh[e]);
                    s = fmaf(f.x, g.x, fmaf(f.y, g.y, s));
                }
            }
            const float p = __half2float(__float2half_rn(ex2(fmaf(s, a.scale_log2, -m))));
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint4 x = __ldg(v + i);
                const __half2* h = reinterpret_cast<const __half2*>(&x);
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    const float2 f = __half22float2(h[e]);
                    o[8 * i + 2 * e] = fmaf(p, f.x, o[8 * i + 2 * e]);
                    o[8 * i + 2 * e + 1] = fmaf(p, f.y, o[8 * i + 2 * e + 1]);
                }
            }
            if ((j & 63) == 63) {  // nothing makes a number of a NaN
                bool all = true;
#pragma unroll
                for (int i = 0; i < 32; i++) all &= o[i] != o[i];
                if (all) break;
            }
        }
#pragma unroll
        for (int i = 0; i < 32; i++)
            if (a.out_f16)
                static_cast<__half*>(a.out)[at + i] = __float2half_rn(o[i] * inv);
            else
                static_cast<float*>(a.out)[at + i] = o[i] * inv;
    }
}

template <int D>
__global__ void __launch_bounds__(KA_THREADS, 1)
    packed_attn(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                const __grid_constant__ CUtensorMap tv, const __grid_constant__ KaArgs a) {
    constexpr int DB = D / 64;  // 64-value blocks of a row: one 128-byte swizzle atom column each
    constexpr int NS = ka_slots<D>();
    constexpr uint32_t TILE = ka_tile_bytes<D>(), BLK = KA_M * 128;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    uint8_t* sQ = smem;             // tiles A, B
    uint8_t* ring = smem + 2 * TILE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(ring + NS * TILE);
    uint64_t* full = bars;          // [NS] a block's TMA bytes
    uint64_t* empty = bars + NS;    // [NS] the MMAs that read it are done
    uint64_t* s_full = bars + 2 * NS;      // [2] scores of a block (and O up to the block before)
    uint64_t* p_full = bars + 2 * NS + 2;  // [2] its weights (a warp each arrives)
    uint64_t* o_full = bars + 2 * NS + 4;  // [2] O complete
    uint64_t* q_full = bars + 2 * NS + 6;   // [2]
    uint64_t* v_clean = bars + 2 * NS + 8;  // V rows past the end are zeroed
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * NS + 9);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    int* place = reinterpret_cast<int*>(tmem_slot + 2);  // what find_pair found

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, kvh = blockIdx.x % a.n_kv_head;
    pdl_launch_dependents();
    // all that needs no input: it runs beside the end of the kernel before.  The tensor memory too: 384 x 168 registers leave no other
    // CTA a place on this SM, so that one of the kernel behind, which may start from here on, cannot take it first
    if (tid == 0) {
        prefetch_tmap(&tq);
        prefetch_tmap(&tk);
        prefetch_tmap(&tv);
        for (int i = 0; i < NS; i++) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        for (int x = 0; x < 2; x++) {
            mbar_init(&s_full[x], 1);
            mbar_init(&p_full[x], 4);
            mbar_init(&o_full[x], 1);
            mbar_init(&q_full[x], 1);
        }
        mbar_init(v_clean, 1);
        *abort_flag = 0;
        fence_mbar_init();
    }
    if (warp == KA_MMA_WARP) {
        tmem_alloc(tmem_slot, KA_TMEM_COLS);
        tmem_relinquish();
    }
    pdl_wait();  // lengths, q, k and v may come from the kernel before

    // ---- which pair of tiles ----
    const int span = a.tiles * a.tokens;
    if (warp == 0) find_pair(a, span, blockIdx.x / a.n_kv_head, place);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const int pair = place[0], q0 = place[1], nq = place[2], k0 = place[3], nk = place[4];
    if (pair < 0) {
        if (warp == KA_MMA_WARP) tmem_dealloc(0, KA_TMEM_COLS);
        return;
    }
    // keys that token t sees, and blocks that a tile needs (its last token sees the most)
    auto seen = [&](int t) { return a.causal ? max(0, min(nk, t + nk - nq + 1)) : nk; };
    auto first_token = [&](int x) { return pair * span + x * a.tokens; };
    auto blocks = [&](int x) {
        const int t = first_token(x);
        return x < a.tiles && t < nq ? (seen(min(nq, t + a.tokens) - 1) + KA_N - 1) / KA_N : 0;
    };
    const int nb0 = blocks(0), nb1 = blocks(1), nmax = max(nb0, nb1);
    // One tile: both halves of the CTA work on it, the first with every other block of keys, the second with those between
    const bool split = a.tiles == 1;
    const int n0 = split ? (nb0 + 1) / 2 : nb0, n1 = split ? nb0 / 2 : nb1;  // blocks of each half
    const bool cut = nmax * KA_N > nk;  // the last block runs past the sequence

    // all 512 columns: they begin at 0, and the MMAs' operands are constants
    constexpr uint32_t TM = 0;
    auto fail = [&](unsigned code) {
        cfi_set_error(a.err, code);
        *abort_flag = 1;
    };

    if (warp >= KA_MMA_WARP) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(KA_REGS_OTHER));
      if (warp == KA_TMA_WARP) {
        bool ok = true;
        if (lane == 0 && nmax > 0) {
            const uint32_t rows = (uint32_t)(a.tokens * a.group);
            // only for a tile that sees keys: another's warps use the place at once
            auto load_q = [&](int x) {
                mbar_arrive_expect_tx(&q_full[x], DB * rows * 128);
                for (int b = 0; b < DB; b++) tma_load_3d(sQ + x * TILE + b * BLK, &tq, 64 * b, kvh * a.group, q0 + first_token(x), &q_full[x]);
            };
            if (nb0 > 0) load_q(0);
            for (int i = 0; ok && i < 2 * nmax; i++) {
                const int st = i % NS;
                ok = mbar_wait(&empty[st], ((uint32_t)(i / NS) & 1) ^ 1, abort_flag);
                if (!ok) break;
                mbar_arrive_expect_tx(&full[st], TILE);
                for (int b = 0; b < DB; b++)
                    tma_load_3d(ring + st * TILE + b * BLK, (i & 1) ? &tv : &tk, 64 * b, kvh, k0 + (i >> 1) * KA_N, &full[st]);
                if (i == 0 && nb1 > 0) load_q(1);  // behind the first keys: tile A begins with these
            }
            if (!ok) fail(0xfb100);
        }
        ok = __shfl_sync(0xffffffffu, (int)ok, 0);
        if (ok && cut) {
            const int i = 2 * nmax - 1, st = i % NS;
            if (__all_sync(0xffffffffu, mbar_wait(&full[st], (uint32_t)(i / NS) & 1, abort_flag))) {
                const int r0 = nk - (nmax - 1) * KA_N;  // first row past the end
                uint4* v = reinterpret_cast<uint4*>(ring + st * TILE);
                for (int c = lane; c < (KA_N - r0) * 8; c += 32)
                    for (int b = 0; b < DB; b++) v[b * (BLK / 16) + r0 * 8 + c] = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(v_clean);
            } else if (lane == 0) {
                fail(0xfb110);
            }
        }
      } else if (warp == KA_MMA_WARP) {
        if (nmax > 0) {
            const uint32_t id_s = idesc_f16(KA_M, KA_N, 0);
            const uint32_t id_o = idesc_f16(KA_M, D, 0) | (1u << 16);  // B (V) MN-major
            // descriptors of Q and the first slot; an offset of n bytes adds n / 16
            const uint64_t dq = sw128_kmajor_desc(smem_u32(sQ)), dk = sw128_kmajor_desc(smem_u32(ring)),
                           dv = sw128_mnmajor_desc(smem_u32(ring), BLK);
            auto scores = [&](int x, int st, int q) {  // S_x = Q_q K'
#pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    const uint32_t off = (kk >> 2) * BLK + (kk & 3) * 32;
                    mma_f16(TM + x * KA_N, dq + ((q * TILE + off) >> 4), dk + st * (TILE >> 4) + (off >> 4), id_s, kk > 0 ? 1u : 0u);
                }
                mma_commit(&s_full[x]);
            };
            auto values = [&](int x, int st, bool first) {  // O_x += P_x V
#pragma unroll
                for (int kk = 0; kk < KA_N / 16; kk++)
                    mma_f16_ts(TM + 256 + x * D, TM + x * KA_N + kk * 8, dv + st * (TILE >> 4) + kk * (16 * 128 >> 4), id_o,
                              (!first || kk > 0) ? 1u : 0u);
            };
            auto ready = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)) != 0; };
            bool ok = true;
            if (split) {
                ok = ready(&q_full[0], 0);
#pragma unroll
                for (int x = 0; x < 2; x++)
                    if (ok && (x ? n1 : n0) > 0) {
                        ok = ready(&full[2 * x], 0);
                        tc_fence_after();
                        if (ok && elect_one()) {
                            scores(x, 2 * x, 0);
                            mma_commit(&empty[2 * x]);
                        }
                    }
                for (int j = 0; ok && j < n0; j++) {
#pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const int n = x ? n1 : n0, b = 2 * j + x, iv = 2 * b + 1, ik = iv + 3, sv = iv % NS, sk = ik % NS;
                        if (j >= n) continue;
                        ok = ready(&full[sv], (uint32_t)(iv / NS) & 1);
                        if (ok && cut && b == nmax - 1) ok = ready(v_clean, 0);
                        ok = ok && ready(&p_full[x], (uint32_t)j & 1);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            values(x, sv, j == 0);
                            mma_commit(&empty[sv]);
                            if (j == n - 1) mma_commit(&o_full[x]);
                        }
                        if (j + 1 < n) {
                            ok = ready(&full[sk], (uint32_t)(ik / NS) & 1);
                            if (!ok) break;
                            if (elect_one()) {
                                scores(x, sk, 0);
                                mma_commit(&empty[sk]);
                            }
                        }
                    }
                }
            } else {
                ok = ready(&full[0], 0);
#pragma unroll
                for (int x = 0; x < 2; x++)
                    if (ok && (x ? n1 : n0) > 0) {
                        ok = ready(&q_full[x], 0);
                        tc_fence_after();
                        if (ok && elect_one()) scores(x, 0, x);
                    }
                if (ok && elect_one()) mma_commit(&empty[0]);
            }
            for (int j = 0; ok && !split && j < nmax; j++) {
                const int iv = 2 * j + 1, ik = 2 * j + 2, sv = iv % NS, sk = ik % NS;
                ok = ready(&full[sv], (uint32_t)(iv / NS) & 1);
                if (ok && cut && j == nmax - 1) ok = ready(v_clean, 0);
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int n = x ? n1 : n0;
                    if (ok && j < n) {
                        ok = ready(&p_full[x], (uint32_t)j & 1);
                        if (!ok) break;
                        tc_fence_after();
                        if (elect_one()) {
                            values(x, sv, j == 0);
                            if (j == n - 1) mma_commit(&o_full[x]);
                        }
                    }
                    if (x == 1 && elect_one()) mma_commit(&empty[sv]);
                    if (j + 1 < n) {
                        ok = ready(&full[sk], (uint32_t)(ik / NS) & 1);
                        if (!ok) break;
                        if (elect_one()) scores(x, sk, x);
                    }
                    if (x == 1 && j + 1 < nmax && elect_one()) mma_commit(&empty[sk]);
                }
            }
            if (!ok && lane == 0) fail(0xfb200);
        }
      }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(KA_REGS_SOFTMAX));
        // ---- softmax: row r of tile x, or of the one tile ----
        const int x = warp >> 2, r = 32 * (warp & 3) + lane, tile = split ? 0 : x;
        const int t = first_token(tile) + r / a.group, n_blocks = x ? n1 : n0;
        const bool valid = r < a.tokens * a.group && t < nq;
        const int limit = valid ? seen(t) : 0;
        const uint32_t trow = TM + ((uint32_t)(32 * (warp & 3)) << 16);
        const uint32_t ts = trow + x * KA_N, to = trow + 256 + x * D;
        // blocks below this one are seen whole by every row of the tile
        const int n_whole = seen(first_token(tile)) / KA_N;
        float m_used = -INFINITY, l = 0.0f;
        bool ok = true;
        for (int j = 0; j < n_blocks; j++) {
            if (!__all_sync(0xffffffffu, mbar_wait(&s_full[x], (uint32_t)j & 1, abort_flag))) {
                ok = false;
                break;
            }
            tc_fence_after();
            uint32_t sv[4][32];
#pragma unroll
            for (int c = 0; c < 4; c++) tmem_ld32(ts + 32 * c, sv[c]);
            tmem_ld_wait();
            const int block = split ? 2 * j + x : j;
            if (block >= n_whole) {
                const int left = limit - block * KA_N;
#pragma unroll
                for (int c = 0; c < 4; c++)
#pragma unroll
                    for (int i = 0; i < 32; i++)
                        if (32 * c + i >= left) sv[c][i] = 0xff800000u;
            }
            float mx4[4];  // chains that do not wait on one another
#pragma unroll
            for (int e = 0; e < 4; e++) {
                mx4[e] = __uint_as_float(sv[e][0]);
#pragma unroll
                for (int i = 1; i < 31; i += 2) mx4[e] = max3(mx4[e], __uint_as_float(sv[e][i]), __uint_as_float(sv[e][i + 1]));
                mx4[e] = fmaxf(mx4[e], __uint_as_float(sv[e][31]));
            }
            const float mx = fmaxf(max3(mx4[0], mx4[1], mx4[2]), mx4[3]) * a.scale_log2;
            const bool grow = valid && (mx > m_used + KA_RESCALE_LOG2 || (m_used == -INFINITY && mx > -INFINITY));
            if (__any_sync(0xffffffffu, grow)) {
                const float alpha = !grow ? 1.0f : m_used == -INFINITY ? 0.0f : ex2(m_used - mx);
                if (grow) m_used = mx;
                l *= alpha;
                if (j > 0) {  // the product before is complete: its MMAs were committed before these scores
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t v[32];
                        tmem_ld32(to + 32 * c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 32; i++) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                        tmem_st32(to + 32 * c, v);
                    }
                }
            }
            const float sub = m_used == -INFINITY ? 0.0f : m_used;  // nothing seen yet: every score is -inf
            const uint64_t scale2 = pair_of(a.scale_log2, a.scale_log2), sub2 = pair_of(-sub, -sub);
            uint64_t sums[2] = {0, 0};
#pragma unroll
            for (int c = 0; c < 4; c++) {
                uint32_t p[16];
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const float2 z = of_pair(fma2(pair_of(__uint_as_float(sv[c][2 * i]), __uint_as_float(sv[c][2 * i + 1])), scale2, sub2));
                    const float e0 = ex2(z.x), e1 = ex2(z.y);
                    sums[i & 1] = add2(sums[i & 1], pair_of(e0, e1));
                    const __half2 h = __floats2half2_rn(e0, e1);
                    p[i] = *reinterpret_cast<const uint32_t*>(&h);
                }
                tmem_st16(ts + 16 * c, p);
            }
            const float2 both = of_pair(add2(sums[0], sums[1]));
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&p_full[x]);
            l += both.x + both.y;
        }
        if (ok && (n_blocks > 0)) ok = __all_sync(0xffffffffu, mbar_wait(&o_full[x], 0, abort_flag));
        float keep = 1.0f, other = 0.0f;  // what the halves of a split tile count for
        // the second half's values by four, [dims / 4][row of the warp], in Q's place; its maxima and sums in the ring's
        float4* half_o = reinterpret_cast<float4*>(sQ + (warp & 3) * (TILE / 2)) + lane;
        float2* half_ml = reinterpret_cast<float2*>(ring + TILE) + r;
        if (split) {
            // everything that was issued is done before anything is written over it
            if (ok && (x ? n0 : n1) > 0) ok = __all_sync(0xffffffffu, mbar_wait(&o_full[x ^ 1], 0, abort_flag));
            tc_fence_after();
            if (x == 1 && ok) {
                *half_ml = make_float2(m_used, l);
                if (n_blocks > 0)
#pragma unroll
                    for (int c = 0; c < D / 32; c++) {
                        uint32_t v[32];
                        tmem_ld32(to + 32 * c, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int i = 0; i < 8; i++)
                            half_o[(8 * c + i) * 32] = make_float4(__uint_as_float(v[4 * i]), __uint_as_float(v[4 * i + 1]),
                                                                   __uint_as_float(v[4 * i + 2]), __uint_as_float(v[4 * i + 3]));
                    }
            }
            asm volatile("bar.sync 1, 256;" ::: "memory");  // the softmax warps, after a failed wait too
            if (x == 0 && ok) {
                const float2 ml = *half_ml;
                const float m = fmaxf(m_used, ml.x);
                keep = m_used == -INFINITY ? 0.0f : ex2(m_used - m);
                other = ml.x == -INFINITY ? 0.0f : ex2(ml.x - m);
                l = l * keep + ml.y * other;
                m_used = m;
            }
        }
        tc_fence_after();
        if (!ok) {
            if (lane == 0) fail(0xfb300 + warp);
        } else if (!split || x == 0) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            const long long at = valid ? (long long)(q0 + t) * a.out_stride + (long long)(kvh * a.group + r % a.group) * D : -1;
            // The warp's 32 rows go through the shared memory of its rows of Q, which nothing reads any more, so that its stores
            // are of whole rows (sixteen prompts of 100 to 1000 tokens, 12/2 heads of 128: 32.7 us with a lane storing its
            // own row in pieces of 16 bytes, 31.0 so; a prompt of 631 in single tiles 11.7 and 11.8).
            uint8_t* rows = (split ? ring : sQ + x * TILE) + (warp & 3) * (TILE / 4);
            auto put = [&](int chunk, int chunks, uint4 v) {
                *reinterpret_cast<uint4*>(rows + (lane * chunks + (chunk ^ (lane & 7))) * 16) = v;
            };
            bool look = n_blocks > 0 && valid && l == 0.0f;  // zeros say nothing
            auto store = [&](int chunks, int size, int first) {  // pieces of 16 bytes a row, bytes of a value, first value
                __syncwarp();
                if (lane < chunks) {  // the first row's
                    const uint4 v = *reinterpret_cast<const uint4*>(rows + lane * 16);
                    look |= size == 2 ? !all_finite_h2(v) : !all_finite(v);
                }
#pragma unroll 4
                for (int i = lane; i < 32 * chunks; i += 32) {
                    const int row = i / chunks, chunk = i % chunks;
                    const long long to = __shfl_sync(0xffffffffu, at, row);
                    const uint4 v = *reinterpret_cast<const uint4*>(rows + (row * chunks + (chunk ^ (row & 7))) * 16);
                    if (to >= 0) *reinterpret_cast<uint4*>(static_cast<uint8_t*>(a.out) + (to + first) * size + 16 * chunk) = v;
                }
                __syncwarp();
            };
#pragma unroll
            for (int c = 0; c < D / 32; c++) {
                uint32_t v[32];
                if (n_blocks > 0) tmem_ld32(to + 32 * c, v);
                tmem_ld_wait();
                if (split && n1 > 0)
#pragma unroll
                    for (int i = 0; i < 8; i++) {
                        const float4 h = half_o[(8 * c + i) * 32];
                        v[4 * i] = __float_as_uint(fmaf(__uint_as_float(v[4 * i]), keep, h.x * other));
                        v[4 * i + 1] = __float_as_uint(fmaf(__uint_as_float(v[4 * i + 1]), keep, h.y * other));
                        v[4 * i + 2] = __float_as_uint(fmaf(__uint_as_float(v[4 * i + 2]), keep, h.z * other));
                        v[4 * i + 3] = __float_as_uint(fmaf(__uint_as_float(v[4 * i + 3]), keep, h.w * other));
                    }
                if (l == 0.0f)
#pragma unroll
                    for (int i = 0; i < 32; i++) v[i] = 0u;
                if (a.out_f16) {
#pragma unroll
                    for (int i = 0; i < 32; i += 8) {
                        uint32_t w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const __half2 h = __floats2half2_rn(__uint_as_float(v[i + 2 * e]) * inv, __uint_as_float(v[i + 2 * e + 1]) * inv);
                            w[e] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                        put(4 * c + i / 8, D / 8, make_uint4(w[0], w[1], w[2], w[3]));
                    }
                    if (c == D / 32 - 1) store(D / 8, 2, 0);
                } else {  // half a row at a time
                    constexpr int HALF = D / 64;
#pragma unroll
                    for (int i = 0; i < 32; i += 4) {
                        float f[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) f[e] = __uint_as_float(v[i + e]) * inv;
                        put(8 * (c % HALF) + i / 4, D / 8, make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])));
                    }
                    if (c % HALF == HALF - 1) store(D / 8, 4, 32 * (c - HALF + 1));
                }
            }
            // not for a NaN among the scores, which the sum of the weights has too
            if (__any_sync(0xffffffffu, look) && valid && l - l == 0.0f)
                repair<D>(a, kvh * a.group + r % a.group, kvh, q0 + t, k0, limit, m_used, inv);
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == KA_MMA_WARP) {
        tc_fence_after();
        tmem_dealloc(TM, KA_TMEM_COLS);
    }
}

typedef CUresult (*PFN_encodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                    const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                    CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

PFN_encodeTiled encode_fn() {
    static PFN_encodeTiled fn = nullptr;
    static std::once_flag once;
    std::call_once(once, [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<PFN_encodeTiled>(p);
        else
            cudaGetLastError();
    });
    return fn;
}

// [token][head][D] f16 with a token stride, loaded in boxes of 64 values x heads x tokens.
bool map_rows(CUtensorMap* m, const void* p, int d, int heads, long long stride, int n, int box_heads, int box_tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)heads, (cuuint64_t)n};
    const cuuint64_t str[2] = {(cuuint64_t)d * 2, (cuuint64_t)stride * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens}, es[3] = {1, 1, 1};
    return encode_fn()(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(p), dims, str, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D> int launch(const CfiPackedAttention* p, cudaStream_t stream) {
    if (!encode_fn()) return (int)cudaErrorNotSupported;
    KaArgs a;
    a.out = p->out;
    a.cu_q = p->cu_q;
    a.cu_kv = p->cu_kv;
    a.out_stride = p->out_stride;
    a.n_seq = p->n_seq;
    a.n_q = p->n_q;
    a.n_kv = p->n_kv;
    a.n_kv_head = p->n_kv_head;
    a.group = p->n_head / p->n_kv_head;
    a.tokens = KA_M / a.group;
    a.out_f16 = p->out_type;
    a.causal = p->causal;
    a.scale_log2 = p->scale * 1.4426950408889634f;
    a.err = cfi_device_error_word();
    a.q = static_cast<const uint8_t*>(p->q);
    a.k = static_cast<const uint8_t*>(p->k);
    a.v = static_cast<const uint8_t*>(p->v);
    a.q_stride = p->q_stride;
    a.k_stride = p->k_stride;
    a.v_stride = p->v_stride;
    // Every sequence adds at most one pair that is not full.  Up to 5/4 pairs an SM a CTA takes a single tile, which halves the
    // chain of the longest; more share the reads of K and V and the CTAs' beginnings and ends.  Single tiles against
    // pairs, us: one prompt of 1024, 12/2 heads of 128, 15 and 22; of 3000 (145 pairs) 39 and 54; of 4096 (196) 67 and
    // 69; of 5000 (240) 90 and 85; four chunks of 300 to 800 after 7000, 14/2 heads of 64 (134), 81 and 91; eight of 100 to
    // 1000 after 2000 (244) 48 and 48; one of 2048, 32/8 heads of 128 (264), 58 and 43.
    auto pairs = [&](int tiles) { return p->n_q / (tiles * a.tokens) + (p->n_seq < p->n_q ? p->n_seq : p->n_q); };
    a.tiles = 4LL * pairs(2) * p->n_kv_head <= 5LL * cfi_sm_count() ? 1 : 2;
    const long long grid = (long long)pairs(a.tiles) * p->n_kv_head;
    if (grid > 0x7fffffffLL) return (int)cudaErrorInvalidValue;
    CUtensorMap tq, tk, tv;
    // no keys at all: the maps still need an extent, and nothing is loaded
    if (!map_rows(&tq, p->q, D, p->n_head, p->q_stride, p->n_q, a.group, a.tokens) ||
        !map_rows(&tk, p->k, D, p->n_kv_head, p->k_stride, p->n_kv > 0 ? p->n_kv : 1, 1, KA_N) ||
        !map_rows(&tv, p->v, D, p->n_kv_head, p->v_stride, p->n_kv > 0 ? p->n_kv : 1, 1, KA_N))
        return (int)cudaErrorInvalidValue;
    static CfiPerDeviceOnce attr;
    cfi_once_per_device(attr, [] { cudaFuncSetAttribute(packed_attn<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ka_smem<D>()); });
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)grid, 1, 1);
    lc.blockDim = dim3(KA_THREADS, 1, 1);
    lc.dynamicSmemBytes = ka_smem<D>();
    lc.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    return (int)cudaLaunchKernelEx(&lc, packed_attn<D>, tq, tk, tv, a);
}

}  // namespace

extern "C" int cfi_packed_attention(const CfiPackedAttention* a, void* stream) {
    if (!a || !a->q || !a->k || !a->v || !a->out || !a->cu_q || !a->cu_kv || a->n_seq < 0 || a->n_seq > 65535 || a->n_q < 0 ||
        a->n_kv < 0 || a->n_head <= 0 || a->n_kv_head <= 0 || a->n_head % a->n_kv_head || a->n_head / a->n_kv_head > 128 ||
        a->n_head > 65535 || (a->head_dim != 64 && a->head_dim != 128) || (a->out_type != 0 && a->out_type != 1) ||
        !(a->scale > 0.0f) || isinf(a->scale))
        return (int)cudaErrorInvalidValue;
    const long long wq = (long long)a->n_head * a->head_dim, wk = (long long)a->n_kv_head * a->head_dim;
    if ((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->out) & 15) ||
        (((uintptr_t)a->cu_q | (uintptr_t)a->cu_kv) & 3) || (a->q_stride | a->k_stride | a->v_stride | a->out_stride) % 8 ||
        a->q_stride < wq || a->out_stride < wq || a->k_stride < wk || a->v_stride < wk)
        return (int)cudaErrorInvalidValue;
    if (a->n_seq == 0 || a->n_q == 0) return 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return a->head_dim == 64 ? launch<64>(a, s) : launch<128>(a, s);
}
