// k_sample.cu -- one token per row of logits: temperature, top-k, top-p, min-p and a given uniform
// number (include/cfi_serve.h gives the definition).
//
// A cluster of CTAs takes a row.  The logits are read once, by bulk copies: each CTA keeps its slice in
// shared memory, the later passes walk it there and meet through distributed shared memory.  Everything
// that is summed is a whole number (a weight is exp(z - max) in units of 2^-40), so no sum depends on its order
// and every CTA of a cluster reaches the same decisions from the same histograms.
//
// All three filters keep a run from the top of the order (larger z first, then lower index).  Where that run
// is short -- it is, when a top-k or a nucleus of a language model's logits is asked for -- the bins of a
// histogram of max - z say down to which depth it can reach, the few elements above that depth are gathered in
// the cluster's first CTA, and that CTA finishes alone with them in registers.  The gathering needs no exact z: bins
// of (max logit - logit) / T are 1/64 wide, far above the rounding of z, and one bin more is taken.
//
// Each filter is a cut, the last element that stays, found
// without sorting, in one CTA or in the whole cluster (more than SA_CAP elements): a histogram over 512 bins finds the bin that the cut falls in; the at most SA_LIST
// elements of that bin are listed and each one's rank is counted against the others.  A fuller bin is divided
// again: first by the next bits of max - z, then by the bits of z itself, after which all that is left is
// equal and the index decides.
#include "../../include/cfi_serve.h"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <stdlib.h>
#include <string.h>
#include <type_traits>

namespace {

using namespace sm100;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = SA_THREADS;   // a thread holds a bin's total
constexpr int SA_LIST = 128;          // boundary-bin elements that are listed
constexpr int SA_CAP = 2048, SA_EACH = SA_CAP / SA_THREADS;  // elements that the first CTA sorts, and a thread's of them
constexpr int SA_CTAS = 8;            // of a cluster: the portable size, two CTAs to an SM at a vocabulary of 150,000
constexpr int SA_MAX_SLICE = 50000;   // floats of a row that one CTA holds
constexpr int SA_AHEAD = 8;           // loads of a pass that are in flight together

struct SaArgs {
    const float* logits;
    long long stride;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t* top_k;
    int32_t* token;
    float* logprob;
    int n_vocab, slice;
    unsigned int* err;
};

struct SaItem {
    uint32_t key;
    int idx;
    unsigned long long w;
};
static_assert((((SA_MAX_SLICE + 6) / 4 / SA_THREADS + 1) | 1) <= 32, "a thread's groups of four are a mask of 128 bits");

struct SaShared {
    uint32_t cnt[2][SA_BINS];
    unsigned long long wt[2][SA_BINS];
    SaItem list[2][SA_LIST];   // the boundary bin's elements: this CTA's, and all
    uint32_t cand[SA_CAP];     // a short run's elements: their indexes, rising
    uint64_t bar;
    unsigned long long scan[SA_WARPS];
    unsigned long long cta_sum, kept_sum;
    float wmax[SA_WARPS];
    float cta_max;
    int n_list, n_own, n_ties, abort;
    int found_bin;
    unsigned long long found_before;
    uint32_t found_n, cut_key;
    int cut_idx;
};

// The same variable of CTA `rank` of the cluster.
template <class T> CFI_DEV const T* peer(const T* p, uint32_t rank) {
    uint64_t out;
    asm volatile("mapa.u64 %0, %1, %2;" : "=l"(out) : "l"(reinterpret_cast<uint64_t>(p)), "r"(rank));
    return reinterpret_cast<const T*>(out);
}

// Larger z, larger key (z is never -0 here).
CFI_DEV uint32_t key_of(float z) {
    const uint32_t b = __float_as_uint(z);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
CFI_DEV float z_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
constexpr double SA_UNIT = 1099511627776.0;  // 2^40
// exp(z - max) in units of 2^-40: 24 bits of expf, scaled without rounding, cut to whole units
CFI_DEV float exp_of(float z, float zmax) { return z == zmax ? 1.0f : expf(z - zmax); }
CFI_DEV unsigned long long weight_of(float e) { return (unsigned long long)(e * (float)SA_UNIT); }
// max - z in units of 2^-22, 27 bits: a weight is zero from 27.8 on
CFI_DEV uint32_t depth_of(float z, float zmax) { return z == zmax ? 0u : (uint32_t)fminf((zmax - z) * 4194304.0f, 134217727.0f); }

CFI_DEV unsigned long long warp_incl(unsigned long long v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long n = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += n;
    }
    return v;
}

// One digit of the order, most significant first: stages 0-2 the depth, 3-6 the key (larger first).
struct SaPrefix {
    int stage = 0;
    uint32_t depth = 0, key = 0;
    CFI_DEV bool digit(uint32_t d, uint32_t k, uint32_t* bin) const {
        k = ~k;
        if (stage < 3) {
            if (stage > 0 && (d >> (27 - 9 * stage)) != depth) return false;
            *bin = (d >> (18 - 9 * stage)) & 511u;
            return true;
        }
        if (d != depth) return false;
        const int sh = stage == 3 ? 23 : stage == 4 ? 14 : 5;
        if (stage > 3 && (k >> (stage == 4 ? 23 : stage == 5 ? 14 : 5)) != key) return false;
        *bin = stage == 6 ? k & 31u : (k >> sh) & 511u;
        return true;
    }
    CFI_DEV void take(uint32_t bin) {
        if (stage < 3)
            depth = depth << 9 | bin;
        else
            key = stage == 6 ? key << 5 | bin : key << 9 | bin;
        stage++;
    }
    // stage 7 holds one key; a prefix holds an element when it is one of those left to decide on
    CFI_DEV bool holds(uint32_t d, uint32_t k) const {
        k = ~k;
        if (stage <= 3) return (d >> (27 - 9 * stage)) == depth;
        return d == depth && (k >> (stage == 4 ? 23 : stage == 5 ? 14 : stage == 6 ? 5 : 0)) == key;
    }
};

// Inclusive sum over the block's threads, and the whole sum.  Ends with every thread past its reads of `scan`.
CFI_DEV unsigned long long block_incl(unsigned long long v, unsigned long long* scan, unsigned long long* total) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    unsigned long long incl = warp_incl(v, lane);
    if (lane == 31) scan[warp] = incl;
    __syncthreads();
    unsigned long long prev = 0, all = 0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; w++) {
        const unsigned long long x = scan[w];
        if (w < warp) prev += x;
        all += x;
    }
    __syncthreads();
    *total = all;
    return incl + prev;
}

__global__ void __launch_bounds__(SA_THREADS, 2) sample_rows(const SaArgs a) {
    extern __shared__ __align__(16) float slice[];
    __shared__ SaShared s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const int row = blockIdx.x / SA_CTAS;
    const int base = rank * a.slice, n = max(0, min(a.slice, a.n_vocab - base));
    if (tid == 0) {
        mbar_init(&s.bar, 1);
        s.abort = 0;
        fence_mbar_init();
    }
    for (int b = tid; b < SA_BINS; b += SA_THREADS) {
        s.cnt[0][b] = 0;
        s.wt[0][b] = 0;
    }
    __syncthreads();
    pdl_launch_dependents();
    pdl_wait();

    // ---- the one read of the row: 16-byte pieces by bulk copies, the ragged ends by loads ----
    const float* src = a.logits + row * a.stride + base;
    const int shift = (int)(reinterpret_cast<uintptr_t>(src) >> 2 & 3), head = min(n, (4 - shift) & 3), body = (n - head) & ~3;
    float* z = slice + shift;  // logit i of the slice is z[i], 16-byte aligned where it is in memory
    // the slice in groups of four: what lies before and behind it in the first and the last never counts
    const int groups = (shift + n + 3) / 4;
    const float4* z4 = reinterpret_cast<const float4*>(slice);
    if (tid >= 64 && tid < 64 + shift) slice[tid - 64] = -INFINITY;
    if (tid >= 96 && tid < 96 + 4 * groups - shift - n) z[n + tid - 96] = -INFINITY;
    if (tid == 0 && body > 0) {
        mbar_arrive_expect_tx(&s.bar, (uint32_t)body * 4);
        for (int i = 0; i < body; i += 8192)
            bulk_g2s(z + head + i, src + head + i, (uint32_t)min(8192, body - i) * 4, &s.bar);
    }
    if (tid < head) z[tid] = src[tid];
    if (tid >= 32 && tid < 32 + n - head - body) z[head + body + tid - 32] = src[head + body + tid - 32];
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = t <= 0.0f;
    const float div = greedy ? 1.0f : t;
    int k = a.top_k ? a.top_k[row] : 0;
    if (greedy) k = 1;
    if (k >= a.n_vocab) k = 0;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float minp = a.min_p ? a.min_p[row] : 0.0f;
    if (body > 0 && !mbar_wait(&s.bar, 0, &s.abort)) {
        cfi_set_error(a.err, 0xfc100);
        s.abort = 1;
    }
    __syncthreads();

    // element i's z: never -0, and -inf for a NaN
    auto scaled = [&](float l) {
        const float v = (div == 1.0f ? l : l / div) + 0.0f;
        return v == v ? v : -INFINITY;
    };
    const int run = ((n + SA_THREADS - 1) / SA_THREADS) | 1;  // each thread's run: odd, so that 32 of them meet no bank twice
    const int r0 = min(n, tid * run), r1 = min(n, r0 + run);
    // f(i, z[i]) for this thread's run, SA_AHEAD loads at a time
    auto walk = [&](auto&& f) {
        int i = r0;
        for (; i + SA_AHEAD <= r1; i += SA_AHEAD) {
            float v[SA_AHEAD];
#pragma unroll
            for (int e = 0; e < SA_AHEAD; e++) v[e] = z[i + e];
#pragma unroll
            for (int e = 0; e < SA_AHEAD; e++) f(i + e, v[e]);
        }
        for (; i < r1; i++) f(i, z[i]);
    };
    // f(g, z4[g]) for groups of four: g0, g0 + step, ... below g1
    auto by_four = [&](int g0, int g1, int step, auto&& f) {
        int g = g0;
        for (; g + 3 * step < g1; g += 4 * step) {
            float4 v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = z4[g + e * step];
#pragma unroll
            for (int e = 0; e < 4; e++) f(g + e * step, v[e]);
        }
        for (; g < g1; g += step) f(g, z4[g]);
    };
    auto max4 = [](const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); };  // a NaN is passed over
    float mx = -INFINITY;
    by_four(tid, groups, SA_THREADS, [&](int, const float4& v) { mx = fmaxf(mx, max4(v)); });
    mx = warp_max(mx);
    if (lane == 0) s.wmax[warp] = mx;
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(lane < SA_WARPS ? s.wmax[lane] : -INFINITY);
        if (lane == 0) s.cta_max = mx;
    }
    cluster_sync();
    float lmax = lane < SA_CTAS ? *peer(&s.cta_max, lane) : -INFINITY;
    lmax = warp_max(lmax);
    const float zmax = scaled(lmax);  // division by a positive number keeps the order
    const bool empty = zmax == -INFINITY;

    // ---- no top-k: every weight counts.  Each thread sums its run; with a top-p, the top of the order by bins ----
    unsigned long long run_sum = 0, whole = 0;
    const float near = 1.0f / div;
    const bool bins_hold = fabsf(zmax) < 8192.0f && near < 1e30f;  // z is exact to far less than a bin
    if (!empty && k <= 0 && bins_hold) {
        const bool binned = p < 1.0f;
        const float floor = lmax - 28.0f * div * 1.0001f;  // no weight at or below this
        auto weigh = [&](float v) {  // zmax is finite: expf(0) is 1
            const unsigned long long w = weight_of(expf(v - zmax));
            run_sum += w;
            const float d = (zmax - v) * 64.0f;
            if (binned && d < (float)SA_BINS) {
                atomicAdd(&s.cnt[0][(int)d], 1u);
                atomicAdd(&s.wt[0][(int)d], w);
            }
        };
        if (div == 1.0f)
            walk([&](int, float l) {
                if (l > floor) weigh(l + 0.0f);
            });
        else
            walk([&](int, float l) {
                if (l > floor) weigh(l / div + 0.0f);
            });
        unsigned long long sum;
        block_incl(run_sum, s.scan, &sum);
        if (tid == 0) s.cta_sum = sum;
        cluster_sync();
#pragma unroll
        for (uint32_t r = 0; r < SA_CTAS; r++) whole += *peer(&s.cta_sum, r);
    }
    uint32_t level = 1;  // histogram 0 has been used
    // ---- a short run: down to which depth? ----
    float floor = INFINITY;  // gather what is larger
    if (!empty && bins_hold && (k > 0 || p < 1.0f)) {
        // bins down to a depth of 8, or 16 where more than a few are asked for; the second turn reaches 32, where no
        // weight is left
        float scale = k > 8 ? 32.0f : 64.0f;
        for (int turn = 0;; turn++) {
            const uint32_t b = turn & 1;
            if (k > 0) {
                if (turn > 0) {
                    s.cnt[b][tid] = 0;
                    __syncthreads();
                }
                const float unit = near * scale, floor = lmax - (float)SA_BINS / unit * 1.0001f;
                by_four(tid, groups, SA_THREADS, [&](int, const float4& v) {
                    if (!(max4(v) > floor)) return;
                    const float l[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float d = (lmax - l[e]) * unit;  // a NaN compares false
                        if (d < (float)SA_BINS) atomicAdd(&s.cnt[b][(int)d], 1u);
                    }
                });
                cluster_sync();
            }
            uint32_t c = 0;
            unsigned long long m = 0;
#pragma unroll
            for (uint32_t r = 0; r < SA_CTAS; r++) {
                c += *peer(&s.cnt[b][tid], r);
                if (k <= 0) m += *peer(&s.wt[b][tid], r);
            }
            // the first bin whose end lies past the run's; with the next one, and one more for the rounding
            unsigned long long all, ignore;
            const unsigned long long upto = block_incl(c, s.scan, &all);
            if (tid == 0) s.found_bin = SA_BINS;
            __syncthreads();
            if (k > 0) {
                if (upto >= (unsigned long long)k && upto - c < (unsigned long long)k) s.found_bin = tid;
            } else {
                const unsigned long long w = block_incl(m, s.scan, &ignore);
                const double limit = (double)p * (double)whole;
                if (!((double)w < limit) && (double)(w - m) < limit) s.found_bin = tid;
            }
            __syncthreads();
            const int bin = s.found_bin;
            if (bin + 2 < SA_BINS) {
                if (tid == bin + 2) s.found_n = (uint32_t)upto;
                __syncthreads();
                if (s.found_n <= SA_CAP) floor = lmax - (float)(bin + 2) / scale * div * 1.00001f;
                __syncthreads();
                break;
            }
            __syncthreads();
            if (k <= 0 || turn == 1) {
                // fewer than k elements have any weight: all of them are gathered
                if (k > 0 && bin == SA_BINS && all <= SA_CAP) floor = lmax - (float)SA_BINS / scale * div * 1.00001f;
                break;
            }
            scale = 16.0f;
            level = 2;
        }
    }

    // ---- cuts.  What stays: key > cut_key, or key == cut_key and index <= cut_idx ----
    uint32_t cut_key = 0;
    int cut_idx = -1;
    auto kept = [&](uint32_t key, int idx) { return key > cut_key || (key == cut_key && idx <= cut_idx); };
    // Lowers the cut to the last element with less than `limit` before it: a count, or a share of the weight.
    // `each` calls its argument with z and index of this thread's elements, threads and elements in index order.
    // ALONE: the elements are this CTA's, at most `count`; else the whole cluster's.
    auto select = [&](auto alone, auto&& each, int count, bool by_weight, double limit, unsigned long long all_weight) {
        constexpr bool ALONE = decltype(alone)::value;
        constexpr uint32_t PEERS = ALONE ? 1 : SA_CTAS;
        auto meet = [] {
            if (ALONE) __syncthreads(); else cluster_sync();
        };
        auto of = [](auto* v, uint32_t r) { return ALONE ? (const std::remove_pointer_t<decltype(v)>*)v : peer(v, r); };
        SaPrefix pre;
        unsigned long long before = 0;
        uint32_t in_bin = (uint32_t)count;
        if (by_weight && all_weight > 0) limit *= (double)all_weight;
        bool scaled_limit = !by_weight || all_weight > 0;
        for (;;) {
            if (!ALONE || in_bin > SA_LIST) {
                const uint32_t b = level++ & 1;
                s.cnt[b][tid] = 0;
                s.wt[b][tid] = 0;
                if (tid == 0) s.found_bin = -1;
                __syncthreads();
                each([&](float v, int idx) {
                    const uint32_t key = key_of(v);
                    uint32_t bin;
                    if (!kept(key, idx) || !pre.digit(depth_of(v, zmax), key, &bin)) return;
                    const unsigned long long w = weight_of(exp_of(v, zmax));
                    if (w == 0) return;
                    atomicAdd(&s.cnt[b][bin], 1u);
                    if (by_weight) atomicAdd(&s.wt[b][bin], w);
                });
                meet();
                uint32_t c = 0;
                unsigned long long m = 0;
#pragma unroll
                for (uint32_t r = 0; r < PEERS; r++) {
                    c += *of(&s.cnt[b][tid], r);
                    if (by_weight) m += *of(&s.wt[b][tid], r);
                }
                if (!by_weight) m = c;
                unsigned long long total;
                const unsigned long long incl = block_incl(m, s.scan, &total) + before;
                if (pre.stage == 0) {
                    if (!scaled_limit) limit *= (double)total;
                    if (!by_weight && total <= (unsigned long long)limit) return;  // nothing to cut
                    if (!(limit > 0.0)) limit = 0.5;                               // the largest always stays
                }
                // the bin of the cut: the last that has less than the limit before it (a later one has weight)
                if (m > 0 && (double)(incl - m) < limit) atomicMax(&s.found_bin, tid);
                __syncthreads();
                if (tid == s.found_bin) {
                    s.found_before = incl - m;
                    s.found_n = c;
                }
                __syncthreads();
                pre.take((uint32_t)s.found_bin);
                before = s.found_before;
                in_bin = s.found_n;
            } else if (pre.stage == 0) {
                if (!(limit > 0.0)) limit = 0.5;
            }
            if (in_bin <= SA_LIST) {
                if (tid == 0) s.n_list = 0;
                __syncthreads();
                each([&](float v, int idx) {
                    const uint32_t key = key_of(v);
                    if (!kept(key, idx) || !pre.holds(depth_of(v, zmax), key)) return;
                    const unsigned long long w = weight_of(exp_of(v, zmax));
                    if (w != 0) s.list[0][atomicAdd(&s.n_list, 1)] = SaItem{key, idx, by_weight ? w : 1ull};
                });
                meet();
                int n_all = 0;
#pragma unroll
                for (uint32_t r = 0; r < PEERS; r++) {
                    const int nr = *of(&s.n_list, r);
                    for (int e = tid; e < nr; e += SA_THREADS) s.list[1][n_all + e] = *of(&s.list[0][e], r);
                    n_all += nr;
                }
                __syncthreads();
                // four threads rank an element: what is before it, and whether one is behind it
                const int e = tid / 4;
                const bool have = e < n_all;
                unsigned long long mine = 0;
                int behind = 0;
                SaItem me = {};
                if (have) {
                    me = s.list[1][e];
                    for (int j = tid & 3; j < n_all; j += 4) {
                        const SaItem o = s.list[1][j];
                        if (o.key > me.key || (o.key == me.key && o.idx < me.idx)) mine += o.w;
                        if (o.key < me.key || (o.key == me.key && o.idx > me.idx)) behind = 1;
                    }
                }
#pragma unroll
                for (int x = 1; x < 4; x <<= 1) {
                    mine += __shfl_xor_sync(0xffffffffu, mine, x);
                    behind |= __shfl_xor_sync(0xffffffffu, behind, x);
                }
                mine += before;
                // the last that stays: the one behind it has the limit before it, or there is none
                if (have && (double)mine < limit && (!behind || !((double)(mine + me.w) < limit))) {
                    s.cut_key = me.key;
                    s.cut_idx = me.idx;
                }
                __syncthreads();
                cut_key = s.cut_key;
                cut_idx = s.cut_idx;
                return;
            }
            if (pre.stage == 7) {  // equal elements: each has the same weight, the index decides
                const uint32_t eq = ~pre.key;
                unsigned long long mine = 0, ties;
                each([&](float v, int idx) { mine += (unsigned long long)(key_of(v) == eq && kept(eq, idx)); });
                unsigned long long ahead = block_incl(mine, s.scan, &ties) - mine;
                if (tid == 0) s.n_ties = (int)ties;
                meet();
#pragma unroll
                for (uint32_t r = 0; r < PEERS; r++)
                    if (!ALONE && r < rank) ahead += (unsigned long long)*of(&s.n_ties, r);
                // how many of them stay: before + i * w < limit for the i-th
                const unsigned long long w = by_weight ? weight_of(exp_of(z_of(eq), zmax)) : 1ull;
                uint32_t lo = 0, hi = in_bin - 1;  // the last i that stays
                while (lo < hi) {
                    const uint32_t mid = (lo + hi + 1) / 2;
                    if ((double)(before + (unsigned long long)mid * w) < limit)
                        lo = mid;
                    else
                        hi = mid - 1;
                }
                if (lo >= ahead && lo < ahead + mine)
                    each([&](float v, int idx) {
                        if (key_of(v) != eq || !kept(eq, idx)) return;
                        if (ahead++ == lo)
                            for (uint32_t r = 0; r < PEERS; r++) *const_cast<int*>(of(&s.cut_idx, r)) = idx;
                    });
                meet();
                cut_key = eq;
                cut_idx = s.cut_idx;
                return;
            }
        }
    };
    // The draw: kept weights in index order.  `ahead`: what the CTAs before this one have.
    auto draw = [&](auto&& each, unsigned long long own, unsigned long long ahead, unsigned long long total) {
        const double ud = (double)a.u[row] * (double)total;
        unsigned long long target = ud > 0.0 ? (unsigned long long)ud : 0ull;
        if (target >= total) target = total - 1;  // u outside [0, 1)
        if (target < ahead || target >= ahead + own) return;
        each([&](float v, int idx) {
            if (!kept(key_of(v), idx)) return;
            const float e = exp_of(v, zmax);
            if (v != zmax && e < minp) return;
            const unsigned long long w = weight_of(e);
            if (ahead <= target && ahead + w > target) {
                a.token[row] = idx;
                if (a.logprob) a.logprob[row] = (v == zmax ? 0.0f : v - zmax) - logf((float)((double)total / SA_UNIT));
            }
            ahead += w;
        });
    };
    auto weight_of_kept = [&](auto&& each) {
        unsigned long long sum = 0;
        each([&](float v, int idx) {
            if (!kept(key_of(v), idx)) return;
            const float e = exp_of(v, zmax);
            if (v == zmax || !(e < minp)) sum += weight_of(e);
        });
        return sum;
    };

    int nc = SA_CAP + 1;
    if (floor < INFINITY) {
        // ---- a short run: gathered in index order by the first CTA, which goes on alone ----
        const int q = ((groups + SA_THREADS - 1) / SA_THREADS) | 1;  // odd: eight threads' groups take every bank once
        const int g0 = min(groups, tid * q), g1 = min(groups, g0 + q);
        unsigned long long hit[2] = {0, 0};
        by_four(g0, g1, 1, [&](int g, const float4& v) {
            if (!(max4(v) > floor)) return;
            const unsigned long long bits = (v.x > floor) | (v.y > floor) << 1 | (v.z > floor) << 2 | (v.w > floor) << 3;
            if (g - g0 < 16) hit[0] |= bits << 4 * (g - g0); else hit[1] |= bits << 4 * (g - g0 - 16);
        });
        const int mine = __popcll(hit[0]) + __popcll(hit[1]);
        unsigned long long own;
        int at = (int)block_incl((unsigned long long)mine, s.scan, &own) - mine;
        if (tid == 0) s.n_own = (int)own;
        cluster_sync();
        nc = 0;
#pragma unroll
        for (uint32_t r = 0; r < SA_CTAS; r++) {
            const int x = *peer(&s.n_own, r);
            if (r < rank) at += x;
            nc += x;
        }
        if (nc <= SA_CAP) {  // as counted, but for what rounding brings in at the edge
            uint32_t* to = const_cast<uint32_t*>(peer(&s.cand[0], 0));
#pragma unroll
            for (int x = 0; x < 2; x++)
                for (unsigned long long h = hit[x]; h; h &= h - 1)
                    to[at++] = (uint32_t)(base + 4 * g0 - shift + 64 * x + __ffsll((long long)h) - 1);
        }
    }
    if (nc <= SA_CAP) {
        cluster_sync();
        if (rank != 0) return;
        float v[SA_EACH];
        int idx[SA_EACH];
        const int each_n = (nc + SA_THREADS - 1) / SA_THREADS;  // a thread's elements, in index order
#pragma unroll
        for (int e = 0; e < SA_EACH; e++) {
            const int x = tid * each_n + e;
            idx[e] = e < each_n && x < nc ? (int)s.cand[x] : -1;
            v[e] = idx[e] >= 0 ? scaled(a.logits[row * a.stride + idx[e]]) : -INFINITY;
        }
        auto each = [&](auto&& f) {
#pragma unroll
            for (int e = 0; e < SA_EACH; e++)
                if (idx[e] >= 0) f(v[e], idx[e]);
        };
        if (k > 0 && k < nc) select(std::true_type{}, each, nc, false, (double)k, 0ull);
        if (p < 1.0f) {
            unsigned long long among = whole;
            if (k > 0) {
                unsigned long long sum = 0;
                each([&](float x, int i) {
                    if (kept(key_of(x), i)) sum += weight_of(exp_of(x, zmax));
                });
                block_incl(sum, s.scan, &among);
            }
            select(std::true_type{}, each, nc, true, (double)p, among);
        }
        const unsigned long long sum = weight_of_kept(each);
        unsigned long long total;
        const unsigned long long upto = block_incl(sum, s.scan, &total);
        draw(each, sum, upto - sum, total);
        return;
    }

    // ---- a long run, or no filter: z in place of the logits ----
    for (int i = tid; i < n; i += SA_THREADS) z[i] = scaled(z[i]);
    __syncthreads();
    auto each = [&](auto&& f) { walk([&](int i, float v) { f(v, base + i); }); };
    if (!empty) {
        if (k > 0) select(std::false_type{}, each, a.n_vocab, false, (double)k, 0ull);
        if (p < 1.0f) select(std::false_type{}, each, a.n_vocab, true, (double)p, 0ull);
        if (k > 0 || p < 1.0f || minp > 0.0f || !bins_hold) run_sum = weight_of_kept(each);
    }
    unsigned long long sum;
    const unsigned long long upto = block_incl(run_sum, s.scan, &sum);
    if (tid == 0) s.kept_sum = sum;
    cluster_sync();
    unsigned long long total = 0, ahead = 0;
#pragma unroll
    for (uint32_t r = 0; r < SA_CTAS; r++) {
        const unsigned long long x = *peer(&s.kept_sum, r);
        if (r < rank) ahead += x;
        total += x;
    }
    if (total > 0) {
        draw(each, run_sum, ahead + upto - run_sum, total);
    } else if (rank == 0 && tid == 0) {
        a.token[row] = -1;
        if (a.logprob) a.logprob[row] = -INFINITY;
    }
    cluster_sync();  // no CTA leaves while another may read its shared memory
}

}  // namespace

extern "C" int cfi_sample(const float* logits, long long row_stride, int n_rows, int n_vocab, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
                          float* logprob, void* stream) {
    if (!logits || !u || !token || n_rows < 0 || n_vocab <= 0 || n_vocab > SA_CTAS * SA_MAX_SLICE || row_stride < n_vocab ||
        (((uintptr_t)logits | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)u |
          (uintptr_t)token | (uintptr_t)logprob) &
         3))
        return (int)cudaErrorInvalidValue;
    if (n_rows == 0) return 0;
    if (n_rows > 0x7fffffff / SA_CTAS) return (int)cudaErrorInvalidValue;
    SaArgs a = {logits, row_stride, temperature, top_p, min_p, u, top_k, token, logprob, n_vocab, 0, cfi_device_error_word()};
    a.slice = (int)(((n_vocab + SA_CTAS - 1) / SA_CTAS + 3) / 4 * 4);
    const size_t smem = (size_t)a.slice * 4 + 32;  // a row's slice keeps its place within 16 bytes
    static CfiPerDeviceOnce attr;
    cfi_once_per_device(attr, [] {
        cudaFuncSetAttribute(sample_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, SA_MAX_SLICE * 4 + 64);
    });
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)n_rows * SA_CTAS, 1, 1);
    lc.blockDim = dim3(SA_THREADS, 1, 1);
    lc.dynamicSmemBytes = smem;
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = SA_CTAS;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 1 : 2;
    return (int)cudaLaunchKernelEx(&lc, sample_rows, a);
}
