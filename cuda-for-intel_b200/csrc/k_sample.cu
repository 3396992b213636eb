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
// the cluster's first CTA, and that CTA sorts them and finishes alone.  The gathering needs no exact z: bins
// of (max logit - logit) / T are 1/64 wide, far above the rounding of z, and one bin more is taken.
//
// Where it is long (more than SA_CAP elements) each filter is a cut, the last element that stays, found
// without sorting: a histogram over 512 bins finds the bin that the cut falls in; the at most SA_LIST
// elements of that bin are listed and each one's rank is counted against the others.  A fuller bin is divided
// again: first by the next bits of max - z, then by the bits of z itself, after which all that is left is
// equal and the index decides.
#include "../../include/cfi_serve.h"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <algorithm>
#include <stdlib.h>
#include <string.h>

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
static_assert(SA_MAX_SLICE <= 65536, "a slice's indexes take 16 bits");

struct SaShared {
    uint32_t cnt[2][SA_BINS];
    unsigned long long wt[2][SA_BINS];
    SaItem list[2][SA_LIST];   // long runs: the boundary bin's elements
    uint32_t cand[SA_CAP];     // short runs: the gathered elements' indexes
    uint16_t own[SA_CAP];      // this CTA's share of them, from its slice's start
    uint64_t bar;
    unsigned long long scan[SA_WARPS];
    unsigned long long cta_sum, kept_sum;
    uint32_t ties[SA_WARPS];
    float wmax[SA_WARPS];
    float cta_max;
    int n_list[2], n_own, n_cand, base, abort;
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

// The sum of v over the block (ties: a word for each warp).
CFI_DEV int block_count(int v, uint32_t* words) {
    v = __reduce_add_sync(0xffffffffu, v);
    if ((threadIdx.x & 31) == 0) words[threadIdx.x >> 5] = (uint32_t)v;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < SA_WARPS; w++) n += (int)words[w];
    __syncthreads();
    return n;
}

// Sorts n (a power of two, at most SA_CAP) numbers in rising order.
CFI_DEV void block_sort(unsigned long long* v, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < n / 2; t += SA_THREADS) {
                const int i = (t & -j) * 2 + (t & (j - 1));  // j is a power of two
                const unsigned long long x = v[i], y = v[i + j];
                if ((x > y) == ((i & k) == 0)) {
                    v[i] = y;
                    v[i + j] = x;
                }
            }
        }
    __syncthreads();
}
CFI_DEV int power_of_two(int n) { return n <= 2 ? 2 : 1 << (32 - __clz(n - 1)); }

__global__ void __launch_bounds__(SA_THREADS) sample_rows(const SaArgs a) {
    extern __shared__ __align__(16) float slice[];
    __shared__ SaShared s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank();
    const int row = blockIdx.x / SA_CTAS;
    const int base = rank * a.slice, n = max(0, min(a.slice, a.n_vocab - base));
    if (tid == 0) {
        mbar_init(&s.bar, 1);
        s.abort = s.n_own = s.n_cand = 0;
        s.kept_sum = 0;
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
    const int chunk = ((n + SA_WARPS - 1) / SA_WARPS + 31) & ~31;  // each warp's run of the slice
    const int w0 = min(n, warp * chunk), w1 = min(n, w0 + chunk);
    const int run = ((n + SA_THREADS - 1) / SA_THREADS) | 1;  // each thread's run: odd, so that 32 of them meet no bank twice
    const int r0 = min(n, tid * run), r1 = min(n, r0 + run);
    // f(i, z[i]) for this warp's run, or this thread's, SA_AHEAD loads at a time
    auto walk = [&](int i0, int i1, int step, auto&& f) {
        for (int i = i0; i < i1; i += step * SA_AHEAD) {
            float v[SA_AHEAD];
#pragma unroll
            for (int e = 0; e < SA_AHEAD; e++) v[e] = i + step * e < i1 ? z[i + step * e] : -INFINITY;
#pragma unroll
            for (int e = 0; e < SA_AHEAD; e++)
                if (i + step * e < i1) f(i + step * e, v[e]);
        }
    };
    float mx = -INFINITY;
    walk(w0 + lane, w1, 32, [&](int, float v) { mx = fmaxf(mx, v); });  // a NaN is passed over
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

    auto logprob_of = [&](float v, unsigned long long total) {
        return (v == zmax ? 0.0f : v - zmax) - logf((float)((double)total / SA_UNIT));
    };
    auto target_of = [&](unsigned long long total) {
        const double ud = (double)a.u[row] * (double)total;
        const unsigned long long target = ud > 0.0 ? (unsigned long long)ud : 0ull;
        return target < total ? target : total - 1;  // u outside [0, 1)
    };

    // ---- no top-k: every weight counts.  Each thread sums its run; with a top-p, the top of the order by bins ----
    unsigned long long run_sum = 0, whole = 0;
    const float near = 1.0f / div;
    const bool bins_hold = fabsf(zmax) < 8192.0f && near < 1e30f;  // z is exact to far less than a bin
    if (!empty && k <= 0 && bins_hold) {
        const bool binned = p < 1.0f && bins_hold;
        walk(r0, r1, 1, [&](int, float l) {
            if (!((lmax - l) * near < 28.0f)) return;  // no weight (or a NaN)
            const float v = scaled(l);
            const unsigned long long w = weight_of(exp_of(v, zmax));
            run_sum += w;
            const float d = (zmax - v) * 64.0f;
            if (binned && d < (float)SA_BINS) {
                atomicAdd(&s.cnt[0][(int)d], 1u);
                atomicAdd(&s.wt[0][(int)d], w);
            }
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
    float depth = -1.0f;  // gather what lies less deep (in units of z)
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
                walk(w0 + lane, w1, 32, [&](int, float l) {
                    const float d = (lmax - l) * near * scale;  // a NaN compares false
                    if (d < (float)SA_BINS) atomicAdd(&s.cnt[b][(int)d], 1u);
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
                if (s.found_n <= SA_CAP) depth = (float)(bin + 2) / scale;
                __syncthreads();
                break;
            }
            __syncthreads();
            if (k <= 0 || turn == 1) {
                // fewer than k elements have any weight: all of them are gathered
                if (k > 0 && bin == SA_BINS && all <= SA_CAP) depth = (float)SA_BINS / scale;
                break;
            }
            scale = 16.0f;
            level = 2;
        }
    }
    if (depth > 0.0f) {
        // ---- gather, in the first CTA ----
        walk(w0 + lane, w1, 32, [&](int i, float l) {
            if ((lmax - l) * near < depth) s.own[atomicAdd(&s.n_own, 1)] = (uint16_t)i;
        });
        __syncthreads();
        const int mine = s.n_own;
        if (tid == 0 && mine > 0) s.base = atomicAdd(const_cast<int*>(peer(&s.n_cand, 0)), mine);
        __syncthreads();
        uint32_t* to = const_cast<uint32_t*>(peer(&s.cand[0], 0));
        for (int e = tid; e < mine; e += SA_THREADS) to[s.base + e] = (uint32_t)(base + s.own[e]);
        cluster_sync();
        if (rank != 0) return;
        // ---- order: larger z, then lower index.  The slice's place is free for what is sorted ----
        unsigned long long *order = reinterpret_cast<unsigned long long*>(slice), *weight = order + SA_CAP;
        const int nc = s.n_cand, size = power_of_two(nc);
        for (int e = tid; e < size; e += SA_THREADS) {
            unsigned long long v = ~0ull;
            if (e < nc) {
                const uint32_t i = s.cand[e];
                v = (unsigned long long)~key_of(scaled(a.logits[row * a.stride + i])) << 32 | i;
            }
            order[e] = v;
        }
        block_sort(order, size);
        unsigned long long w[SA_EACH], part = 0;
        float e[SA_EACH];
#pragma unroll
        for (int i = 0; i < SA_EACH; i++) {
            const int r = SA_EACH * tid + i;
            w[i] = 0;
            e[i] = 0.0f;
            if (r < nc) {
                e[i] = exp_of(z_of(~(uint32_t)(order[r] >> 32)), zmax);
                w[i] = k > 0 && r >= k ? 0ull : weight_of(e[i]);
                weight[r] = w[i];
            }
            part += w[i];
        }
        unsigned long long among;
        unsigned long long before = block_incl(part, s.scan, &among) - part;
        const double limit = (double)p * (double)(k > 0 ? among : whole);
        int stays = 0;
        unsigned long long upto = 0;  // up to the last of this thread's that stays
#pragma unroll
        for (int i = 0; i < SA_EACH; i++) {
            if (w[i] > 0 && (tid + i == 0 || ((!(p < 1.0f) || (double)before < limit) && !(e[i] < minp)))) {
                stays++;
                upto = before + w[i];
            }
            before += w[i];
        }
        const int kept = block_count(stays, s.ties);
        if (stays > 0 && SA_EACH * tid + stays == kept) s.kept_sum = upto;
        // ---- the draw, in index order: index and rank are sorted again ----
        uint32_t idx[SA_EACH];
        const int size2 = power_of_two(kept);
#pragma unroll
        for (int i = 0; i < SA_EACH; i++) idx[i] = SA_EACH * tid + i < kept ? (uint32_t)order[SA_EACH * tid + i] : ~0u;
        unsigned long long* again = weight + SA_CAP;
#pragma unroll
        for (int i = 0; i < SA_EACH; i++)
            if (SA_EACH * tid + i < size2) again[SA_EACH * tid + i] = (unsigned long long)idx[i] << 32 | (uint32_t)(SA_EACH * tid + i);
        block_sort(again, size2);
        const unsigned long long total = s.kept_sum, target = target_of(total);
        int rk[SA_EACH];
        part = 0;
#pragma unroll
        for (int i = 0; i < SA_EACH; i++) {
            const int r = SA_EACH * tid + i;
            rk[i] = r < kept ? (int)(uint32_t)again[r] : 0;
            w[i] = r < kept ? weight[rk[i]] : 0ull;
            part += w[i];
        }
        unsigned long long ignore;
        before = block_incl(part, s.scan, &ignore) - part;
#pragma unroll
        for (int i = 0; i < SA_EACH; i++) {
            if (w[i] > 0 && before <= target && before + w[i] > target) {
                const unsigned long long x = order[rk[i]];
                a.token[row] = (int)(uint32_t)x;
                if (a.logprob) a.logprob[row] = logprob_of(z_of(~(uint32_t)(x >> 32)), total);
            }
            before += w[i];
        }
        return;
    }

    // ---- a long run, or none: z in place of the logits ----
    for (int i = w0 + lane; i < w1; i += 32) z[i] = scaled(z[i]);
    __syncthreads();

    // what stays: key > cut_key, or key == cut_key and index <= cut_idx
    uint32_t cut_key = 0;
    int cut_idx = -1;
    uint32_t lists = 0;
    auto kept = [&](uint32_t key, int idx) { return key > cut_key || (key == cut_key && idx <= cut_idx); };

    // Lowers the cut to the last element with less than `limit` before it (count or weight).
    auto select = [&](bool by_weight, double limit_in) {
        SaPrefix pre;
        double limit = limit_in;
        unsigned long long before = 0;
        for (;;) {
            const uint32_t b = level++ & 1;
            s.cnt[b][tid] = 0;
            s.wt[b][tid] = 0;
            __syncthreads();
            for (int i = w0 + lane; i < w1; i += 32) {
                const float v = z[i];
                const uint32_t key = key_of(v);
                uint32_t bin;
                if (!kept(key, base + i) || !pre.digit(depth_of(v, zmax), key, &bin)) continue;
                const unsigned long long w = weight_of(exp_of(v, zmax));
                if (w == 0) continue;
                atomicAdd(&s.cnt[b][bin], 1u);
                if (by_weight) atomicAdd(&s.wt[b][bin], w);
            }
            cluster_sync();
            uint32_t c = 0;
            unsigned long long m = 0;
#pragma unroll
            for (uint32_t r = 0; r < SA_CTAS; r++) {
                c += *peer(&s.cnt[b][tid], r);
                if (by_weight) m += *peer(&s.wt[b][tid], r);
            }
            if (!by_weight) m = c;
            unsigned long long incl = warp_incl(m, lane);
            if (lane == 31) s.scan[warp] = incl;
            __syncthreads();
            unsigned long long prev = 0, total = 0;
            for (int w = 0; w < SA_WARPS; w++) {
                const unsigned long long x = s.scan[w];
                if (w < warp) prev += x;
                total += x;
            }
            if (pre.stage == 0) {
                if (by_weight)
                    limit = limit_in * (double)total;
                else if (total <= (unsigned long long)limit_in) {
                    __syncthreads();
                    return;  // nothing to cut
                }
                if (!(limit > 0.0)) limit = 0.5;  // the largest always stays
            }
            incl += prev + before;
            // the bin of the cut: the last that has less than the limit before it (a later one has weight)
            if (tid == 0) s.found_bin = -1;
            __syncthreads();
            if (m > 0 && (double)(incl - m) < limit) atomicMax(&s.found_bin, tid);
            __syncthreads();
            if (tid == s.found_bin) {
                s.found_before = incl - m;
                s.found_n = c;
            }
            __syncthreads();
            const int bin = s.found_bin;
            before = s.found_before;
            const uint32_t in_bin = s.found_n;
            if (bin < 0) return;  // no element has weight: a row of -inf
            pre.take((uint32_t)bin);
            if (in_bin <= SA_LIST) {
                const uint32_t lb = lists++ & 1;
                if (tid == 0) s.n_list[lb] = 0;
                __syncthreads();
                for (int i = w0 + lane; i < w1; i += 32) {
                    const float v = z[i];
                    const uint32_t key = key_of(v);
                    if (!kept(key, base + i) || !pre.holds(depth_of(v, zmax), key)) continue;
                    const unsigned long long w = weight_of(exp_of(v, zmax));
                    if (w == 0) continue;
                    const int at = atomicAdd(&s.n_list[lb], 1);
                    s.list[lb][at] = SaItem{key, base + i, by_weight ? w : 1ull};
                }
                cluster_sync();
                // every CTA ranks every element: thread e's is the e-th of the lists one behind another
                SaItem me = {};
                bool have = false;
                int e = tid;
#pragma unroll
                for (uint32_t r = 0; r < SA_CTAS; r++) {
                    const int nr = *peer(&s.n_list[lb], r);
                    if (!have && e < nr) {
                        me = *peer(&s.list[lb][e], r);
                        have = true;
                    }
                    if (!have) e -= nr;
                }
                if (have) {
                    unsigned long long mine = before;
                    bool last = true;  // no element behind this one stays
#pragma unroll
                    for (uint32_t r = 0; r < SA_CTAS; r++) {
                        const int nr = *peer(&s.n_list[lb], r);
                        const SaItem* l = peer(&s.list[lb][0], r);
                        for (int j = 0; j < nr; j++) {
                            const SaItem o = l[j];
                            if (o.key > me.key || (o.key == me.key && o.idx < me.idx)) mine += o.w;
                        }
                    }
                    last = (double)mine < limit && !((double)(mine + me.w) < limit);
                    // the last of the bin has no other behind it, whatever the limit
                    if ((double)mine < limit && !last) {
                        bool behind = false;
                        for (uint32_t r = 0; r < SA_CTAS && !behind; r++) {
                            const int nr = *peer(&s.n_list[lb], r);
                            const SaItem* l = peer(&s.list[lb][0], r);
                            for (int j = 0; j < nr && !behind; j++) {
                                const SaItem o = l[j];
                                behind = o.key < me.key || (o.key == me.key && o.idx > me.idx);
                            }
                        }
                        last = !behind;
                    }
                    if (last) {
                        s.cut_key = me.key;
                        s.cut_idx = me.idx;
                    }
                }
                __syncthreads();
                cut_key = s.cut_key;
                cut_idx = s.cut_idx;
                __syncthreads();
                return;
            }
            if (pre.stage == 7) {  // equal elements: each has the same weight, the index decides
                const uint32_t eq = ~pre.key;
                uint32_t mine = 0;
                for (int i = w0 + lane; i < w1; i += 32) {
                    const uint32_t key = key_of(z[i]);
                    mine += (uint32_t)(key == eq && kept(key, base + i));
                }
                for (int o = 16; o > 0; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
                if (lane == 0) s.ties[warp] = mine;
                cluster_sync();
                // how many of them stay: before + i * w < limit for the i-th; w from the bin's total
                const unsigned long long w = by_weight ? weight_of(exp_of(z_of(eq), zmax)) : 1ull;
                uint32_t lo = 0, hi = in_bin - 1;  // the last i that stays
                while (lo < hi) {
                    const uint32_t mid = (lo + hi + 1) / 2;
                    if ((double)(before + (unsigned long long)mid * w) < limit)
                        lo = mid;
                    else
                        hi = mid - 1;
                }
                uint32_t ahead = 0;
#pragma unroll
                for (uint32_t r = 0; r < SA_CTAS; r++)
                    for (int q = 0; q < SA_WARPS; q++)
                        if (r < rank || (r == rank && q < warp)) ahead += *peer(&s.ties[q], r);
                if (lo >= ahead && lo < ahead + mine) {  // the warp that has it
                    for (int i = w0; i < w1; i += 32) {
                        const bool is = i + lane < w1 && key_of(z[i + lane]) == eq && kept(eq, base + i + lane);
                        const uint32_t bal = __ballot_sync(0xffffffffu, is);
                        if (is && ahead + __popc(bal & ((1u << lane) - 1)) == lo)
#pragma unroll
                            for (uint32_t r = 0; r < SA_CTAS; r++) *const_cast<int*>(peer(&s.cut_idx, r)) = base + i + lane;
                        ahead += __popc(bal);
                    }
                }
                cluster_sync();
                cut_key = eq;
                cut_idx = s.cut_idx;
                __syncthreads();
                return;
            }
        }
    };

    if (!empty) {
        if (k > 0) select(false, (double)k);
        if (p < 1.0f) select(true, (double)p);
    }
    // ---- the draw: kept weights in index order ----
    auto weight_at = [&](int i) -> unsigned long long {
        const float v = z[i];
        if (!kept(key_of(v), base + i)) return 0ull;
        const float e = exp_of(v, zmax);
        return v == zmax || !(e < minp) ? weight_of(e) : 0ull;
    };
    if (!empty && (k > 0 || p < 1.0f || minp > 0.0f || !bins_hold)) {
        run_sum = 0;
        for (int i = r0; i < r1; i++) run_sum += weight_at(i);
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
    if (total == 0) {
        if (rank == 0 && tid == 0) {
            a.token[row] = -1;
            if (a.logprob) a.logprob[row] = -INFINITY;
        }
    } else {
        const unsigned long long target = target_of(total);
        ahead += upto - run_sum;
        if (target >= ahead && target < ahead + run_sum) {
            for (int i = r0; i < r1; i++) {
                ahead += weight_at(i);
                if (ahead > target) {
                    a.token[row] = base + i;
                    if (a.logprob) a.logprob[row] = logprob_of(z[i], total);
                    break;
                }
            }
        }
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
    // a row's slice keeps its place within 16 bytes; three arrays of SA_CAP numbers take its place later
    const size_t smem = std::max((size_t)a.slice * 4 + 16, (size_t)SA_CAP * 3 * 8);
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
