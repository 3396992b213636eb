// k_sample.cu -- one token per row of logits: temperature, top-k, top-p, min-p and a given uniform
// number (include/cfi_serve.h gives the definition).
//
// The logits are one read of memory; what bounds a call is the chain of passes behind it, each of which needs the
// last one's answer.  Few rows: a cluster of CTAs takes a row, each keeps its slice in shared memory,
// walks it there and meets the others through distributed shared memory (one row of 151936 with a nucleus among the
// first 50: 12.6 us).  Many: a CTA takes a row and streams it from memory, as many rows at once as fit (256 rows, top-k
// 50: 44 us, 3.5 TB/s; greedy: 34 us, 4.6 TB/s; without a filter, two reads and an exponential of everything: 81 us).
// Everything that is summed is a whole number (a weight is exp(z - max) in units of 2^-40), so no sum depends on its
// order and every CTA of a cluster reaches the same decisions from the same histograms.
//
// All three filters keep a run from the top of the order (larger z first, then lower index).  Where that run
// is short -- it is, when a top-k or a nucleus of a language model's logits is asked for -- the bins of a
// histogram of max - z, of the largest of each group of elements or of all, say down to which depth it can reach, the
// few elements above that depth are gathered in one CTA, and that CTA finishes alone with them in registers.  The
// gathering needs no exact z: bins of (max logit - logit) / T are at least 1/64 wide, far above the rounding of z, and
// one bin more is taken.
//
// A long nucleus: the bin that its end falls in is gathered and ranked alone, and the kept weights are summed over the row.
//
// Each filter is a cut, the last element that stays, found without sorting, in one CTA or in the whole cluster
// (more than SA_CAP elements): a histogram over 512 bins finds the bin that the cut falls in; the at most SA_LIST
// elements of that bin are listed and each one's rank is counted against the others.  A fuller bin is divided
// again: first by the next bits of max - z, then by the bits of z itself, after which all that is left is
// equal and the index decides.
#include "../../include/cfi_serve.h"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"
#include "quotient.h"

#include <stdlib.h>
#include <string.h>
#include <algorithm>
#include <type_traits>

namespace {

using namespace sm100;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = SA_THREADS;   // a thread holds a bin's total
constexpr int SA_LIST = 128;          // boundary-bin elements that are listed
constexpr int SA_CAP = 2048, SA_EACH = SA_CAP / SA_THREADS;  // elements that the first CTA sorts, and a thread's of them
constexpr int SA_CTAS = 8;            // of a cluster: the portable size, two CTAs to an SM at a vocabulary of 150,000
constexpr int SA_MAX_SLICE = 50000;   // floats of a row that one CTA holds
constexpr int SA_BLOCK4 = 256;         // float4 of a block: 32 lanes' groups of eight
constexpr int SA_AHEAD = 8;           // loads of a pass that are in flight together

struct SaArgs {
    const float* logits;
    long long stride;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t* top_k;
    int32_t* token;
    float* logprob;
    int n_vocab, slice;
    int n_rows;
    int spare;  // of many rows: how many whole() ones clusters take, 0 for all rows
    unsigned int* err;
};

// A row's parameters as they act
struct SaRow {
    bool greedy;
    float div, p, minp;
    int k;  // 0: no top-k
    CFI_DEV SaRow(const SaArgs& a, int row) {
        const float t = a.temperature ? __ldcg(a.temperature + row) : 1.0f;
        greedy = t <= 0.0f;
        div = greedy ? 1.0f : t;
        k = greedy ? 1 : a.top_k ? __ldcg(a.top_k + row) : 0;
        if (k < 0 || k >= a.n_vocab) k = 0;
        p = a.top_p ? __ldcg(a.top_p + row) : 1.0f;
        minp = a.min_p ? __ldcg(a.min_p + row) : 0.0f;
    }
    // rows that are long work for one CTA: a nucleus of the whole row, and what more than a few are kept of
    CFI_DEV bool whole(int n_vocab) const { return n_vocab > SA_CAP && (k > SA_CAP / 2 || (k == 0 && p < 1.0f)); }
};

struct SaItem {
    uint32_t key;
    int idx;
    unsigned long long w;
};
constexpr int SA_MAX_BLOCKS = (SA_CTAS * SA_MAX_SLICE + 6) / 4 / SA_BLOCK4 + 1;
static_assert(SA_MAX_BLOCKS <= SA_THREADS, "a thread holds a block's sum");
static_assert((((SA_MAX_SLICE + 6) / 4 / SA_THREADS + 1) | 1) <= 32, "a thread's groups of four are a mask of 128 bits");

struct SaShared {
    uint32_t cnt[2][SA_BINS];
    union {
        struct {
            uint32_t wlo[2][SA_BINS], whi[2][SA_BINS];  // sums of weights in two words
        };
        float logit[SA_CAP];  // from sample_row, the logits of cand, until SaHeld has them
    };
    SaItem list[2][SA_LIST];   // the boundary bin's elements: this CTA's, and all
    uint32_t cand[SA_CAP];     // a short run's elements: their indexes, rising
    uint64_t bar;
    unsigned long long scan[SA_WARPS];
    unsigned long long cta_sum, kept_sum;
    float wmax[SA_WARPS];
    float cta_max;
    int n_list, n_own, n_ties, abort;
    int row;
    int found_bin;
    unsigned long long found_before;
    uint32_t found_n, cta_n, cut_key;
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
// The same in two halves of 20 bits, by roundings to zero at 2^23: a conversion to 64 bits takes eight times as long, and a
// thread adds a few thousand halves in 32 bits
CFI_DEV void weight_of(float e, uint32_t* hi, uint32_t* lo) {
    const float h = __fmaf_rz(e, 1048576.0f, 8388608.0f), rest = fmaf(e, 1048576.0f, 8388608.0f - h);
    *hi = __float_as_uint(h) - 0x4b000000u;
    *lo = __float_as_uint(__fmaf_rz(rest, 1048576.0f, 8388608.0f)) - 0x4b000000u;
}
// A sum in two words: what passes the lower one is carried.  An addition of 64 bits in shared memory is a loop that waits
// for every other thread of its bin: 782 of one bin took 28 us, in two words 2.
CFI_DEV void sum_add(uint32_t* lo, uint32_t* hi, unsigned long long w) {
    const uint32_t low = (uint32_t)w, old = atomicAdd(lo, low), high = (uint32_t)(w >> 32) + (old + low < old);
    if (high) atomicAdd(hi, high);
}
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

// Element z of a logit: never -0, and -inf for a NaN
CFI_DEV float scaled_of(float l, float div) {
    const float v = (div == 1.0f ? l : l / div) + 0.0f;
    return v == v ? v : -INFINITY;
}

// The divisor of a row whose largest logit is lmax.  Where its quotient by T passes the largest float, T is below 2^-127 of it and every
// other logit at least 2^-24 of it away, so that only its equals have weight; so they do by the divisor that makes it 2^100.
CFI_DEV float held_div(float lmax, float div) { return isinf(lmax / div) && !isinf(lmax) ? fabsf(lmax) * 0x1p-100f : div; }

// The cut of a row.  What stays: key > cut_key, or key == cut_key and index <= cut_idx.  `each` calls its argument
// with z and index of this thread's elements; of `in_order`, threads and elements are in index order.
struct SaCut {
    SaShared& s;
    const SaArgs& a;
    const int row;
    const uint32_t rank;
    const float zmax, minp;
    uint32_t level = 1;  // the histogram that is used next: 0 is used before the first select
    uint32_t cut_key = 0;
    int cut_idx = -1;

    CFI_DEV bool kept(uint32_t key, int idx) const { return key > cut_key || (key == cut_key && idx <= cut_idx); }
    CFI_DEV unsigned long long weight_kept(float v, int idx) const {
        if (!kept(key_of(v), idx)) return 0;
        const float e = exp_of(v, zmax);
        return v == zmax || !(e < minp) ? weight_of(e) : 0;
    }
    template <class E> CFI_DEV unsigned long long weight_of_kept(E&& each) const {
        unsigned long long sum = 0;
        each([&](float v, int idx) { sum += weight_kept(v, idx); });
        return sum;
    }
    // The uniform number's place among `total` units
    CFI_DEV unsigned long long target_of(unsigned long long total) const {
        const double ud = (double)__ldcg(a.u + row) * (double)total;
        const unsigned long long target = ud > 0.0 ? (unsigned long long)ud : 0ull;
        return target < total ? target : total - 1;  // u outside [0, 1)
    }
    CFI_DEV void drawn(float v, int idx, unsigned long long total) const {
        a.token[row] = idx;
        if (a.logprob) a.logprob[row] = (v == zmax ? 0.0f : v - zmax) - logf((float)((double)total / SA_UNIT));
    }
    // The draw: kept weights in index order.  `own`: this thread's, `ahead`: those of the threads before it.
    template <class E>
    CFI_DEV void draw(E&& in_order, unsigned long long own, unsigned long long ahead, unsigned long long total) const {
        const unsigned long long target = target_of(total);
        if (target < ahead || target >= ahead + own) return;
        in_order([&](float v, int idx) {
            const unsigned long long w = weight_kept(v, idx);
            if (ahead <= target && ahead + w > target) drawn(v, idx, total);
            ahead += w;
        });
    }
    // Lowers the cut to the last element with less than `limit` before it: a count, or a share of the weight;
    // `before`: of what lies above all elements.  ALONE: the elements are this CTA's, at most `count`; else the
    // whole cluster's.
    template <bool ALONE, class E, class O>
    CFI_DEV void select(E&& each, O&& in_order, int count, bool by_weight, double limit, unsigned long long all_weight,
                        unsigned long long before = 0, SaPrefix pre = {}) {
        const int tid = threadIdx.x;
        constexpr uint32_t PEERS = ALONE ? 1 : SA_CTAS;
        auto meet = [] {
            if (ALONE) __syncthreads(); else cluster_sync();
        };
        auto of = [](auto* v, uint32_t r) { return ALONE ? (const std::remove_pointer_t<decltype(v)>*)v : peer(v, r); };
        uint32_t in_bin = (uint32_t)count;
        if (by_weight && all_weight > 0) limit *= (double)all_weight;
        bool scaled_limit = !by_weight || all_weight > 0;
        for (;;) {
            if (!ALONE || in_bin > SA_LIST) {
                const uint32_t b = level++ & 1;
                s.cnt[b][tid] = 0;
                s.wlo[b][tid] = 0;
                s.whi[b][tid] = 0;
                if (tid == 0) s.found_bin = -1;
                __syncthreads();
                each([&](float v, int idx) {
                    const uint32_t key = key_of(v);
                    uint32_t bin;
                    if (!kept(key, idx) || !pre.digit(depth_of(v, zmax), key, &bin)) return;
                    const unsigned long long w = weight_of(exp_of(v, zmax));
                    if (w == 0) return;
                    atomicAdd(&s.cnt[b][bin], 1u);
                    if (by_weight) sum_add(&s.wlo[b][bin], &s.whi[b][bin], w);
                });
                meet();
                uint32_t c = 0;
                unsigned long long m = 0;
#pragma unroll
                for (uint32_t r = 0; r < PEERS; r++) {
                    c += *of(&s.cnt[b][tid], r);
                    if (by_weight) m += (unsigned long long)*of(&s.whi[b][tid], r) << 32 | *of(&s.wlo[b][tid], r);
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
                in_order([&](float v, int idx) { mine += (unsigned long long)(key_of(v) == eq && kept(eq, idx)); });
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
                    in_order([&](float v, int idx) {
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
    }
};

// Elements in the registers of one CTA, a thread's in index order: those whose indexes s.cand holds, rising.
struct SaHeld {
    float v[SA_EACH];
    int idx[SA_EACH];
    // `logits`: theirs in the same order, or null to read them again
    CFI_DEV SaHeld(const SaCut& cut, int nc, const float* logits, float div) {
        const int each_n = (nc + SA_THREADS - 1) / SA_THREADS;
#pragma unroll
        for (int e = 0; e < SA_EACH; e++) {
            const int x = threadIdx.x * each_n + e;
            idx[e] = e < each_n && x < nc ? (int)cut.s.cand[x] : -1;
            v[e] = -INFINITY;
            if (idx[e] >= 0) v[e] = scaled_of(logits ? logits[x] : __ldcg(cut.a.logits + cut.row * cut.a.stride + idx[e]), div);
        }
        if (logits) __syncthreads();  // their place is free
    }
    template <class F> CFI_DEV void operator()(F&& f) const {
#pragma unroll
        for (int e = 0; e < SA_EACH; e++)
            if (idx[e] >= 0) f(v[e], idx[e]);
    }
};

// The cut among those of the nc elements of s.cand that are in(z), which have `before` units above them.
template <class F>
CFI_DEV void rank_edge(SaCut& cut, int nc, const float* logits, float div, double limit, unsigned long long before, int bin,
                       F&& in) {
    SaHeld each(cut, nc, logits, div);
#pragma unroll
    for (int e = 0; e < SA_EACH; e++)
        if (!in(each.v[e])) each.idx[e] = -1;
    // a bin of 1/32 lies in one of the first histogram's
    SaPrefix pre;
    pre.take((uint32_t)bin >> 1);
    cut.select<true>(each, each, nc, true, limit, 1ull, before, pre);
}

// A short run, alone: s.cand holds the indexes of nc elements, rising, with all that can stay among them.  `whole`: the weight
// that a top-p is a share of, 0 where it is that of these elements as the top-k leaves them.
CFI_DEV void finish_short(SaCut& cut, int nc, const float* logits, float div, int k, float p, unsigned long long whole) {
    const SaHeld each(cut, nc, logits, div);
    if (k > 0 && k < nc) cut.select<true>(each, each, nc, false, (double)k, 0ull);
    if (p < 1.0f) {
        unsigned long long among = whole;
        if (among == 0) {
            unsigned long long sum = 0;
            each([&](float x, int i) {
                if (cut.kept(key_of(x), i)) sum += weight_of(exp_of(x, cut.zmax));
            });
            block_incl(sum, cut.s.scan, &among);
        }
        cut.select<true>(each, each, nc, true, (double)p, among);
    }
    const unsigned long long sum = cut.weight_of_kept(each);
    unsigned long long total;
    const unsigned long long upto = block_incl(sum, cut.s.scan, &total);
    cut.draw(each, sum, upto - sum, total);
}

// l / T in three forms.  The last, for ordinary T and l only, gives the same value as the division, without its branch.
struct SaByOne {
    CFI_DEV float operator()(float l) const { return l; }
};
struct SaByDivision {
    float t;
    CFI_DEV float operator()(float l) const { return l / t; }
};
struct SaByReciprocal {
    float t, r;
    CFI_DEV float operator()(float l) const { return quotient_by(l, t, r); }
};

// One row, by a cluster: this CTA has the n logits from `base`.
CFI_DEV void sample_row(const SaArgs& a, SaShared& s, float* slice, uint32_t rank, int row) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int base = rank * a.slice, n = max(0, min(a.slice, a.n_vocab - base));

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
    if (tid < head) z[tid] = __ldcg(src + tid);
    if (tid >= 32 && tid < 32 + n - head - body) z[head + body + tid - 32] = __ldcg(src + head + body + tid - 32);
    const SaRow par(a, row);
    const float p = par.p, minp = par.minp;
    const int k = par.k;
    if (body > 0 && !mbar_wait(&s.bar, 0, &s.abort)) {
        cfi_set_error(a.err, 0xfc100);
        s.abort = 1;
    }
    __syncthreads();

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
    // this thread's groups, in index order; an odd number: eight threads' groups take every bank once
    const int q = ((groups + SA_THREADS - 1) / SA_THREADS) | 1, g0 = min(groups, tid * q), g1 = min(groups, g0 + q);
    float largest = -INFINITY;  // of them
    by_four(g0, g1, 1, [&](int, const float4& v) { largest = fmaxf(largest, max4(v)); });
    float mx = warp_max(largest);
    if (lane == 0) s.wmax[warp] = mx;
    __syncthreads();
    if (warp == 0) {
        mx = warp_max(lane < SA_WARPS ? s.wmax[lane] : -INFINITY);
        if (lane == 0) s.cta_max = mx;
    }
    cluster_sync();
    float lmax = lane < SA_CTAS ? *peer(&s.cta_max, lane) : -INFINITY;
    lmax = warp_max(lmax);
    const float div = held_div(lmax, par.div);
    auto scaled = [&](float l) { return scaled_of(l, div); };
    const float zmax = scaled(lmax);  // division by a positive number keeps the order
    const bool empty = zmax == -INFINITY;

    // ---- a top-p of the whole row: the sum of all weights, and the top of the order by bins ----
    unsigned long long whole = 0;
    const float near = 1.0f / div;
    const bool bins_hold = fabsf(zmax) < 8192.0f && near < 1e30f;  // z is exact to far less than a bin
    if (!empty && k <= 0 && p < 1.0f && bins_hold) {
        const float floor = lmax - 28.0f * div * 1.0001f;  // no weight at or below this
        unsigned long long run_sum = 0;
        auto weigh = [&](float v) {  // zmax is finite: expf(0) is 1
            const unsigned long long w = weight_of(expf(v - zmax));
            run_sum += w;
            const float d = (zmax - v) * 32.0f;
            if (d < (float)SA_BINS) {
                atomicAdd(&s.cnt[0][(int)d], 1u);
                sum_add(&s.wlo[0][(int)d], &s.whi[0][(int)d], w);
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
    // ---- a short run: down to which depth?  What is above is gathered in index order by the first CTA ----
    uint32_t level = 0;  // the next histogram; the first is zero, or has the sums above
    int edge = -1;       // a long run's end: the bin that it lies in
    double limit = 0.0;
    int nc = SA_CAP + 1;
    if (!empty && bins_hold && (k > 0 || p < 1.0f)) {
        // A top-k: bins of the threads' largest first, down to a depth of 8, or 16 where more than a few are asked for: as
        // many elements reach as deep as the k-th of these, and few more where k is a small share of them (one row of
        // 151936, k 50: 13.9 -> 12.6 us; 1000 of 5000 would fail so and take 2 us longer).  Else, or where that is too
        // many or there are fewer, bins of all elements, and then down to 32, where no weight is left.
        const bool small_share = 4LL * k <= SA_CTAS * (a.slice / 4 / (((a.slice / 4 + SA_THREADS - 1) / SA_THREADS) | 1));
#pragma unroll 1
        for (int turn = k > 0 && small_share ? 0 : 1; turn < 3; turn++) {
            const float scale = turn == 2 ? 16.0f : k > 8 || k <= 0 ? 32.0f : 64.0f;
            const uint32_t b = level++ & 1;
            if (k > 0) {
                if (level > 1) {
                    s.cnt[b][tid] = 0;
                    __syncthreads();
                }
                const float unit = near * scale, window = lmax - (float)SA_BINS / unit * 1.0001f;
                auto bin = [&](float l) {
                    const float d = (lmax - l) * unit;  // a NaN compares false
                    if (d < (float)SA_BINS) atomicAdd(&s.cnt[b][(int)d], 1u);
                };
                if (turn == 0) {
                    if (largest > window) bin(largest);
                } else {
                    by_four(g0, g1, 1, [&](int, const float4& v) {
                        if (!(max4(v) > window)) return;
                        bin(v.x);
                        bin(v.y);
                        bin(v.z);
                        bin(v.w);
                    });
                }
                cluster_sync();
            }
            uint32_t c = 0;
            unsigned long long m = 0;
#pragma unroll
            for (uint32_t r = 0; r < SA_CTAS; r++) {
                c += *peer(&s.cnt[b][tid], r);
                if (k <= 0) m += (unsigned long long)*peer(&s.whi[b][tid], r) << 32 | *peer(&s.wlo[b][tid], r);
            }
            // the first bin whose end lies past the run's; with the next one, and one more for the rounding
            unsigned long long all, ignore;
            if (tid == 0) s.found_bin = SA_BINS;
            const unsigned long long upto = block_incl(c, s.scan, &all);
            if (k > 0) {
                if (upto >= (unsigned long long)k && upto - c < (unsigned long long)k) s.found_bin = tid;
            } else {
                const unsigned long long w = block_incl(m, s.scan, &ignore);
                limit = fmax((double)p * (double)whole, 0.5);  // the largest always stays
                if (!((double)w < limit) && (double)(w - m) < limit) {
                    s.found_bin = tid;
                    s.found_before = w - m;
                    s.cta_n = c;
                }
            }
            __syncthreads();
            const int found = s.found_bin;
            float floor = INFINITY, top = INFINITY;  // gather what is larger than the one and not than the other
            if (found + 2 < SA_BINS) {
                if (tid == found + 2) s.found_n = (uint32_t)upto;
                __syncthreads();
                if (turn == 0 || s.found_n <= SA_CAP) {
                    floor = lmax - (float)(found + 2) / scale * div * 1.00001f;
                } else if (k <= 0 && s.cta_n <= SA_CAP * 3 / 4) {
                    edge = found;  // a bin and the rounding on both sides
                    floor = lmax - ((float)found + 1.1f) / scale * div * 1.00001f;
                    if (found > 0) top = lmax - ((float)found - 0.1f) / scale * div * 0.99999f;
                }
            } else if (turn == 2 && found == SA_BINS && all <= SA_CAP) {
                floor = lmax - (float)SA_BINS / scale * div * 1.00001f;  // fewer than k elements have any weight
            }
            __syncthreads();
            if (floor < INFINITY) {
                unsigned long long hit[2] = {0, 0};
                if (largest > floor)
                    by_four(g0, g1, 1, [&](int g, const float4& v) {
                        if (!(max4(v) > floor)) return;
                        auto in = [&](float l) { return (unsigned long long)(l > floor && l <= top); };
                        const unsigned long long bits = in(v.x) | in(v.y) << 1 | in(v.z) << 2 | in(v.w) << 3;
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
                    float* to_logit = const_cast<float*>(peer(&s.logit[0], 0));
#pragma unroll
                    for (int x = 0; x < 2; x++)
                        for (unsigned long long h = hit[x]; h; h &= h - 1) {
                            const int i = 4 * g0 - shift + 64 * x + __ffsll((long long)h) - 1;
                            to_logit[at] = z[i];
                            to[at++] = (uint32_t)(base + i);
                        }
                    break;
                }
                edge = -1;
            }
            if (k <= 0 || (turn == 1 && found + 2 < SA_BINS)) break;  // a long run
        }
    }

    SaCut cut = {s, a, row, rank, zmax, minp, level};
    bool ranked = false;
    if (nc <= SA_CAP) {
        cluster_sync();
        if (edge < 0) {
            if (rank == 0) finish_short(cut, nc, s.logit, div, k, p, whole);
            return;
        }
        if (rank == 0) {
            rank_edge(cut, nc, s.logit, div, limit, s.found_before, edge,
                      [&](float v) { return (int)((zmax - v) * 32.0f) == edge; });
            if (tid == 0) {
                s.cut_key = cut.cut_key;
                s.cut_idx = cut.cut_idx;
            }
        }
        cluster_sync();
        cut.cut_key = *peer(&s.cut_key, 0);
        cut.cut_idx = *peer(&s.cut_idx, 0);
        ranked = true;
    }

    // ---- a long run, or no filter ----
    const bool filter = !empty && !ranked && (k > 0 || p < 1.0f);
    auto each = [&](auto&& f) { walk([&](int i, float v) { f(filter ? v : scaled(v), base + i); }); };
    if (filter) {  // z in place of the logits: many passes
        for (int i = tid; i < n; i += SA_THREADS) z[i] = scaled(z[i]);
        __syncthreads();
        if (k > 0) cut.select<false>(each, each, a.n_vocab, false, (double)k, 0ull);
        if (p < 1.0f) cut.select<false>(each, each, a.n_vocab, true, (double)p, 0ull);
    }
    // the kept weights of this thread's run, without branches: the exponentials of a batch are in flight together
    const float v_cut = cut.cut_key == 0 ? -INFINITY : z_of(cut.cut_key);
    auto sum_of_kept = [&](auto by) {
        uint32_t hi = 0, lo = 0;
        walk([&](int i, float l) {
            float v = by(l) + 0.0f;
            v = v == v ? v : -INFINITY;
            const float e = expf(v == zmax ? 0.0f : v - zmax);
            const bool stays = ((v == zmax) | !(e < minp)) & ((v > v_cut) | ((v == v_cut) & (base + i <= cut.cut_idx)));
            uint32_t h, w;
            weight_of(stays ? e : 0.0f, &h, &w);
            hi += h;
            lo += w;
        });
        return ((unsigned long long)hi << 20) + lo;
    };
    const unsigned long long run_sum = empty ? 0 : filter || div == 1.0f ? sum_of_kept(SaByOne{}) : sum_of_kept(SaByDivision{div});
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
        cut.draw(each, run_sum, ahead + upto - run_sum, total);
    } else if (rank == 0 && tid == 0) {
        a.token[row] = -1;
        if (a.logprob) a.logprob[row] = -INFINITY;
    }
    cluster_sync();  // no CTA leaves while another may read its shared memory
}

// Which is the row with `wanted` whole() ones before it?  -1: none; `count`: how many there are in all, as far as it was
// looked for.
CFI_DEV int whole_row(const SaArgs& a, SaShared& s, int wanted, int* count) {
    const int tid = threadIdx.x;
    if (tid == 0) s.row = -1;
    int before = 0;
    for (int first = 0; first < a.n_rows && before <= max(wanted, a.spare); first += SA_THREADS) {
        const bool mine = first + tid < a.n_rows && SaRow(a, first + tid).whole(a.n_vocab);
        unsigned long long here;
        const int upto = before + (int)block_incl(mine, s.scan, &here);
        if (mine && upto - 1 == wanted) s.row = first + tid;
        before += (int)here;
    }
    __syncthreads();
    *count = before;
    return s.row;
}

// SPARE: behind stream_rows, cluster i takes the i-th of the whole() rows where they are few.
template <bool SPARE> __global__ void __launch_bounds__(SA_THREADS, 2) sample_rows(const SaArgs a) {
    extern __shared__ __align__(16) float slice[];
    __shared__ SaShared s;
    const int tid = threadIdx.x;
    if (tid == 0) {
        mbar_init(&s.bar, 1);
        s.abort = 0;
        fence_mbar_init();
    }
    s.cnt[0][tid] = 0;
    s.wlo[0][tid] = 0;
    s.whi[0][tid] = 0;
    __syncthreads();
    pdl_launch_dependents();
    if (!SPARE) {
        pdl_wait();
        sample_row(a, s, slice, cluster_ctarank(), blockIdx.x / SA_CTAS);
        return;
    }
    // stream_rows lets this kernel start after its own wait: what that waited for is complete, and is read past L1.
    // The end waits for stream_rows itself, so that the next kernel's wait is for both.
    int count;
    const int row = whole_row(a, s, blockIdx.x / SA_CTAS, &count);
    if (row >= 0 && count <= a.spare) sample_row(a, s, slice, cluster_ctarank(), row);
    pdl_wait();
}

// ---- many rows: a CTA takes one ----
// The row is streamed past registers, and of each group of 32 logits the largest is kept.  A block is 1024 logits,
// and a lane's eight float4 of it, 128 logits apart, are its group: no lane waits for another.  The group maxima say
// almost all: the row's maximum; a depth that k elements reach at least, namely k groups' largest; and where the few
// elements above a depth are, so that only their groups are read again.
struct SaStream {
    const float4* z4;  // logit i is element shift + i
    int shift, n, groups, blocks;

    CFI_DEV int index(int b, int j, int lane, int c) const { return 4 * (SA_BLOCK4 * b + 32 * j + lane) + c - shift; }
    // the row's first and last float4 hold what is not the row's: it is not read
    CFI_DEV float4 edge(int g) const {
        float v[4];
        const float* z = reinterpret_cast<const float*>(z4);
#pragma unroll
        for (int c = 0; c < 4; c++) {
            const int i = 4 * g + c;
            v[c] = i >= shift && i < shift + n ? __ldcg(z + i) : -INFINITY;
        }
        return make_float4(v[0], v[1], v[2], v[3]);
    }
    CFI_DEV bool inner(int b) const { return b > 0 && SA_BLOCK4 * (b + 1) < groups; }
    CFI_DEV float4 at(int b, int j, int lane) const {
        const int g = SA_BLOCK4 * b + 32 * j + lane;
        return g > 0 && g < groups - 1 ? __ldcg(z4 + g) : edge(g);
    }
    // four float4 of a lane, in eights
    static CFI_DEV constexpr int step(int e) { return 128 * (e / 4) + e % 4; }
    CFI_DEV void load(int b, int j0, int lane, float (&l)[2][8]) const {
        float4 v[4];
        if (inner(b)) {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = __ldcg(z4 + SA_BLOCK4 * b + 32 * (j0 + j) + lane);
        } else {
#pragma unroll
            for (int j = 0; j < 4; j++) v[j] = at(b, j0 + j, lane);
        }
#pragma unroll
        for (int j = 0; j < 4; j++) {
            l[j / 2][j % 2 * 4] = v[j].x;
            l[j / 2][j % 2 * 4 + 1] = v[j].y;
            l[j / 2][j % 2 * 4 + 2] = v[j].z;
            l[j / 2][j % 2 * 4 + 3] = v[j].w;
        }
    }
    CFI_DEV void load(int b, int lane, float4 (&v)[8]) const {
        if (inner(b)) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = __ldcg(z4 + SA_BLOCK4 * b + 32 * j + lane);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = at(b, j, lane);
        }
    }
};

CFI_DEV float max_of(const float4& v) { return fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)); }  // a NaN is passed over

// One row, by this CTA alone.
CFI_DEV void stream_row(const SaArgs& a, SaShared& s, float* slice, int row) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const SaRow par(a, row);
    if (a.spare > 0 && par.whole(a.n_vocab)) {
        int count;
        whole_row(a, s, 0, &count);
        if (count <= a.spare) return;
    }
    const float p = par.p, minp = par.minp;
    const int k = par.k;
    s.cnt[0][tid] = 0;
    s.cnt[1][tid] = 0;
    s.wlo[0][tid] = 0;
    s.whi[0][tid] = 0;
    const float* src = a.logits + row * a.stride;
    SaStream in;
    in.shift = (int)(reinterpret_cast<uintptr_t>(src) >> 2 & 3);
    in.z4 = reinterpret_cast<const float4*>(src - in.shift);
    in.n = a.n_vocab;
    in.groups = (in.shift + in.n + 3) / 4;
    in.blocks = (in.groups + SA_BLOCK4 - 1) / SA_BLOCK4;
    unsigned long long* part = reinterpret_cast<unsigned long long*>(slice);  // of each block, what is summed or counted
    float* gm = slice + 2 * in.blocks;                                        // of each group, the largest,
    uint32_t* hits = reinterpret_cast<uint32_t*>(gm + 32 * in.blocks);        // and which are gathered

    // ---- the read from memory ----
    float mx = -INFINITY;
    for (int b = warp; b < in.blocks; b += SA_WARPS) {
        float4 v[8];
        in.load(b, lane, v);
        float m = max_of(v[0]);
#pragma unroll
        for (int j = 1; j < 8; j++) m = fmaxf(m, max_of(v[j]));
        m = fmaxf(m, -INFINITY);  // NaN in all of them
        gm[32 * b + lane] = m;
        mx = fmaxf(mx, m);
    }
    mx = warp_max(mx);
    if (lane == 0) s.wmax[warp] = mx;
    __syncthreads();
    const float lmax = warp_max(lane < SA_WARPS ? s.wmax[lane] : -INFINITY);
    const float div = held_div(lmax, par.div), zmax = scaled_of(lmax, div);
    if (zmax == -INFINITY) {
        if (tid == 0) {
            a.token[row] = -1;
            if (a.logprob) a.logprob[row] = -INFINITY;
        }
        return;
    }
    const float near = 1.0f / div;
    const bool bins_hold = fabsf(zmax) < 8192.0f && near < 1e30f;
    const float nothing = bins_hold ? lmax - 28.0f * div * 1.0001f : -INFINITY;  // no weight at or below this
    const bool few = a.n_vocab <= SA_CAP;
    SaCut cut = {s, a, row, 0, zmax, minp};

    // f(divided by, eight logits, first) for this thread's elements of groups that reach above `floor`, the e-th with index
    // first + SaStream::step(e), and g(block) after each block
    const bool ordinary = bins_hold && div > 0x1p-60f && div < 0x1p60f;
    auto walk = [&](float floor, auto&& f, auto&& g) {
        for (int b = warp; b < in.blocks; b += SA_WARPS) {
            if (gm[32 * b + lane] > floor) {
#pragma unroll 1
                for (int j0 = 0; j0 < 8; j0 += 4) {
                    float l[2][8];
                    in.load(b, j0, lane, l);
                    const int first = in.index(b, j0, lane, 0);
                    if (div == 1.0f) {
                        f(SaByOne{}, l[0], first);
                        f(SaByOne{}, l[1], first + 256);
                        continue;
                    }
                    float least_abs = INFINITY;
#pragma unroll
                    for (int e = 0; e < 16; e++) least_abs = fminf(least_abs, fabsf(l[e / 8][e % 8]));
                    if (ordinary && least_abs > 0x1p-60f) {
                        const SaByReciprocal by = {div, near};
                        f(by, l[0], first);
                        f(by, l[1], first + 256);
                    } else {
                        f(SaByDivision{div}, l[0], first);
                        f(SaByDivision{div}, l[1], first + 256);
                    }
                }
            }
            g(b);
        }
    };
    // f(value, index) for this thread's elements that have weight, in no order
    auto each = [&](auto&& f) {
        for (int b = warp; b < in.blocks; b += SA_WARPS)
            if (gm[32 * b + lane] > nothing)
#pragma unroll 1
                for (int j0 = 0; j0 < 8; j0 += 4) {
                    float l[2][8];
                    in.load(b, j0, lane, l);
#pragma unroll
                    for (int e = 0; e < 16; e++)
                        if (l[e / 8][e % 8] > nothing)
                            f(scaled_of(l[e / 8][e % 8], div), in.index(b, j0, lane, 0) + 256 * (e / 8) + SaStream::step(e % 8));
                }
    };
    const int run = (a.n_vocab + SA_THREADS - 1) / SA_THREADS, r0 = min(a.n_vocab, tid * run), r1 = min(a.n_vocab, r0 + run);
    auto in_order = [&](auto&& f) {
        for (int i = r0; i < r1; i++) f(scaled_of(__ldcg(src + i), div), i);
    };
    // The elements above `floor` and up to `top` to s.cand in index order; how many.
    auto gather = [&](float floor, float top) {
        if (tid == 0) s.n_list = 0;
        __syncthreads();
        for (int i = tid; i < 32 * in.blocks; i += SA_THREADS) {
            hits[i] = 0;
            if (gm[i] > floor) {
                const int at = atomicAdd(&s.n_list, 1);
                if (at < SA_CAP) s.cand[at] = (uint32_t)i;
            }
        }
        __syncthreads();
        const int listed = s.n_list;
        if (listed > SA_CAP && top == INFINITY) return SA_CAP + 1;
        auto look = [&](int i) {  // a thread a group: its eight loads are in flight together
            float4 v[8];
            in.load(i >> 5, i & 31, v);
            uint32_t mask = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float l[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
                for (int c = 0; c < 4; c++) mask |= (uint32_t)(l[c] > floor && l[c] <= top) << (4 * j + c);
            }
            hits[i] = mask;
        };
        if (listed <= SA_CAP) {
            for (int x = tid; x < listed; x += SA_THREADS) look((int)s.cand[x]);
        } else {
            for (int i = tid; i < 32 * in.blocks; i += SA_THREADS)
                if (gm[i] > floor) look(i);
        }
        __syncthreads();
        for (int b = warp; b < in.blocks; b += SA_WARPS) {
            const uint32_t count = __reduce_add_sync(0xffffffffu, __popc(hits[32 * b + lane]));
            if (lane == 0) part[b] = count;
        }
        __syncthreads();
        unsigned long long all;
        const unsigned long long mine = tid < in.blocks ? part[tid] : 0, upto = block_incl(mine, s.scan, &all);
        if (tid < in.blocks) part[tid] = upto - mine;
        __syncthreads();
        if (all > SA_CAP) return SA_CAP + 1;
        for (int b = warp; b < in.blocks; b += SA_WARPS) {
            const uint32_t mask = hits[32 * b + lane];
            if (!__any_sync(0xffffffffu, mask)) continue;
            // how many of each eighth lie in the lanes up to this one: eight counts of at most 128 in two words
            uint32_t upto[2], eighths[2];
#pragma unroll
            for (int w = 0; w < 2; w++) {
                uint32_t n = mask >> 16 * w & 0xffffu;  // four masks of four bits, then their counts, a byte each
                n = (n & 0xfu) | (n & 0xf0u) << 4 | (n & 0xf00u) << 8 | (n & 0xf000u) << 12;
                n = (n & 0x05050505u) + (n >> 1 & 0x05050505u);
                n = (n & 0x03030303u) + (n >> 2 & 0x03030303u);
                eighths[w] = n;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const uint32_t x = __shfl_up_sync(0xffffffffu, n, o);
                    if (lane >= o) n += x;
                }
                upto[w] = n;
            }
            int at = (int)part[b];
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const int sh = 8 * (j & 3);
                const int mine = eighths[j >> 2] >> sh & 0xff, incl = upto[j >> 2] >> sh & 0xff;
                int to = at + incl - mine;
                for (uint32_t four = mask >> 4 * j & 15u; four; four &= four - 1)
                    s.cand[to++] = (uint32_t)in.index(b, j, lane, __ffs((int)four) - 1);
                at += (int)(__shfl_sync(0xffffffffu, upto[j >> 2], 31) >> sh & 0xff);
            }
        }
        __syncthreads();
        return (int)all;
    };

    // ---- a short run: all elements that can stay, in s.cand ----
    int nc = SA_CAP + 1;
    bool decided = k == 0 && !(p < 1.0f);  // the cut is known
    float least = nothing;                 // nothing stays at or below this
    if (few && (k > 0 || p < 1.0f)) {
        nc = gather(-INFINITY, INFINITY);
    } else if (bins_hold && k > 0) {
        // bins down to a depth of 8, or 16 where more than a few are asked for; the second turn reaches 32
        for (int turn = 0; turn < 2; turn++) {
            const float unit = near * (turn ? 16.0f : k > 8 ? 32.0f : 64.0f), window = lmax - (float)SA_BINS / unit * 1.0001f;
            if (turn) {
                __syncthreads();
                s.cnt[0][tid] = 0;
                s.cnt[1][tid] = 0;
            }
            if (tid == 0) s.found_bin = SA_BINS;
            __syncthreads();
            auto bin = [&](float l, uint32_t* into) {
                const float d = (lmax - l) * unit;  // a NaN compares false
                if (d < (float)SA_BINS) atomicAdd(into + (int)d, 1u);
            };
            for (int i = tid; i < 32 * in.blocks; i += SA_THREADS)
                if (gm[i] > window) bin(gm[i], s.cnt[0]);
            __syncthreads();
            // the bin in which the k-th largest group maximum lies: the k-th element is no deeper
            const uint32_t g = s.cnt[0][tid];
            unsigned long long all, upto = block_incl(g, s.scan, &all);
            if (upto >= (unsigned long long)k && upto - g < (unsigned long long)k) s.found_bin = tid;
            __syncthreads();
            const int reach = s.found_bin + 2;  // one bin more for the rounding
            if (reach < SA_BINS) {
                nc = gather(lmax - (float)reach / unit * 1.00001f, INFINITY);
                if (nc <= SA_CAP) break;
            }
            // too many, or fewer such groups: the elements themselves are counted
            __syncthreads();
            if (tid == 0) s.found_bin = SA_BINS;
            const float floor = reach + 2 < SA_BINS ? lmax - (float)(reach + 2) / unit * 1.0001f : window;
            for (int b = warp; b < in.blocks; b += SA_WARPS)
                if (gm[32 * b + lane] > floor) {
                    float4 v[8];
                    in.load(b, lane, v);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        if (v[j].x > floor) bin(v[j].x, s.cnt[1]);
                        if (v[j].y > floor) bin(v[j].y, s.cnt[1]);
                        if (v[j].z > floor) bin(v[j].z, s.cnt[1]);
                        if (v[j].w > floor) bin(v[j].w, s.cnt[1]);
                    }
                }
            __syncthreads();
            const uint32_t c = s.cnt[1][tid];
            upto = block_incl(c, s.scan, &all);
            if (upto >= (unsigned long long)k && upto - c < (unsigned long long)k) s.found_bin = tid;
            __syncthreads();
            const int found = s.found_bin;
            if (found + 2 < SA_BINS) {
                nc = gather(lmax - (float)(found + 2) / unit * 1.00001f, INFINITY);
                break;
            }
            if (turn == 1 && all <= SA_CAP) nc = gather(window, INFINITY);  // fewer than k have any weight
        }
    } else if (bins_hold && p < 1.0f) {
        // the whole sum, and the weights by bins of 1/32 down to a depth of 16: what lies deeper is a small share of the
        // largest's weight for each 1e5 elements
        uint32_t hi = 0, lo = 0;
        auto depth_bin = [&](float v) { return (zmax - v) * 32.0f; };
        walk(nothing, [&](auto by, const float (&l)[8], int) {
            float d[8];
            uint32_t h[8], w[8];
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float v = by(l[e]) + 0.0f;
                d[e] = depth_bin(v);
                weight_of(l[e] > nothing ? expf(v - zmax) : 0.0f, &h[e], &w[e]);
                hi += h[e];
                lo += w[e];
            }
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (d[e] < (float)SA_BINS) sum_add(&s.wlo[0][(int)d[e]], &s.whi[0][(int)d[e]], ((unsigned long long)h[e] << 20) + w[e]);
        }, [](int) {});
        if (tid == 0) s.found_bin = SA_BINS;
        unsigned long long whole, ignore;
        block_incl(((unsigned long long)hi << 20) + lo, s.scan, &whole);
        const double limit = fmax((double)p * (double)whole, 0.5);  // the largest always stays
        const unsigned long long m = (unsigned long long)s.whi[0][tid] << 32 | s.wlo[0][tid], w = block_incl(m, s.scan, &ignore);
        if (!((double)w < limit) && (double)(w - m) < limit) {
            s.found_bin = tid;
            s.found_before = w - m;
        }
        __syncthreads();
        const int found = s.found_bin;
        if (found < SA_BINS) {
            // the run's end lies in one bin: only that is ranked, gathered with the rounding on both sides
            const unsigned long long before = s.found_before;
            const float unit = near * 32.0f, floor = lmax - ((float)found + 1.1f) / unit * 1.00001f;
            const int edge = gather(floor, found > 0 ? lmax - ((float)found - 0.1f) / unit * 0.99999f : INFINITY);
            if (edge <= SA_CAP) {
                rank_edge(cut, edge, nullptr, div, limit, before, found, [&](float v) { return (int)depth_bin(v) == found; });
                least = floor;
                decided = true;
            }
        }
    }
    if (nc <= SA_CAP) {
        finish_short(cut, nc, nullptr, div, k, p, 0ull);
        return;
    }

    // ---- a long run, or no filter ----
    if (!decided) {
        if (k > 0) cut.select<true>(each, in_order, a.n_vocab, false, (double)k, 0ull);
        if (p < 1.0f) {
            unsigned long long sum = 0, among;
            each([&](float v, int idx) {
                if (cut.kept(key_of(v), idx)) sum += weight_of(exp_of(v, zmax));
            });
            block_incl(sum, s.scan, &among);
            cut.select<true>(each, in_order, a.n_vocab, true, (double)p, among);
        }
    }
    const float v_cut = cut.cut_key == 0 ? -INFINITY : z_of(cut.cut_key);
    // without branches: all that a warp has in flight is wanted
    auto weigh = [&](auto by, float l, int first, int step, uint32_t* hi, uint32_t* lo) {
        const float v = by(l) + 0.0f, e = expf(v == zmax ? 0.0f : v - zmax);
        const bool stays = (l > least) & ((v == zmax) | !(e < minp)) & ((v > v_cut) | ((v == v_cut) & (step <= cut.cut_idx - first)));
        weight_of(stays ? e : 0.0f, hi, lo);
    };
    uint32_t hi = 0, lo = 0;
    walk(least, [&](auto by, const float (&l)[8], int first) {
#pragma unroll
        for (int e = 0; e < 8; e++) {
            uint32_t h, w;
            weigh(by, l[e], first, SaStream::step(e), &h, &w);
            hi += h;
            lo += w;
        }
    }, [&](int b) {
        const uint32_t h = __reduce_add_sync(0xffffffffu, hi), w = __reduce_add_sync(0xffffffffu, lo);
        if (lane == 0) part[b] = ((unsigned long long)h << 20) + w;
        hi = lo = 0;
    });
    __syncthreads();
    unsigned long long total;
    const unsigned long long mine = tid < in.blocks ? part[tid] : 0, upto = block_incl(mine, s.scan, &total);
    const unsigned long long target = cut.target_of(total);
    if (target >= upto - mine && target < upto) {  // one thread: the block that the number falls in
        s.found_bin = tid;
        s.found_before = upto - mine;
    }
    __syncthreads();
    if (warp != 0) return;
    const int b = s.found_bin;
    unsigned long long ahead = s.found_before;
#pragma unroll 1
    for (int j = 0; j < 8; j++) {
        const float4 v = in.at(b, j, lane);
        const float l[4] = {v.x, v.y, v.z, v.w};
        unsigned long long w[4], own = 0;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            uint32_t h, x;
            weigh(SaByDivision{div}, l[c], in.index(b, j, lane, c), 0, &h, &x);
            own += w[c] = ((unsigned long long)h << 20) + x;
        }
        unsigned long long at = ahead + warp_incl(own, lane) - own;
#pragma unroll
        for (int c = 0; c < 4; c++) {
            if (at <= target && at + w[c] > target) cut.drawn(scaled_of(l[c], div), in.index(b, j, lane, c), total);
            at += w[c];
        }
        ahead = __shfl_sync(0xffffffffu, at, 31);
    }
}

__global__ void __launch_bounds__(SA_THREADS, 2) stream_rows(const SaArgs a) {
    extern __shared__ __align__(16) float slice[];
    __shared__ SaShared s;
    if (a.spare > 0) {
        pdl_wait();
        pdl_launch_dependents();  // sample_rows reads what this one waited for
    } else {
        pdl_launch_dependents();
        pdl_wait();
    }
    stream_row(a, s, slice, blockIdx.x);
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
    SaArgs a = {logits, row_stride, temperature, top_p, min_p, u, top_k, token, logprob, n_vocab, 0, n_rows, 0, cfi_device_error_word()};
    a.slice = (int)(((n_vocab + SA_CTAS - 1) / SA_CTAS + 3) / 4 * 4);
    const int blocks = (n_vocab + 6) / 4 / SA_BLOCK4 + 1;
    static CfiPerDeviceOnce attr;
    cfi_once_per_device(attr, [] {
        cudaFuncSetAttribute(sample_rows<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, SA_MAX_SLICE * 4 + 64);
        cudaFuncSetAttribute(sample_rows<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, SA_MAX_SLICE * 4 + 64);
        cudaFuncSetAttribute(stream_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, SA_MAX_BLOCKS * 264);
    });
    const char* ep = getenv("CFI_PDL");
    const int pdl = ep && strcmp(ep, "0") == 0 ? 0 : 1;
    auto launch = [&](void (*kernel)(SaArgs), int ctas, size_t smem, bool cluster) {
        cudaLaunchConfig_t lc = {};
        lc.gridDim = dim3((unsigned)ctas, 1, 1);
        lc.blockDim = dim3(SA_THREADS, 1, 1);
        lc.dynamicSmemBytes = smem;
        lc.stream = static_cast<cudaStream_t>(stream);
        cudaLaunchAttribute at[2];
        at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        at[0].val.programmaticStreamSerializationAllowed = pdl;
        at[1].id = cudaLaunchAttributeClusterDimension;
        at[1].val.clusterDim.x = SA_CTAS;
        at[1].val.clusterDim.y = 1;
        at[1].val.clusterDim.z = 1;
        lc.attrs = at;
        lc.numAttrs = cluster ? 2 : 1;
        return cudaLaunchKernelEx(&lc, kernel, a);
    };
    // Clusters while all run together: 37 rows of 151936 with all kinds of parameters take 30 us, a CTA a row 43; 74
    // rows 55 and 46, 256 rows 136 and 100; one row of 1500 without a filter 5.2 and 10, 16 with all kinds 20 and 14.  Then
    // rows that are long work for one CTA are left to clusters behind, where these are no more than run together and the
    // rows are long: 256 rows of 151936 152 -> 100 us, of 65536 70 -> 60, of 32000 43 and 43; where no row is such that
    // launch costs 9 us.
    const int at_once = 2 * cfi_sm_count() / SA_CTAS;
    const size_t slice_bytes = (size_t)a.slice * 4 + 32;  // a row's slice keeps its place within 16 bytes
    if (n_rows <= at_once) return (int)launch(sample_rows<false>, n_rows * SA_CTAS, slice_bytes, true);
    a.spare = top_p && n_vocab >= 65536 ? at_once : 0;
    const cudaError_t e = launch(stream_rows, n_rows, (size_t)blocks * 264, false);
    if (e != cudaSuccess || a.spare == 0) return (int)e;
    return (int)launch(sample_rows<true>, at_once * SA_CTAS, slice_bytes, true);
}
