// k_sample.cu -- one token per row of logits: temperature, top-k, top-p, min-p and a given uniform
// number (include/cfi_serve.h gives the definition).
//
// A cluster of CTAs takes a row.  The logits are read once: each CTA keeps its slice of z = logit /
// temperature in shared memory, the later passes walk it there and meet through distributed shared memory.
// Everything that is summed is a whole number (a weight is exp(z - max) in units of 2^-40), so no sum
// depends on its order and every CTA of a cluster reaches the same decisions from the same histograms.
//
// All three filters keep a run from the top of the order (larger z first, then lower index), so each
// is a cut: the last element that stays.  A cut is found without sorting: a histogram over 512 bins of
// max - z finds the bin that the cut falls in; the at most SA_LIST elements of that bin are listed and each
// one's rank is counted against the others.  A fuller bin is divided again: first by the next bits of
// max - z, then by the bits of z itself, after which all that is left is equal and the index decides.
#include "../../include/cfi_serve.h"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <stdlib.h>
#include <string.h>

namespace {

using namespace sm100;

constexpr int SA_THREADS = 512, SA_WARPS = SA_THREADS / 32;
constexpr int SA_BINS = SA_THREADS;   // a thread holds a bin's total
constexpr int SA_LIST = 256;          // boundary-bin elements of one CTA that are listed
constexpr int SA_MAX_CTAS = 8;
constexpr int SA_MAX_SLICE = 50000;   // floats of a row that one CTA holds
constexpr int SA_MAX_VOCAB = SA_MAX_CTAS * SA_MAX_SLICE;

struct SaArgs {
    const float* logits;
    long long stride;
    const float *temperature, *top_p, *min_p, *u;
    const int32_t* top_k;
    int32_t* token;
    float* logprob;
    int n_vocab, slice;
};

struct SaItem {
    uint32_t key;
    int idx;
    unsigned long long w;
};

struct SaShared {
    uint32_t cnt[2][SA_BINS];
    unsigned long long wt[2][SA_BINS];
    SaItem list[2][SA_LIST];
    unsigned long long sums[SA_WARPS];
    uint32_t ties[SA_WARPS];
    unsigned long long scan[SA_WARPS];
    uint32_t scan_n[SA_WARPS];
    float wmax[SA_WARPS];
    float cta_max;
    int n_list[2];
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
// exp(z - max) in units of 2^-40: 24 bits of expf, scaled without rounding, cut to whole units
CFI_DEV float exp_of(float z, float zmax) { return z == zmax ? 1.0f : expf(z - zmax); }
CFI_DEV unsigned long long weight_of(float e) { return (unsigned long long)(e * 1099511627776.0f); }
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

__global__ void __launch_bounds__(SA_THREADS) sample_rows(const SaArgs a) {
    extern __shared__ float z[];
    __shared__ SaShared s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t rank = cluster_ctarank(), ctas = cluster_nctarank();
    const int row = blockIdx.x / ctas;
    const int base = rank * a.slice, n = max(0, min(a.slice, a.n_vocab - base));
    const int chunk = ((n + SA_WARPS - 1) / SA_WARPS + 31) & ~31;  // each warp's run of the slice
    const int w0 = min(n, warp * chunk), w1 = min(n, w0 + chunk);
    pdl_launch_dependents();
    pdl_wait();

    const float t = a.temperature ? a.temperature[row] : 1.0f;
    const bool greedy = t <= 0.0f;
    const float div = greedy ? 1.0f : t;
    int k = a.top_k ? a.top_k[row] : 0;
    if (greedy) k = 1;
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    const float minp = a.min_p ? a.min_p[row] : 0.0f;

    // ---- the one read of the row ----
    const float* src = a.logits + row * a.stride + base;
    float mx = -INFINITY;
    for (int i = w0 + lane; i < w1; i += 32) {
        float v = src[i] / div + 0.0f;
        v = v == v ? v : -INFINITY;
        z[i] = v;
        mx = fmaxf(mx, v);
    }
    mx = warp_max(mx);
    if (lane == 0) s.wmax[warp] = mx;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < SA_WARPS; w++) mx = fmaxf(mx, s.wmax[w]);
        s.cta_max = mx;
    }
    cluster_sync();
    float zmax = -INFINITY;
    for (uint32_t r = 0; r < ctas; r++) zmax = fmaxf(zmax, *peer(&s.cta_max, r));

    // what stays: key > cut_key, or key == cut_key and index <= cut_idx
    uint32_t cut_key = 0;
    int cut_idx = -1;
    uint32_t level = 0, lists = 0;
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
            for (uint32_t r = 0; r < ctas; r++) {
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
                for (uint32_t r = 0; r < ctas; r++) {
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
                    for (uint32_t r = 0; r < ctas; r++) {
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
                        for (uint32_t r = 0; r < ctas && !behind; r++) {
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
                const float zq = __uint_as_float(eq & 0x80000000u ? eq & 0x7fffffffu : ~eq);
                const unsigned long long w = by_weight ? weight_of(exp_of(zq, zmax)) : 1ull;
                uint32_t lo = 0, hi = in_bin - 1;  // the last i that stays
                while (lo < hi) {
                    const uint32_t mid = (lo + hi + 1) / 2;
                    if ((double)(before + (unsigned long long)mid * w) < limit)
                        lo = mid;
                    else
                        hi = mid - 1;
                }
                uint32_t ahead = 0;
                for (uint32_t r = 0; r < ctas; r++)
                    for (int q = 0; q < SA_WARPS; q++)
                        if (r < rank || (r == rank && q < warp)) ahead += *peer(&s.ties[q], r);
                if (lo >= ahead && lo < ahead + mine) {  // the warp that has it
                    for (int i = w0; i < w1; i += 32) {
                        const bool is = i + lane < w1 && key_of(z[i + lane]) == eq && kept(eq, base + i + lane);
                        const uint32_t bal = __ballot_sync(0xffffffffu, is);
                        if (is && ahead + __popc(bal & ((1u << lane) - 1)) == lo)
                            for (uint32_t r = 0; r < ctas; r++) *const_cast<int*>(peer(&s.cut_idx, r)) = base + i + lane;
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

    const bool empty = zmax == -INFINITY;
    if (!empty) {
        if (k > 0 && k < a.n_vocab) select(false, (double)k);
        if (p < 1.0f) select(true, (double)p);
    }
    // ---- the draw: kept weights in index order ----
    auto weight_at = [&](int i) -> unsigned long long {
        const float v = z[i];
        if (!kept(key_of(v), base + i)) return 0ull;
        const float e = exp_of(v, zmax);
        return v == zmax || e >= minp ? weight_of(e) : 0ull;
    };
    unsigned long long sum = 0;
    if (!empty)
        for (int i = w0 + lane; i < w1; i += 32) sum += weight_at(i);
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s.sums[warp] = sum;
    cluster_sync();
    unsigned long long total = 0, ahead = 0;
    for (uint32_t r = 0; r < ctas; r++)
        for (int q = 0; q < SA_WARPS; q++) {
            const unsigned long long x = *peer(&s.sums[q], r);
            if (r < rank || (r == rank && q < warp)) ahead += x;
            total += x;
        }
    if (total == 0) {
        if (rank == 0 && tid == 0) {
            a.token[row] = -1;
            if (a.logprob) a.logprob[row] = -INFINITY;
        }
    } else {
        const double ud = (double)a.u[row] * (double)total;
        unsigned long long target = ud > 0.0 ? (unsigned long long)ud : 0ull;
        if (target >= total) target = total - 1;  // u outside [0, 1)
        if (target >= ahead && target < ahead + sum) {
            for (int i = w0; i < w1; i += 32) {
                const unsigned long long w = i + lane < w1 ? weight_at(i + lane) : 0ull;
                const unsigned long long incl = ahead + warp_incl(w, lane);
                const uint32_t over = __ballot_sync(0xffffffffu, incl > target);
                if (over) {
                    if (lane == __ffs(over) - 1) {
                        a.token[row] = base + i + lane;
                        if (a.logprob) {
                            const float d = z[i + lane] == zmax ? 0.0f : z[i + lane] - zmax;
                            a.logprob[row] = d - logf((float)((double)total / 1099511627776.0));
                        }
                    }
                    break;
                }
                ahead = __shfl_sync(0xffffffffu, incl, 31);
            }
        }
    }
    cluster_sync();  // no CTA leaves while another may read its shared memory
}

}  // namespace

extern "C" int cfi_sample(const float* logits, long long row_stride, int n_rows, int n_vocab, const float* temperature,
                          const int32_t* top_k, const float* top_p, const float* min_p, const float* u, int32_t* token,
                          float* logprob, void* stream) {
    if (!logits || !u || !token || n_rows < 0 || n_vocab <= 0 || n_vocab > SA_MAX_VOCAB || row_stride < n_vocab ||
        (((uintptr_t)logits | (uintptr_t)temperature | (uintptr_t)top_k | (uintptr_t)top_p | (uintptr_t)min_p | (uintptr_t)u |
          (uintptr_t)token | (uintptr_t)logprob) &
         3))
        return (int)cudaErrorInvalidValue;
    if (n_rows == 0) return 0;
    if (n_rows > 0x7fffffff / SA_MAX_CTAS) return (int)cudaErrorInvalidValue;
    SaArgs a = {logits, row_stride, temperature, top_p, min_p, u, top_k, token, logprob, n_vocab, 0};
    unsigned ctas = SA_MAX_CTAS;
    a.slice = (int)(((n_vocab + ctas - 1) / ctas + 3) / 4 * 4);
    const size_t smem = (size_t)a.slice * 4;
    static CfiPerDeviceOnce attr;
    cfi_once_per_device(attr, [] {
        cudaFuncSetAttribute(sample_rows, cudaFuncAttributeMaxDynamicSharedMemorySize, SA_MAX_SLICE * 4 + 64);
    });
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t lc = {};
    lc.gridDim = dim3((unsigned)n_rows * ctas, 1, 1);
    lc.blockDim = dim3(SA_THREADS, 1, 1);
    lc.dynamicSmemBytes = smem;
    lc.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute at[2];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = ctas;
    at[0].val.clusterDim.y = 1;
    at[0].val.clusterDim.z = 1;
    at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[1].val.programmaticStreamSerializationAllowed = 1;
    lc.attrs = at;
    lc.numAttrs = (ep && strcmp(ep, "0") == 0) ? 1 : 2;
    return (int)cudaLaunchKernelEx(&lc, sample_rows, a);
}
