// k_paged_place.cu -- page tables, slots, positions and packed offsets of a batch made on the device, and pages given back
// (include/cfi_serve.h).  Whole numbers only: what a call writes does not depend on any order.
//
// Every CTA adds up for itself what the sequences hold, get and need (a thread takes some in a row, then one scan over the
// threads), so that no CTA waits for another; the pages, tokens and positions of the lists are then shared out, and each finds its
// sequence by bisection among the sums in shared memory.  The state is changed by the last CTA, when all have read it.
//
// Bound by latency: rows, lengths, table and lists are read one after the other, a memory round trip each.
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <algorithm>
#include <stdlib.h>
#include <string.h>

namespace {

// Elements of a CTA at least, and its threads.  Measured (place and trim of a step of 64, of sixteen prompts, of 1024 sequences with
// 1.9 million positions): 1024, 2048, 4096, 32768 elements 9.4, 9.2, 9.6, 10.4 us; 14.5, 14.7, 14.5, 22.5; 19.3, 19.3, 19.3, 23.7; 256, 512,
// 1024 threads 8.8, 9.2, 12.1; 13.7, 14.7, 18.3; 30.7, 19.3, 23.2.  (With the CTAs counted early: 8.5, 13.8 and 18.0.)
constexpr int PP_SHARE = 2048;
constexpr int PP_THREADS = 512, PP_SEQS = 8192, PP_ROWS = 65536;

struct PpArgs {
    CfiPageTable t;
    CfiPagedPlace p;  // of a trim: rows, n_new (what to keep), n_seq, status
    int page_shift;
    unsigned int* counter;  // CTAs that have read the state; zero between calls
};

// Sums over the threads: those of the threads before this one, and all.
struct Sums {
    long long q, kv;  // new tokens, positions
    int pages, taken;  // that hold them; of those, new ones
};
CFI_DEV Sums operator+(const Sums& a, const Sums& b) { return {a.q + b.q, a.kv + b.kv, a.pages + b.pages, a.taken + b.taken}; }
CFI_DEV Sums scan(Sums x, Sums* total) {
    __shared__ Sums s_warp[PP_THREADS / 32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums y = {__shfl_up_sync(0xffffffffu, incl.q, o), __shfl_up_sync(0xffffffffu, incl.kv, o), __shfl_up_sync(0xffffffffu, incl.pages, o),
                        __shfl_up_sync(0xffffffffu, incl.taken, o)};
        if (lane >= o) incl = incl + y;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    Sums before = {0, 0, 0, 0}, all = {0, 0, 0, 0};
    for (int w = 0; w < PP_THREADS / 32; w++) {
        if (w == warp) before = all;
        all = all + s_warp[w];
    }
    __syncthreads();
    *total = all;
    return {before.q + incl.q - x.q, before.kv + incl.kv - x.kv, before.pages + incl.pages - x.pages, before.taken + incl.taken - x.taken};
}

// Marks row r; true where it was marked before or there is no such row.
CFI_DEV bool bad_row(uint32_t* seen, int r, int n_rows) {
    if ((unsigned)r >= (unsigned)n_rows) return true;
    return atomicOr(&seen[r >> 5], 1u << (r & 31)) >> (r & 31) & 1;
}

// The sequence that element i belongs to: the last whose part of the packed list begins at or before it.
CFI_DEV int sequence_of(const int* cu, int n, int i) {
    int lo = 0, hi = n - 1;  // cu[lo] <= i < cu[hi + 1]
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (cu[mid] <= i) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Thread 0 says that its CTA has read the state; true where all others have: this one may change it.
CFI_DEV bool last_to_read(unsigned int* counter) {
    if (gridDim.x == 1) return true;
    __threadfence();
    const bool last = atomicAdd(counter, 1u) == gridDim.x - 1;
    if (last) *counter = 0u;
    return last;
}

__global__ void __launch_bounds__(PP_THREADS) paged_place(const __grid_constant__ PpArgs a) {
    extern __shared__ int smem[];
    const CfiPageTable& t = a.t;
    const CfiPagedPlace& p = a.p;
    const int n = p.n_seq, tid = threadIdx.x, mask = t.page_size - 1;
    int *cu_q = smem, *cu_kv = cu_q + n + 1, *cu_pages = cu_kv + n + 1, *first = cu_pages + n + 1, *row = first + n;  // first: of the pages taken
    uint32_t* seen = reinterpret_cast<uint32_t*>(row + n);
    __shared__ int s_why, s_last;
    sm100::pdl_launch_dependents();
    for (int i = tid; i < (t.n_rows + 31) / 32; i += PP_THREADS) seen[i] = 0;
    if (tid == 0) s_why = 0x7fffffff;
    sm100::pdl_wait();
    __syncthreads();
    const int each = (n + PP_THREADS - 1) / PP_THREADS, s0 = min(n, tid * each), s1 = min(n, s0 + each);
    const int n_free = min(max(*t.n_free, 0), t.n_pages);
    Sums mine = {0, 0, 0, 0};
    int why = 0x7fffffff;
    for (int s = s0; s < s1; s++) {
        const int r = p.rows[s], add = p.n_new[s];
        cu_q[s] = add;
        row[s] = r;
        if (bad_row(seen, r, t.n_rows) || add < 0) {
            why = min(why, (int)CFI_PLACE_BAD_ROW);
            continue;
        }
        const int held = t.cached[r];
        cu_kv[s] = held;
        const long long after = (long long)held + add;
        if (held < 0) {
            why = min(why, (int)CFI_PLACE_BAD_ROW);
        } else if (after > (long long)t.max_pages << a.page_shift || after > 0x7fffffffLL - mask) {
            why = min(why, (int)CFI_PLACE_TOO_LONG);
        } else {
            const int pages = (int)((after + mask) >> a.page_shift);
            mine = mine + Sums{add, after, pages, pages - ((held + mask) >> a.page_shift)};
        }
    }
    Sums all;
    Sums at = scan(mine, &all);
    if (all.kv > 0x7fffffffLL) why = min(why, (int)CFI_PLACE_TOO_LONG);
    if (all.q > p.max_new || (p.context && all.kv > p.max_context)) why = min(why, (int)CFI_PLACE_NO_ROOM);
    if (all.taken > n_free) why = min(why, (int)CFI_PLACE_NO_PAGES);
    if (why != 0x7fffffff) atomicMin(&s_why, why);
    __syncthreads();
    const bool ok = s_why == 0x7fffffff, writes = blockIdx.x == 0;
    for (int s = s0; s < s1; s++) {
        const int add = ok ? cu_q[s] : 0, held = ok ? cu_kv[s] : 0, pages = (held + add + mask) >> a.page_shift;
        cu_q[s] = ok ? (int)at.q : 0;
        cu_kv[s] = ok ? (int)at.kv : 0;
        cu_pages[s] = at.pages;
        first[s] = at.taken;
        if (writes) {
            p.cu_q[s] = cu_q[s];
            p.cu_kv[s] = cu_kv[s];
            p.lens[s] = held + add;
        }
        at = at + Sums{add, held + add, pages, pages - ((held + mask) >> a.page_shift)};
    }
    if (tid == 0) {
        cu_q[n] = ok ? (int)all.q : 0;
        cu_kv[n] = ok ? (int)all.kv : 0;
        cu_pages[n] = ok ? all.pages : 0;
        if (writes) {
            p.status[0] = ok ? (int)CFI_PLACED : s_why;
            p.cu_q[n] = cu_q[n];
            p.cu_kv[n] = cu_kv[n];
        }
        s_last = ok && last_to_read(a.counter);
    }
    __syncthreads();
    auto held = [&](int s) { return cu_kv[s + 1] - cu_kv[s] - (cu_q[s + 1] - cu_q[s]); };
    // page i of sequence s
    auto page = [&](int s, int i) {
        const int old = (held(s) + mask) >> a.page_shift;
        return i < old ? t.table[(long long)row[s] * t.max_pages + i] : t.free_pages[n_free - 1 - (first[s] + i - old)];
    };
    const int all_pages = cu_pages[n], all_q = cu_q[n], all_kv = cu_kv[n], lane = tid & 31;
    const uint32_t id = blockIdx.x * PP_THREADS + tid, threads = gridDim.x * PP_THREADS;
    for (uint32_t x = id; x < (uint32_t)p.max_new; x += threads) {
        long long slot = -1;
        int pos = 0;
        if (x < (uint32_t)all_q) {
            const int s = sequence_of(cu_q, n, x);
            pos = held(s) + x - cu_q[s];
            slot = ((long long)page(s, pos >> a.page_shift) << a.page_shift) + (pos & mask);
        }
        p.slots[x] = slot;
        p.positions[x] = pos;
    }
    // a page to a lane, 32 in a row to a warp, which then writes their positions together
    for (uint32_t base = id & ~31u; base < (uint32_t)all_pages; base += threads) {
        const uint32_t x = base + lane;
        int to = 0, begin = 0, count = 0;  // the page; where in the context its positions go, and how many
        if (x < (uint32_t)all_pages) {
            const int s = sequence_of(cu_pages, n, x), i = x - cu_pages[s], len = cu_kv[s + 1] - cu_kv[s];
            to = page(s, i);
            begin = cu_kv[s] + (i << a.page_shift);
            count = min(t.page_size, len - (i << a.page_shift));
            p.batch_table[(long long)s * t.max_pages + i] = to;
            if (i >= (held(s) + mask) >> a.page_shift) t.table[(long long)row[s] * t.max_pages + i] = to;
        }
        if (!p.context) continue;
        const int lanes = min(t.page_size, 32), at_once = 32 / lanes;  // of a page; pages
        for (int k = lane / lanes; k < 32; k += at_once) {
            const long long slot = (long long)__shfl_sync(0xffffffffu, to, k) << a.page_shift;
            const int b = __shfl_sync(0xffffffffu, begin, k), c = __shfl_sync(0xffffffffu, count, k);
            for (int j = lane % lanes; j < c; j += lanes) p.context[b + j] = slot + j;
        }
    }
    if (p.context)
        for (uint32_t x = all_kv + id; x < (uint32_t)p.max_context; x += threads) p.context[x] = -1;
    if (!s_last) return;
    for (int s = s0; s < s1; s++) t.cached[row[s]] = cu_kv[s + 1] - cu_kv[s];
    if (tid == 0) *t.n_free = n_free - all.taken;
}

__global__ void __launch_bounds__(PP_THREADS) paged_trim(const __grid_constant__ PpArgs a) {
    extern __shared__ int smem[];
    const CfiPageTable& t = a.t;
    const int n = a.p.n_seq, tid = threadIdx.x, mask = t.page_size - 1;
    const int32_t* keep = a.p.n_new;
    int *first = smem, *from = first + n + 1, *row = from + n, *now = row + n;  // of the pages given back; the first such of a row
    uint32_t* seen = reinterpret_cast<uint32_t*>(now + n);
    __shared__ int s_why, s_last;
    sm100::pdl_launch_dependents();
    for (int i = tid; i < (t.n_rows + 31) / 32; i += PP_THREADS) seen[i] = 0;
    if (tid == 0) s_why = 0x7fffffff;
    sm100::pdl_wait();
    __syncthreads();
    const int each = (n + PP_THREADS - 1) / PP_THREADS, s0 = min(n, tid * each), s1 = min(n, s0 + each);
    const int n_free = min(max(*t.n_free, 0), t.n_pages);
    Sums mine = {0, 0, 0, 0};
    int why = 0x7fffffff;
    for (int s = s0; s < s1; s++) {
        const int r = a.p.rows[s], most = max(keep[s], 0);
        row[s] = r;
        if (bad_row(seen, r, t.n_rows)) {
            why = min(why, (int)CFI_PLACE_BAD_ROW);
            continue;
        }
        const int held = t.cached[r];
        if (held < 0) {
            why = min(why, (int)CFI_PLACE_BAD_ROW);
        } else if (held > (long long)t.max_pages << a.page_shift || held > 0x7fffffff - mask) {
            why = min(why, (int)CFI_PLACE_TOO_LONG);
        } else {
            now[s] = min(held, most);
            first[s] = mine.pages;
            from[s] = (now[s] + mask) >> a.page_shift;
            const int gone = ((held + mask) >> a.page_shift) - from[s];
            mine = mine + Sums{0, gone, gone, 0};
        }
    }
    Sums all;
    const Sums at = scan(mine, &all);
    if (all.kv > t.n_pages - n_free) why = min(why, (int)CFI_PLACE_NO_PAGES);
    if (why != 0x7fffffff) atomicMin(&s_why, why);
    __syncthreads();
    const bool ok = s_why == 0x7fffffff;
    if (tid == 0 && blockIdx.x == 0) a.p.status[0] = ok ? (int)CFI_PLACED : s_why;
    if (!ok) return;
    for (int s = s0; s < s1; s++) first[s] += at.pages;
    if (tid == 0) {
        first[n] = all.pages;
        s_last = last_to_read(a.counter);
    }
    __syncthreads();
    for (uint32_t x = blockIdx.x * PP_THREADS + tid; x < (uint32_t)all.pages; x += gridDim.x * PP_THREADS) {
        const int s = sequence_of(first, n, x);
        t.free_pages[n_free + all.pages - 1 - x] = t.table[(long long)row[s] * t.max_pages + from[s] + x - first[s]];
    }
    if (!s_last) return;
    for (int s = s0; s < s1; s++) t.cached[row[s]] = now[s];
    if (tid == 0) *t.n_free = n_free + all.pages;
}

bool table_ok(const CfiPageTable* t) {
    return t && t->table && t->cached && t->free_pages && t->n_free &&
           !(((uintptr_t)t->table | (uintptr_t)t->cached | (uintptr_t)t->free_pages | (uintptr_t)t->n_free) & 3) && t->n_rows > 0 &&
           t->n_rows <= PP_ROWS && t->max_pages > 0 && t->page_size >= 16 && t->page_size <= 256 && (t->page_size & (t->page_size - 1)) == 0 &&
           t->n_pages > 0;
}
size_t seen_bytes(const CfiPageTable* t) { return (size_t)(t->n_rows + 31) / 32 * 4; }

// `work`: an upper bound of the elements that are read or written.
int go(const void* fn, PpArgs& a, size_t smem, long long work, cudaStream_t stream) {
    const long long ctas = std::min<long long>(cfi_sm_count(), std::max<long long>(1, work / PP_SHARE));
    if (ctas > 1) {
        int err = 0;
        a.counter = static_cast<unsigned int*>(cfi_stream_buffer(CFI_BUF_COUNTERS, 4, stream, &err));
        if (!a.counter) return err;
    }
    a.page_shift = __builtin_ctz((unsigned)a.t.page_size);
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3((unsigned)ctas, 1, 1);
    c.blockDim = dim3(PP_THREADS, 1, 1);
    c.dynamicSmemBytes = smem;
    c.stream = stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = (ep && strcmp(ep, "0") == 0) ? 0 : 1;
    void* args[1] = {&a};
    return (int)cudaLaunchKernelExC(&c, fn, args);
}
constexpr int PP_SMEM = PP_ROWS / 8 + (5 * PP_SEQS + 3) * 4;
void allow_smem() {
    static CfiPerDeviceOnce once;
    cfi_once_per_device(once, [] {
        cudaFuncSetAttribute(paged_place, cudaFuncAttributeMaxDynamicSharedMemorySize, PP_SMEM);
        cudaFuncSetAttribute(paged_trim, cudaFuncAttributeMaxDynamicSharedMemorySize, PP_SMEM);
    });
}

}  // namespace

extern "C" int cfi_paged_place(const CfiPageTable* t, const CfiPagedPlace* p, void* stream) {
    if (!table_ok(t) || !p || p->n_seq < 0 || p->n_seq > PP_SEQS || p->max_new < 0 || p->max_context < 0 || !p->lens || !p->batch_table ||
        !p->cu_q || !p->cu_kv || !p->status || (p->max_new && (!p->slots || !p->positions)) || (p->n_seq && (!p->rows || !p->n_new)) ||
        (((uintptr_t)p->rows | (uintptr_t)p->n_new | (uintptr_t)p->lens | (uintptr_t)p->batch_table | (uintptr_t)p->cu_q |
          (uintptr_t)p->cu_kv | (uintptr_t)p->positions | (uintptr_t)p->status) & 3) ||
        (((uintptr_t)p->slots | (uintptr_t)p->context) & 7))
        return (int)cudaErrorInvalidValue;
    PpArgs a = {*t, *p, 0, nullptr};
    allow_smem();
    return go((const void*)paged_place, a, (size_t)(5 * p->n_seq + 3) * 4 + seen_bytes(t),
              (long long)p->n_seq * t->max_pages + p->max_new + (p->context ? p->max_context : 0), static_cast<cudaStream_t>(stream));
}

extern "C" int cfi_paged_trim(const CfiPageTable* t, const int32_t* rows, const int32_t* keep, int n_seq, int32_t* status, void* stream) {
    if (!table_ok(t) || n_seq < 0 || n_seq > PP_SEQS || (n_seq && (!rows || !keep)) || !status ||
        (((uintptr_t)rows | (uintptr_t)keep | (uintptr_t)status) & 3))
        return (int)cudaErrorInvalidValue;
    PpArgs a = {};
    a.t = *t;
    a.p.rows = rows;
    a.p.n_new = keep;
    a.p.n_seq = n_seq;
    a.p.status = status;
    allow_smem();
    return go((const void*)paged_trim, a, (size_t)(4 * n_seq + 1) * 4 + seen_bytes(t), (long long)n_seq * t->max_pages,
              static_cast<cudaStream_t>(stream));
}
