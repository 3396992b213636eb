// k_paged_place.cu -- page tables, slots, positions and packed offsets of a batch made on the device, and pages given back
// (include/cfi_serve.h).  Whole numbers only: what a call writes does not depend on any order.
//
// A CTA adds up what the sequences hold, get and need (a thread takes some in a row, then one scan over the threads); every
// element of the lists then finds its sequence by bisection among the sums in shared memory.
#include "paged_cache.cuh"
#include "sm100_ptx.cuh"
#include "cfi_kernels.h"

#include <stdlib.h>
#include <string.h>

namespace {

constexpr int PP_THREADS = 1024, PP_SEQS = 8192, PP_ROWS = 65536;

struct PpArgs {
    CfiPageTable t;
    CfiPagedPlace p;  // of a trim: rows, n_new (what to keep), n_seq, status
    int page_shift;
};

// Sums over the threads of three numbers: those of the threads before this one, and all.
struct Sums {
    long long q, kv;
    int pages;
};
CFI_DEV Sums operator+(const Sums& a, const Sums& b) { return {a.q + b.q, a.kv + b.kv, a.pages + b.pages}; }
CFI_DEV Sums scan(Sums x, Sums* total) {
    __shared__ Sums s_warp[32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Sums incl = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums y = {__shfl_up_sync(0xffffffffu, incl.q, o), __shfl_up_sync(0xffffffffu, incl.kv, o), __shfl_up_sync(0xffffffffu, incl.pages, o)};
        if (lane >= o) incl = incl + y;
    }
    if (lane == 31) s_warp[warp] = incl;
    __syncthreads();
    Sums before = {0, 0, 0}, all = {0, 0, 0};
    for (int w = 0; w < PP_THREADS / 32; w++) {
        if (w == warp) before = all;
        all = all + s_warp[w];
    }
    __syncthreads();
    *total = all;
    return {before.q + incl.q - x.q, before.kv + incl.kv - x.kv, before.pages + incl.pages - x.pages};
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

__global__ void __launch_bounds__(PP_THREADS) paged_place(const __grid_constant__ PpArgs a) {
    extern __shared__ int smem[];
    const CfiPageTable& t = a.t;
    const CfiPagedPlace& p = a.p;
    const int n = p.n_seq, tid = threadIdx.x, mask = t.page_size - 1;
    int *cu_q = smem, *cu_kv = cu_q + n + 1, *first = cu_kv + n + 1, *row = first + n;  // first: of the pages taken
    uint32_t* seen = reinterpret_cast<uint32_t*>(row + n);
    __shared__ int s_why;
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    for (int i = tid; i < (t.n_rows + 31) / 32; i += PP_THREADS) seen[i] = 0;
    if (tid == 0) s_why = 0x7fffffff;
    __syncthreads();
    const int each = (n + PP_THREADS - 1) / PP_THREADS, s0 = min(n, tid * each), s1 = min(n, s0 + each);
    const int n_free = min(max(*t.n_free, 0), t.n_pages);
    Sums mine = {0, 0, 0};
    int why = 0x7fffffff;
    for (int s = s0; s < s1; s++) {
        const int r = p.rows[s], add = p.n_new[s];
        if (bad_row(seen, r, t.n_rows) || add < 0) {
            why = min(why, (int)CFI_PLACE_BAD_ROW);
            continue;
        }
        row[s] = r;
        const int held = t.cached[r];
        const long long after = (long long)held + add;
        if (held < 0) why = min(why, (int)CFI_PLACE_BAD_ROW);
        else if (after > (long long)t.max_pages << a.page_shift || after > 0x7fffffffLL - mask) why = min(why, (int)CFI_PLACE_TOO_LONG);
        else mine = mine + Sums{add, after, (int)((after + mask) >> a.page_shift) - ((held + mask) >> a.page_shift)};
    }
    Sums all;
    Sums at = scan(mine, &all);
    if (all.kv > 0x7fffffffLL) why = min(why, (int)CFI_PLACE_TOO_LONG);
    if (all.q > p.max_new || (p.context && all.kv > p.max_context)) why = min(why, (int)CFI_PLACE_NO_ROOM);
    if (all.pages > n_free) why = min(why, (int)CFI_PLACE_NO_PAGES);
    if (why != 0x7fffffff) atomicMin(&s_why, why);
    __syncthreads();
    const bool ok = s_why == 0x7fffffff;
    for (int s = s0; s < s1; s++) {
        int add = 0, after = 0, need = 0;
        if (ok) {
            add = p.n_new[s];
            const int held = t.cached[row[s]];
            after = held + add;
            need = ((after + mask) >> a.page_shift) - ((held + mask) >> a.page_shift);
        }
        cu_q[s] = (int)(ok ? at.q : 0);
        cu_kv[s] = (int)(ok ? at.kv : 0);
        first[s] = at.pages;
        p.cu_q[s] = cu_q[s];
        p.cu_kv[s] = cu_kv[s];
        p.lens[s] = after;
        at = at + Sums{add, after, need};
    }
    if (tid == 0) {
        p.status[0] = ok ? (int)CFI_PLACED : s_why;
        p.cu_q[n] = cu_q[n] = ok ? (int)all.q : 0;
        p.cu_kv[n] = cu_kv[n] = ok ? (int)all.kv : 0;
    }
    __syncthreads();
    // page i of sequence s, which held `old` pages before
    auto page = [&](int s, int i, int old) {
        return i < old ? t.table[(long long)row[s] * t.max_pages + i] : t.free_pages[n_free - 1 - (first[s] + i - old)];
    };
    auto held = [&](int s) { return cu_kv[s + 1] - cu_kv[s] - (cu_q[s + 1] - cu_q[s]); };
    for (int s = tid >> 5; ok && s < n; s += PP_THREADS / 32) {
        const int old = (held(s) + mask) >> a.page_shift, pages = (cu_kv[s + 1] - cu_kv[s] + mask) >> a.page_shift;
        for (int i = tid & 31; i < pages; i += 32) {
            const int id = page(s, i, old);
            p.batch_table[(long long)s * t.max_pages + i] = id;
            if (i >= old) t.table[(long long)row[s] * t.max_pages + i] = id;
        }
    }
    for (int i = tid; i < p.max_new; i += PP_THREADS) {
        long long slot = -1;
        int pos = 0;
        if (i < cu_q[n]) {
            const int s = sequence_of(cu_q, n, i), h = held(s);
            pos = h + i - cu_q[s];
            slot = ((long long)page(s, pos >> a.page_shift, (h + mask) >> a.page_shift) << a.page_shift) + (pos & mask);
        }
        p.slots[i] = slot;
        p.positions[i] = pos;
    }
    for (int i = tid; p.context && i < p.max_context; i += PP_THREADS) {
        long long slot = -1;
        if (i < cu_kv[n]) {
            const int s = sequence_of(cu_kv, n, i), pos = i - cu_kv[s];
            slot = ((long long)page(s, pos >> a.page_shift, (held(s) + mask) >> a.page_shift) << a.page_shift) + (pos & mask);
        }
        p.context[i] = slot;
    }
    if (!ok) return;
    for (int s = s0; s < s1; s++) t.cached[row[s]] = cu_kv[s + 1] - cu_kv[s];
    if (tid == 0) *t.n_free = n_free - all.pages;
}

__global__ void __launch_bounds__(PP_THREADS) paged_trim(const __grid_constant__ PpArgs a) {
    extern __shared__ int smem[];
    const CfiPageTable& t = a.t;
    const int n = a.p.n_seq, tid = threadIdx.x, mask = t.page_size - 1;
    const int32_t* keep = a.p.n_new;
    int *first = smem, *from = first + n + 1, *row = from + n;  // of the pages given back; the first such of a row
    uint32_t* seen = reinterpret_cast<uint32_t*>(row + n);
    __shared__ int s_why;
    sm100::pdl_launch_dependents();
    sm100::pdl_wait();
    for (int i = tid; i < (t.n_rows + 31) / 32; i += PP_THREADS) seen[i] = 0;
    if (tid == 0) s_why = 0x7fffffff;
    __syncthreads();
    const int each = (n + PP_THREADS - 1) / PP_THREADS, s0 = min(n, tid * each), s1 = min(n, s0 + each);
    const int n_free = min(max(*t.n_free, 0), t.n_pages);
    Sums mine = {0, 0, 0};
    int why = 0x7fffffff;
    for (int s = s0; s < s1; s++) {
        const int r = a.p.rows[s];
        row[s] = r;
        if (bad_row(seen, r, t.n_rows)) {
            why = min(why, (int)CFI_PLACE_BAD_ROW);
            continue;
        }
        const int held = t.cached[r], now = min(held, max(keep[s], 0));
        if (held < 0) {
            why = min(why, (int)CFI_PLACE_BAD_ROW);
        } else if (held > (long long)t.max_pages << a.page_shift || held > 0x7fffffff - mask) {
            why = min(why, (int)CFI_PLACE_TOO_LONG);
        } else {
            first[s] = mine.pages;
            from[s] = (now + mask) >> a.page_shift;
            const int gone = ((held + mask) >> a.page_shift) - from[s];
            mine = mine + Sums{0, gone, gone};
        }
    }
    Sums all;
    const Sums at = scan(mine, &all);
    if (all.kv > t.n_pages - n_free) why = min(why, (int)CFI_PLACE_NO_PAGES);
    if (why != 0x7fffffff) atomicMin(&s_why, why);
    __syncthreads();
    if (s_why != 0x7fffffff) {
        if (tid == 0) a.p.status[0] = s_why;
        return;
    }
    for (int s = s0; s < s1; s++) {
        first[s] += at.pages;
        t.cached[row[s]] = min(t.cached[row[s]], max(keep[s], 0));
    }
    if (tid == 0) {
        first[n] = all.pages;
        *t.n_free = n_free + all.pages;
        a.p.status[0] = CFI_PLACED;
    }
    __syncthreads();
    for (int s = tid >> 5; s < n; s += PP_THREADS / 32)
        for (int i = tid & 31; i < first[s + 1] - first[s]; i += 32)
            t.free_pages[n_free + all.pages - 1 - (first[s] + i)] = t.table[(long long)row[s] * t.max_pages + from[s] + i];
}

bool table_ok(const CfiPageTable* t) {
    return t && t->table && t->cached && t->free_pages && t->n_free &&
           !(((uintptr_t)t->table | (uintptr_t)t->cached | (uintptr_t)t->free_pages | (uintptr_t)t->n_free) & 3) && t->n_rows > 0 &&
           t->n_rows <= PP_ROWS && t->max_pages > 0 && t->page_size >= 16 && t->page_size <= 256 && (t->page_size & (t->page_size - 1)) == 0 &&
           t->n_pages > 0;
}
size_t seen_bytes(const CfiPageTable* t) { return (size_t)(t->n_rows + 31) / 32 * 4; }

int go(const void* fn, PpArgs& a, size_t smem, cudaStream_t stream) {
    a.page_shift = __builtin_ctz((unsigned)a.t.page_size);
    const char* ep = getenv("CFI_PDL");
    cudaLaunchConfig_t c = {};
    c.gridDim = dim3(1, 1, 1);
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
constexpr int PP_SMEM = PP_ROWS / 8 + (4 * PP_SEQS + 2) * 4;
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
    PpArgs a = {*t, *p, 0};
    allow_smem();
    return go((const void*)paged_place, a, (size_t)(4 * p->n_seq + 2) * 4 + seen_bytes(t), static_cast<cudaStream_t>(stream));
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
    return go((const void*)paged_trim, a, (size_t)(3 * n_seq + 1) * 4 + seen_bytes(t), static_cast<cudaStream_t>(stream));
}
