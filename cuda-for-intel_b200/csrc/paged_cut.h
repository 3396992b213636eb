// paged_cut.h -- how cfi_paged_attention cuts its list of units into runs, one a CTA: CTA b has the units
// [b * quota, paged_run_end(b * quota)) of `total`.  A total may be as large as an int: no sum here passes it.
#pragma once
#ifdef __CUDACC__
#define CFI_CUT __host__ __device__ __forceinline__
#else
#define CFI_CUT inline
#endif

// Units of a run: the smallest that `ctas` runs of it hold all, and at least `least`.
CFI_CUT int paged_quota(int total, int ctas, int least) {
    const int q = total / ctas + (total % ctas != 0);
    return q > least ? q : least;
}
// CTAs that have a run
CFI_CUT int paged_runs(int total, int quota) { return (total - 1) / quota + 1; }
CFI_CUT int paged_run_end(int begin, int quota, int total) {
    return quota < total - begin ? begin + quota : total;
}
