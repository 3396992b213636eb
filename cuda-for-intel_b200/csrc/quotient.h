// quotient.h -- l / t from r, the reciprocal of t rounded to nearest, without a division.
#pragma once
#include <math.h>
#ifdef __CUDACC__
#define CFI_QUOTIENT __host__ __device__ __forceinline__
#else
#define CFI_QUOTIENT inline
#endif

// Markstein (Computation of elementary functions on the IBM RISC System/6000, 1990): corrections by the exact remainder end at the
// quotient rounded to nearest, the first within an ulp of it.  For t and |l| where neither the quotient nor the
// remainder leaves the normal numbers: the same value as l / t.
CFI_QUOTIENT float quotient_by(float l, float t, float r) {
    const float q0 = l * r, q1 = fmaf(fmaf(-q0, t, l), r, q0);
    return fmaf(fmaf(-q1, t, l), r, q1);
}
