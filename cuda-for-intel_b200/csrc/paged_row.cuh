// paged_row.cuh -- eight values of a row of K or V on their way into a paged cache (paged_cache.cuh).  Four neighbouring
// lanes, 8 values each, make a block of 32; all lanes of a warp call together.
//
// Q8_0: d = max|x| / 127, q = rn(x * (1/d)), stored scale f16(d); read back as f16(q * scale).
// Q4_1: d = (max - min) / 15, q = floor((x - min) / d + 1/2), stored f16(d) and f16(min), all rounded from the exact values.  The
// quotient in 32 bits is off by less than 2^-16 (2^-24 of it each by range and difference, 2^-22 by the quotient): where a value of a
// warp comes nearer to a border than that, its values are compared with their borders, 30 (x - min) with (2 q + 1) (max - min), as sums of
// two f32 numbers each (differences of f16 values meet borders exactly).  d is off by 2 units of its last place in 32 bits and worked out
// in 64 (a difference that 64 bits do not hold as the sum of two) where a border of f16 is nearer or d is no normal f16 number; the
// quotients only where a block's range is below 1.5e-35 or above 9e5.
#pragma once
#include "paged_cache.cuh"

CFI_DEV int to_s8(float x) {  // to the nearest, ties to even; the ends at +-128, a NaN 0
    int q;
    asm("cvt.rni.sat.s8.f32 %0, %1;" : "=r"(q) : "f"(x));
    return q;
}
CFI_DEV uint32_t bytes_of(int a, int b, int c, int d) {
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

// A lane's 8 values, as f32 and as f16.
struct Row8 {
    float x[8];
    uint4 h;
};

template <bool SRC_F16> CFI_DEV float block_max(const Row8& r) {  // of a block that has a NaN: NaN
    float m;
    if (SRC_F16) {
        __half2 h = abs_h2(r.h.x);
        h = __hmax2_nan(__hmax2_nan(h, abs_h2(r.h.y)), __hmax2_nan(abs_h2(r.h.z), abs_h2(r.h.w)));
        h = __hmax2_nan(h, __lowhigh2highlow(h));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) h = __hmax2_nan(h, __shfl_xor_sync(0xffffffffu, h, o));
        m = __low2float(h);
    } else {
        m = 0.0f;
        uint32_t nan = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            m = fmaxf(m, fabsf(r.x[j]));  // drops a NaN
            nan |= (uint32_t)(r.x[j] != r.x[j]);
        }
        if (nan) m = __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            const float other = __shfl_xor_sync(0xffffffffu, m, o);
            m = other != other ? other : m != m ? m : fmaxf(m, other);
        }
    }
    return m;
}

// Values 8 g .. 8 g + 7 of position `off` of a region; nothing is written where `ok` is false.
template <int D, bool SRC_F16> CFI_DEV void put_q8_0(const Row8& r, uint8_t* region, int page_shift, int off, int g, bool ok) {
    const float m = block_max<SRC_F16>(r);
    const float d = m / 127.0f, id = d > 0.0f ? 1.0f / d : 0.0f;
    int q[8];
#pragma unroll
    for (int j = 0; j < 8; j++) q[j] = to_s8(r.x[j] * id);
    const uint32_t w[2] = {bytes_of(q[0], q[1], q[2], q[3]), bytes_of(q[4], q[5], q[6], q[7])};
    if (!ok) return;
    *reinterpret_cast<uint2*>(region + (size_t)off * D + g * 8) = make_uint2(w[0], w[1]);
    if ((g & 3) == 0)
        *reinterpret_cast<uint16_t*>(region + (size_t)(D << page_shift) + ((size_t)off * (D / 32) + g / 4) * 2) =
            d != d ? (uint16_t)0x7fff : f2h_bits(d);
}

CFI_DEV float min_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
CFI_DEV float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
// The least and the largest of a block; both NaN where it has one.
template <bool SRC_F16> CFI_DEV void block_ends(const Row8& r, float* lo, float* hi) {
    if (SRC_F16) {
        const __half2 *h = reinterpret_cast<const __half2*>(&r.h);
        const __half2 a = __hmin2_nan(__hmin2_nan(h[0], h[1]), __hmin2_nan(h[2], h[3])), b = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
        // the negative of the least beside the largest
        __half2 e = __hmax2_nan(__halves2half2(__hneg(__low2half(a)), __low2half(b)), __halves2half2(__hneg(__high2half(a)), __high2half(b)));
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) e = __hmax2_nan(e, __shfl_xor_sync(0xffffffffu, e, o));
        *lo = -__low2float(e);
        *hi = __high2float(e);
    } else {
        float a = r.x[0], b = r.x[0];
#pragma unroll
        for (int j = 1; j < 8; j++) {
            a = min_nan(a, r.x[j]);
            b = max_nan(b, r.x[j]);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            a = min_nan(a, __shfl_xor_sync(0xffffffffu, a, o));
            b = max_nan(b, __shfl_xor_sync(0xffffffffu, b, o));
        }
        *lo = a;
        *hi = b;
    }
}

// a - b, and what that was rounded by
struct Apart {
    double x, rest;
};
CFI_DEV Apart apart(double a, double b) {
    const double x = a - b, back = x - a;
    return {x, (a - (x - back)) - (b + back)};
}

template <int D, bool SRC_F16> CFI_DEV void put_q4_1(const Row8& r, uint8_t* region, int off, int g, bool of_v, bool ok) {
    float lo, hi;
    block_ends<SRC_F16>(r, &lo, &hi);
    const float range = hi - lo, inv = __fdividef(15.0f, range), d32 = range * (1.0f / 15.0f);
    // where 32 bits do not hold the quotients (f16 values are not that near to one another); where d is outside f16's normal numbers or at a border
    // of them.  Blocks of one value, whose q and d are 0, need neither: rows of zeros are common, and so are a warp's lanes without a row.
    const bool wide = !(d32 <= 6.0e4f) || (!SRC_F16 && d32 < 1e-36f && range != 0.0f),
               tie = !(d32 >= 6.2e-5f && d32 <= 6.0e4f) ? range != 0.0f : (__float_as_uint(d32) & 0x1fffu) - 0x0ffcu <= 8u;
    // v + 1.5 * 2^23 is rounded to a whole number, whose last bits are q: with each times 16 and the next, the rest adds up to
    // a number of its own
    uint32_t w = 0, rest = 0;
    float far = 0.0f;
#pragma unroll
    for (int j = 7; j >= 0; j--) {
        const float v = (r.x[j] - lo) * inv, y = v + 12582912.0f;
        far = fmaxf(far, fabsf(v - (y - 12582912.0f)));
        w = w * 16 + __float_as_uint(y);
        rest = rest * 16 + 0x4b400000u;
    }
    w -= rest;
    if (far > 0.49998f && !wide) {  // often, where the values are f16 numbers
        const float rb = range - hi, range_lo = (hi - (range - rb)) - (lo + rb);  // what the difference was rounded by
        w = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const float t = r.x[j] - lo, tb = t - r.x[j], t_lo = (r.x[j] - (t - tb)) - (lo + tb);
            const float v = t * inv, near = (v + 12582912.0f) - 12582912.0f;
            const float twice = 2.0f * near + (v >= near ? 1.0f : -1.0f), p = twice * range;  // of the border that is next
            const float over = (fmaf(30.0f, t, -p) - fmaf(twice, range, -p)) + fmaf(30.0f, t_lo, -twice * range_lo);
            w |= (uint32_t)((int)(twice + (over >= 0.0f ? 1.0f : -1.0f)) >> 1) << (4 * j);
        }
    }
    uint16_t d = f2h_bits(d32);
    if (tie) {
        const Apart all = apart(hi, lo);
        double d64 = all.x / 15.0;
        // exactly so: what the difference was rounded by decides where d lies on a border
        if (all.rest != 0.0 && fma(-15.0, d64, all.x) == 0.0) d64 = __longlong_as_double(__double_as_longlong(d64) + (all.rest > 0.0 ? 1 : -1));
        d = __half_as_ushort(__double2half(d64));
        if (wide) {
            w = 0;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const Apart t = apart(r.x[j], lo);
                const double v = t.x * 15.0 / all.x, near = rint(v), twice = 2.0 * near + (v >= near ? 1.0 : -1.0), p = twice * all.x;
                const double over = (fma(30.0, t.x, -p) - fma(twice, all.x, -p)) + fma(30.0, t.rest, -twice * all.rest);
                w |= all.x > 0.0 ? (uint32_t)((int)(twice + (over >= 0.0 ? 1.0 : -1.0)) >> 1) << (4 * j) : 0;
            }
        }
    }
    if (range == 0.0f) w = 0;
    uint16_t m = f2h_bits(lo);
    if ((d & 0x7c00) == 0x7c00 || (m & 0x7c00) == 0x7c00) {
        d = m = 0x7fff;
        w = 0;
    }
    if (!ok) return;
    const int row = off % Q41_TILE, b = g >> 2, c = g & 3;
    uint8_t* tile = region + Q41<D>::tile_at(off);
    if (of_v) {
        *reinterpret_cast<uint16_t*>(tile + Q41<D>::v_at(row, b, 2 * c)) = (uint16_t)w;
        *reinterpret_cast<uint16_t*>(tile + Q41<D>::v_at(row, b, 2 * c + 1)) = (uint16_t)(w >> 16);
    } else {
        *reinterpret_cast<uint32_t*>(tile + Q41<D>::k_at(row, b, c)) = w;
    }
    if (c == 0) *reinterpret_cast<uint16_t*>(tile + Q41<D>::scale_at(row, b)) = d;
    if (c == 1) *reinterpret_cast<uint16_t*>(tile + Q41<D>::min_at(row, b)) = m;
}

template <int D, int TY, bool SRC_F16>
CFI_DEV void put_row8(const Row8& r, uint8_t* region, int page_shift, int off, int g, bool of_v, bool ok) {
    if (TY == CACHE_F16) {
        if (ok) *reinterpret_cast<uint4*>(region + ((size_t)off * D + g * 8) * 2) = r.h;
    } else if (TY == CACHE_Q8_0) {
        put_q8_0<D, SRC_F16>(r, region, page_shift, off, g, ok);
    } else {
        put_q4_1<D, SRC_F16>(r, region, off, g, of_v, ok);
    }
}
