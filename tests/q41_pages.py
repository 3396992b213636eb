"""Q4_1 pages of a paged cache (include/cfi_serve.h) in numpy, from the header's words: the values of a pool, and blocks quantised
by the definition in 64 bits."""
import numpy as np


def region_bytes(page, dim):
    return page * dim * 5 // 8


def values(pool_bytes, pages, kv, page, dim, of_v):
    """Every slot of a pool in 64 bits: [slot, head, dim]."""
    t = pool_bytes.reshape(pages, kv, page // 16, dim * 10)
    nib = t[..., :dim * 8].reshape(pages, kv, page // 16, 16, dim // 2)
    par = np.ascontiguousarray(t[..., dim * 8:]).view(np.float16).astype(np.float64).reshape(pages, kv, page // 16, 16, 2, dim // 32)
    out = np.empty((pages, kv, page // 16, 16, dim))
    for r in range(16):
        for b in range(dim // 32):
            for i in range(32):
                if of_v:
                    g = i // 4
                    if dim == 128 and r in (2, 3, 6, 7, 10, 11, 14, 15):
                        g ^= 4
                    at, half = g * (dim // 16) + 2 * b + i % 4 // 2, i % 2
                else:
                    at, half = i // 8 * (dim // 8) + 4 * b + i % 8 // 2, i % 2
                n = nib[:, :, :, r, at] >> (4 * half) & 15
                with np.errstate(invalid="ignore", over="ignore"):
                    out[:, :, :, r, 32 * b + i] = n * par[:, :, :, r, 0, b] + par[:, :, :, r, 1, b]
    return out.reshape(pages, kv, page, dim).transpose(0, 2, 1, 3).reshape(pages * page, kv, dim)


def quantised(x):
    """What rows of values are stored as."""
    b = np.asarray(x, dtype=np.float64).reshape(-1, 32)
    with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
        lo, hi = b.min(1, keepdims=True), b.max(1, keepdims=True)
        wide = hi - lo
        q = np.zeros_like(b)
        for i in range(1, 16):  # the borders, met by what is not below them; differences of f32 values are exact here
            q += (30.0 * (b - lo) >= (2 * i - 1) * wide) & (wide > 0)
        d, m = (wide / 15.0).astype(np.float16).astype(np.float64), lo.astype(np.float16).astype(np.float64)
        bad = ~(np.isfinite(b).all(1, keepdims=True) & np.isfinite(d) & np.isfinite(m))
        return np.where(bad, np.nan, q * d + m).reshape(np.shape(x))
