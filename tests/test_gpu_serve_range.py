"""The serving operators at the ends of their ranges: one key that outweighs a long flat tail, small and large
values of Q8_0 blocks, small and large queries, batches past the sequences that a lane keeps, logits whose
quotient by the temperature overflows.

Bounds, as in test_gpu_serve.py: a score is off by at most EPS_S times the sum of its products' magnitudes times
the scale, a weight by that much twice (numerator and sum) and 2^-20 twice for the exponential.  Three more terms count
here.  A weight is held to 22 bits or to 2^-40 of the largest, whichever is coarser.  A sum of n positions is n / 16
additions in 32 bits one after another, each off by an ulp of 2^-23 at most.  An output is compared with its own
size where the largest value has no part in it."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
from test_gpu_serve import DEV, EPS_S, attend, decode_case, fits, garbage_pool, pool_rows, sample, stream  # noqa: E402

pytestmark = pytest.mark.gpu
F16, F32, Q8 = cfi.T_F16, cfi.T_F32, cfi.Q8_0


def filled(ty, kv, dim, page, k, v):
    """Pools that hold the rows k and v [position, kv * dim] at slots 0, 1, ..."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(1)
    pages = -(-k.shape[0] // page)
    pools = [garbage_pool(ty, pages, kv, page, dim, gen) for _ in "kv"]
    cache = cfi.paged_cache(ty, pools[0].data_ptr(), pools[1].data_ptr(), pages, page, kv, dim)
    slots = torch.arange(k.shape[0], device=DEV)
    cfi.paged_kv_store(cache, k.data_ptr(), v.data_ptr(), slots.data_ptr(), k.shape[0], stream=stream())
    rows = [pool_rows(p, ty, pages, kv, page, dim)[:k.shape[0]] for p in pools]
    return cache, pools, rows


def attention(cache, q, table, lens, scale):
    batch, width = q.shape
    out = torch.full_like(q, 7.0)
    cfi.paged_attention(cache, q.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(), batch, width // cache.head_dim,
                        table.shape[1], scale, stream=stream())
    torch.cuda.synchronize()
    return out.double().cpu().numpy().reshape(batch, -1, cache.head_dim)


# ---- weights ----
@pytest.mark.parametrize("ty", [F16, Q8])
@pytest.mark.parametrize("heads,kv,dim,batch,n", [(14, 2, 64, 64, 65536), (32, 8, 128, 8, 65000), (12, 2, 128, 1, 700)])
@pytest.mark.parametrize("gap", [10.0, 14.3, 17.0, 17.5, 18.7])
def test_one_key_over_a_long_flat_tail(ty, heads, kv, dim, batch, n, gap):
    """The first key outweighs each of the others by e^gap and has no value; the others are equal and share one page."""
    page = 16
    scale = 1.0 / math.sqrt(dim)
    k = torch.zeros(2 * page, kv * dim, device=DEV)
    k[0] = 1.0
    v = torch.ones(2 * page, kv * dim, device=DEV)
    v[0] = 0.0
    cache, pools, (K, V) = filled(ty, kv, dim, page, k, v)
    width = -(-n // page)
    table = torch.ones(batch, width, dtype=torch.int32, device=DEV)
    table[:, 0] = 0
    lens = torch.full((batch,), n, dtype=torch.int32, device=DEV)
    q = torch.full((batch, heads * dim), gap / (dim * scale), device=DEV)
    got = attention(cache, q, table, lens, scale)
    score = float(q[0, 0].double()) * scale * K[0, 0].sum()
    tail = (n - 1) * math.exp(-score)
    want = tail / (1 + tail) * float(V[1, 0, 0])
    tol = want * (2 * EPS_S * score + 2 * 2.0 ** -20 + -(-n // 16) * 2.0 ** -23) + n * 2.0 ** -40
    assert np.abs(got - want).max() <= tol, (float(np.abs(got - want).max()) / want, tol / want)


def values_case(ty, heads, kv, dim, n, amplitude, seed=0):
    """Random scores over n positions of values of the given amplitude [position, 1 or dim]; compared block by block of 32 dims."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + n)
    page = 32
    k = torch.randn(n, kv * dim, generator=gen, device=DEV)
    v = torch.randn(n, kv, dim, generator=gen, device=DEV).clamp(-3, 3) * amplitude.to(DEV)[:, None]
    cache, pools, (K, V) = filled(ty, kv, dim, page, k, v.reshape(n, -1).contiguous())
    q = torch.randn(1, heads * dim, generator=gen, device=DEV)
    table = torch.arange(-(-n // page), dtype=torch.int32, device=DEV)[None].contiguous()
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    scale = 1.0 / math.sqrt(dim)
    got = attention(cache, q, table, lens, scale)[0]
    Q = q.double().cpu().numpy().reshape(heads, dim)
    g = heads // kv
    for h in range(kv):
        qq = Q[h * g:(h + 1) * g]
        want = attend(qq, K[:, h], V[:, h], scale)
        S = float((np.abs(qq) @ np.abs(K[:, h]).T).max() * scale)
        largest = np.abs(V[:, h]).max()
        for b in range(0, dim, 32):
            tol = (2 * EPS_S * S + 2 * 2.0 ** -20 + -(-n // 16) * 2.0 ** -23) * np.abs(V[:, h, b:b + 32]).max() + n * 2.0 ** -40 * largest
            err = np.abs(got[h * g:(h + 1) * g, b:b + 32] - want[:, b:b + 32])
            assert (err <= tol).all(), (h, b, float((err / tol).max()))


@pytest.mark.parametrize("ty", [F16, Q8])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("n", [5, 600, 9000])
def test_values_of_all_sizes(ty, heads, kv, dim, n):
    """Values from f16's smallest normal ones to its largest, the same everywhere, growing and falling along the positions, and
    of another size in each block of 32 dims."""
    one = torch.ones(n, 1)
    for size in (1.0, 1.3e-3, 1.3e-4, 2e4):
        values_case(ty, heads, kv, dim, n, one * size)
    steps = torch.linspace(0, 1, n)[:, None]
    values_case(ty, heads, kv, dim, n, 1e-3 * 1e7 ** steps)
    values_case(ty, heads, kv, dim, n, 1e4 * 1e-7 ** steps)
    blocks = torch.tensor([1e-3, 30.0, 1.0, 1e3])[torch.arange(dim) // 32 % 4][None].expand(n, dim)
    values_case(ty, heads, kv, dim, n, blocks)
    values_case(ty, heads, kv, dim, n, blocks.roll(32, 1))


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128)])
def test_values_of_q8_0_past_f16(heads, kv, dim):
    """A block's scale may be any f16, its values then pass f16's range."""
    values_case(Q8, heads, kv, dim, 700, torch.full((700, 1), 1e6))


@pytest.mark.parametrize("ty", [F16, Q8])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("n", [5, 600, 9000])
def test_large_equal_scores(ty, heads, kv, dim, n):
    """Scores of 2e8 that are all the same: the mean of values whose size changes along the positions, as if they were zero."""
    page = 16
    gen = torch.Generator(device=DEV)
    gen.manual_seed(n)
    k = torch.full((n, kv * dim), 100.0, device=DEV)
    for grow in (1e6, 1e-6):
        v = torch.randn(n, kv * dim, generator=gen, device=DEV).clamp(-3, 3) * max(1.0, 1 / grow) * 1e-3 * grow ** torch.linspace(0, 1, n, device=DEV)[:, None]
        cache, pools, (K, V) = filled(ty, kv, dim, page, k, v)
        q = torch.full((1, heads * dim), 3e5, device=DEV)
        table = torch.arange(-(-n // page), dtype=torch.int32, device=DEV)[None].contiguous()
        got = attention(cache, q, table, torch.tensor([n], dtype=torch.int32, device=DEV), 1.0 / math.sqrt(dim))[0]
        want = np.repeat(V.mean(0), heads // kv, axis=0)
        tol = (2 * 2.0 ** -20 + -(-n // 16) * 2.0 ** -23 + n * 2.0 ** -40) * np.abs(V).max()
        assert np.abs(got - want).max() <= tol, (grow, float(np.abs(got - want).max() / tol))


# ---- queries ----
def queries_case(ty, heads, kv, dim, n, q_size, k_size, seed=0):
    """q_size and k_size: one number, or one for each dim."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + n + dim)
    page = 16
    of = lambda x: torch.as_tensor(x, dtype=torch.float32, device=DEV)  # noqa: E731
    k = (torch.randn(n, kv, dim, generator=gen, device=DEV).clamp(-3, 3) * of(k_size)).reshape(n, -1).contiguous()
    v = torch.randn(n, kv * dim, generator=gen, device=DEV)
    cache, pools, (K, V) = filled(ty, kv, dim, page, k, v)
    q = (torch.randn(1, heads, dim, generator=gen, device=DEV) * of(q_size)).reshape(1, -1).contiguous()
    table = torch.arange(-(-n // page), dtype=torch.int32, device=DEV)[None].contiguous()
    lens = torch.tensor([n], dtype=torch.int32, device=DEV)
    scale = 1.0 / math.sqrt(dim)
    got = attention(cache, q, table, lens, scale)[0]
    Q = q.double().cpu().numpy().reshape(heads, dim)
    g = heads // kv
    for h in range(kv):
        qq = Q[h * g:(h + 1) * g]
        want = attend(qq, K[:, h], V[:, h], scale)
        S = np.abs(qq) @ np.abs(K[:, h]).T * scale  # of each head its largest
        tol = (2 * EPS_S * S.max(1, keepdims=True) + 2 * 2.0 ** -20 + -(-n // 16) * 2.0 ** -23) * np.abs(V[:, h]).max()
        err = np.abs(got[h * g:(h + 1) * g] - want)
        assert (err <= tol).all(), (h, float((err / tol).max()))


@pytest.mark.parametrize("ty", [F16, Q8])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128)])
@pytest.mark.parametrize("q_size,k_size", [(1e-2, 1e2), (1e-4, 1e4), (1e-6, 2e4), (1e3, 1e-3), (1e6, 1e-3), (1e30, 1.0), (1e-30, 1.0)])
def test_queries_of_all_sizes(ty, heads, kv, dim, q_size, k_size):
    """A query's size is its own matter: 22 bits of each value whatever that is.  (1e30: one key takes all.)"""
    for n in (3, 1500):
        if q_size < 1e20:
            queries_case(ty, heads, kv, dim, n, q_size, k_size)
        else:  # no rounding of the scores reaches the distance of two of them
            one_takes_all(ty, heads, kv, dim, n, q_size)


def one_takes_all(ty, heads, kv, dim, n, q_size):
    page = 16
    k = torch.zeros(n, kv * dim, device=DEV)
    k[:] = (torch.arange(n, device=DEV) * 0.5 / n)[:, None]
    k[n // 2] = 2.0
    v = torch.randn(n, kv * dim, generator=torch.Generator(device=DEV).manual_seed(n), device=DEV)
    cache, pools, (K, V) = filled(ty, kv, dim, page, k, v)
    q = torch.full((1, heads * dim), q_size, device=DEV)
    table = torch.arange(-(-n // page), dtype=torch.int32, device=DEV)[None].contiguous()
    got = attention(cache, q, table, torch.tensor([n], dtype=torch.int32, device=DEV), 1.0 / math.sqrt(dim))[0]
    want = np.repeat(V[n // 2], heads // kv, axis=0)
    assert (np.abs(got - want) <= 2 * 2.0 ** -20 * np.abs(want)).all()


@pytest.mark.parametrize("ty", [F16, Q8])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128)])
def test_queries_with_outlier_channels(ty, heads, kv, dim):
    """Large channels of K (a block of 32 of them, as Q8_0 scales them) beside small ones of q, and the reverse."""
    wide = torch.arange(dim) // 32 == 1
    for q_size, k_size in ((torch.where(wide, 1e-4, 1.0), torch.where(wide, 1e4, 1.0)),
                           (torch.where(wide, 1e2, 1e-2), torch.where(wide, 1e-2, 1e2))):
        queries_case(ty, heads, kv, dim, 1500, q_size, k_size)


@pytest.mark.parametrize("ty", [F16, Q8])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
def test_bad_queries_and_rows_stay_where_they_are(ty, bad):
    """A query head of zeros is a mean, one with a NaN or an infinity is NaN, and the other heads and sequences are what they are
    without it; so are they beside a NaN among another sequence's or another kv head's rows."""
    heads, kv, dim, page, n = 12, 2, 64, 16, 300
    gen = torch.Generator(device=DEV)
    gen.manual_seed(3)
    k, v = (torch.randn(2 * n, kv * dim, generator=gen, device=DEV) for _ in "kv")
    q = torch.randn(2, heads * dim, generator=gen, device=DEV)
    q[0, 2 * dim:3 * dim] = 0
    at = torch.arange(-(-2 * n // page), dtype=torch.int32, device=DEV)
    table = torch.stack([at[:19], at[18:37]]).contiguous()
    lens = torch.tensor([n, 294], dtype=torch.int32, device=DEV)
    cache, pools, (K, V) = filled(ty, kv, dim, page, k, v)
    want = attention(cache, q, table, lens, 0.125)
    mean = V[:n, 0].mean(0)
    assert np.abs(want[0, 2] - mean).max() <= (2 * 2.0 ** -20 + 19 * 2.0 ** -23) * np.abs(V).max()
    r = q.clone()
    r[0, 5 * dim + 7] = bad
    got = attention(cache, r, table, lens, 0.125)
    assert np.isnan(got[0, 5]).all()
    rest = np.ones((2, heads), bool)
    rest[0, 5] = False
    np.testing.assert_array_equal(got[rest], want[rest])
    for which in range(2):
        rows = [k.clone(), v.clone()]
        rows[which][37, dim + 40] = math.nan  # kv head 1, of the first sequence alone
        cache, pools, _ = filled(ty, kv, dim, page, *rows)
        got = attention(cache, q, table, lens, 0.125)
        reach = slice(0, dim) if which == 0 else slice(32, dim) if ty == Q8 else slice(40, 41)
        assert np.isnan(got[0, 6:, reach]).all()
        np.testing.assert_array_equal(got[0, :6], want[0, :6])
        np.testing.assert_array_equal(got[1], want[1])


# ---- packed prompts ----
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128), (40, 2, 64)])
@pytest.mark.parametrize("nq,nk", [([1, 40, 300], [1, 40, 300]), ([200, 130, 3], [333, 100, 700]), ([3000, 50], [3000, 800])])
@pytest.mark.parametrize("ot", [F32, F16])
def test_packed_attention_bad_values_reach_who_sees_them(heads, kv, dim, nq, nk, ot):
    """Non-finite values of a key leave the queries that do not see it, and the other dims, as they are; who sees one gets it.
    A NaN among a key's own numbers makes NaN of all of those, and of nothing else."""
    gen = torch.Generator(device=DEV)
    gen.manual_seed(heads + sum(nq))
    g, scale = heads // kv, 1.0 / math.sqrt(dim)
    q = (torch.randn(sum(nq), heads * dim, generator=gen, device=DEV) * 1.5).half()
    k, v = (torch.randn(sum(nk), kv * dim, generator=gen, device=DEV).half() for _ in "kv")
    cq, ck = (np.cumsum([0] + n) for n in (nq, nk))
    clean_k, clean_v = k.clone(), v.clone()
    where = {}  # of each sequence: key and dims of V in kv head 0, key of K in kv head 1
    for s, (n, m) in enumerate(zip(nq, nk)):
        at = max(0, m - 1 - n // 2)
        where[s] = at, max(0, m - 1 - n // 3)
        v[ck[s] + at, 5] = math.nan
        v[ck[s] + at, 40] = math.inf
        k[ck[s] + where[s][1], dim + 9] = math.nan
    out = torch.full((sum(nq), heads * dim), 7.0, dtype=torch.float16 if ot == F16 else torch.float32, device=DEV)
    du, dk = (torch.from_numpy(c.astype(np.int32)).to(DEV) for c in (cq, ck))
    cfi.packed_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), du.data_ptr(), dk.data_ptr(), len(nq), sum(nq), sum(nk),
                         heads, kv, dim, scale, out_type=ot, stream=stream())
    torch.cuda.synchronize()
    assert cfi.lib().cfi_device_error() == 0
    for s, (n, m) in enumerate(zip(nq, nk)):
        Q = q[cq[s]:cq[s + 1]].double().reshape(n, kv, g, dim).permute(1, 2, 0, 3)
        K, V = (x[ck[s]:ck[s + 1]].double().reshape(m, kv, dim).permute(1, 0, 2)[:, None] for x in (clean_k, clean_v))
        got = out[cq[s]:cq[s + 1]].double().reshape(n, kv, g, dim).permute(1, 2, 0, 3)
        last = torch.arange(n, device=DEV) + (m - n)  # the last key that a query sees
        x = (Q @ K.transpose(2, 3)) * scale
        x = x.masked_fill(torch.arange(m, device=DEV)[None] > last[:, None], -math.inf)
        p = torch.softmax(x, -1)
        p[:, :, last < 0] = 0
        want = p @ V
        S = float((Q.abs() @ K.abs().transpose(2, 3)).max() * scale)
        tol = (2 * EPS_S * S + 2 * 2.0 ** -20 + 2.0 ** -11) * float(V.abs().max())
        if ot == F16:
            tol = tol + 2.0 ** -11 * want.abs() + 2.0 ** -25
        sees_v, sees_k = last >= where[s][0], last >= where[s][1]
        near = (got - want).abs() <= tol
        assert torch.isnan(got[0][:, sees_v][..., 5]).all() and not torch.isfinite(got[0][:, sees_v][..., 40]).any()
        near[0][:, sees_v, 5] = True
        near[0][:, sees_v, 40] = True
        assert torch.isnan(got[1][:, sees_k]).all()
        near[1][:, sees_k] = True
        assert near.all(), (s, torch.nonzero(~near)[:4].tolist(), int((~near).sum()))


# ---- batches ----
@pytest.mark.parametrize("ty", [F16, Q8])
@pytest.mark.parametrize("heads,kv,dim,batch", [(14, 2, 64, 129), (12, 2, 128, 300), (4, 1, 64, 1000)])
def test_many_sequences(ty, heads, kv, dim, batch):
    """More sequences than the lanes keep the lengths of, in tables that a CTA takes whole with four warps and in longer ones."""
    rng = np.random.default_rng(batch)
    lens = [int(x) for x in rng.integers(-1, 200, batch)]
    decode_case(ty, heads, kv, dim, 16, lens, F32, F32)[1]()
    lens[batch - 3] = 3000
    decode_case(ty, heads, kv, dim, 16, lens, F32, F32)[1]()
    decode_case(ty, heads, kv, dim, 64, lens[::-1], F16, F16, pad=8)[1]()


# ---- sampling ----
@pytest.mark.parametrize("rows", [6, 80])
@pytest.mark.parametrize("vocab", [40, 5000, 70000])
def test_sample_temperature_whose_quotient_overflows(rows, vocab):
    """logit / temperature may pass the largest float: the largest logits share the weight all the same, whatever their
    sign, and nothing else has any."""
    rng = np.random.default_rng(vocab)
    z = rng.normal(size=(rows, vocab)).astype(np.float32)
    low = np.finfo(np.float32).min
    t = np.ones(rows, np.float32)
    for r in range(rows):
        kind = r % 6
        a, b = vocab // 3, vocab // 2
        if kind == 0:
            z[r, b], t[r] = 9.0, 1e-39
            z[r, a] = 8.0
        elif kind == 1:
            z[r] -= 20.0
            z[r, b], t[r] = -1.0, 1e-40
        elif kind == 2:
            z[r, [a, b]], t[r] = 9.0, 1e-39
        elif kind == 3:
            z[r], t[r] = low, 0.7
        elif kind == 4:
            z[r], t[r] = low, 0.7
            z[r, b] = -3.0
        else:
            z[r, b], t[r] = np.finfo(np.float32).max, 0.5
    u = np.full(rows, 0.75, np.float32)
    for k, p in ((0, 1.0), (7, 0.9), (0, 0.9)):
        token, lp = sample(torch.from_numpy(z).to(DEV), u, t, [k] * rows, [p] * rows)
        for r in range(rows):
            kind = r % 6
            a, b = vocab // 3, vocab // 2
            if kind == 2:
                assert token[r] == b and abs(lp[r] + math.log(2)) <= 1e-6, (r, k, p)
            elif kind == 3:
                count = math.ceil((k or vocab) * np.float64(np.float32(p)) - 1e-6)
                assert token[r] == int(0.75 * count) and abs(lp[r] + math.log(count)) <= 4e-6 * math.log(count), (r, k, p)
            else:
                assert token[r] == b and lp[r] == 0, (r, k, p, token[r])


def test_sample_small_temperatures_stay_exact():
    """Down to where the quotient just holds."""
    rng = np.random.default_rng(4)
    z = rng.normal(size=(5, 3000)).astype(np.float32)
    t = np.array([1e-3, 1e-10, 1e-30, 1e-37, 2e-38], np.float32)
    u = rng.random(5).astype(np.float32)
    token, lp = sample(torch.from_numpy(z).to(DEV), u, t)
    for r in range(5):
        assert fits(z[r], u[r], token[r], lp[r], t[r])


# ---- graphs ----
def test_a_captured_step_is_replayed_with_new_inputs():
    """Rows stored, read back, attended to packed and by single tokens, logits sampled, twice over in one graph: replayed with other
    rows, slots, tables, lengths and settings it gives what the calls give one after another."""
    heads, kv, dim, page, pages, n, batch, rows, vocab = 12, 2, 64, 16, 40, 300, 3, 40, 66000
    gen = torch.Generator(device=DEV)
    gen.manual_seed(11)
    size = cfi.paged_page_bytes(Q8, page, kv, dim) * pages
    pools = torch.zeros(2, size, dtype=torch.uint8, device=DEV)
    cache = cfi.paged_cache(Q8, pools[0].data_ptr(), pools[1].data_ptr(), pages, page, kv, dim)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=DEV)  # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=DEV)  # noqa: E731
    x = dict(k=f32(n, kv * dim), v=f32(n, kv * dim), slots=torch.zeros(n, dtype=torch.int64, device=DEV), table=i32(batch, 12),
             lens=i32(batch), q=f32(batch, heads * dim), pq=torch.zeros(n, heads * dim, dtype=torch.float16, device=DEV), cu=i32(3),
             z=f32(rows, vocab), t=f32(rows), top_k=i32(rows), top_p=f32(rows), u=f32(rows))
    y = dict(back=torch.zeros(2, n, kv * dim, dtype=torch.float16, device=DEV), one=f32(batch, heads * dim), many=f32(n, heads * dim),
             token=i32(rows), logprob=f32(rows))
    p = lambda t: t.data_ptr()  # noqa: E731

    def step(s):
        cfi.paged_kv_store(cache, p(x["k"]), p(x["v"]), p(x["slots"]), n, stream=s)
        cfi.paged_kv_load(cache, p(x["slots"]), p(y["back"][0]), p(y["back"][1]), n, stream=s)
        cfi.packed_attention(p(x["pq"]), p(y["back"][0]), p(y["back"][1]), p(y["many"]), p(x["cu"]), p(x["cu"]), 2, n, n, heads, kv, dim, 0.125,
                             stream=s)
        cfi.paged_attention(cache, p(x["q"]), p(y["one"]), p(x["table"]), p(x["lens"]), batch, heads, 12, 0.125, stream=s)
        cfi.sample(p(x["z"]), p(x["u"]), p(y["token"]), rows, vocab, p(x["t"]), p(x["top_k"]), p(x["top_p"]), 0, p(y["logprob"]), stream=s)

    def inputs(seed):
        g = torch.Generator(device=DEV)
        g.manual_seed(seed)
        r = np.random.default_rng(seed)
        for name in ("k", "v", "q", "pq"):
            x[name].copy_(torch.randn(x[name].shape, generator=g, device=DEV))
        x["z"].copy_(torch.randn(rows, vocab, generator=g, device=DEV) * 3)
        x["slots"].copy_(torch.randperm(pages * page, generator=g, device=DEV)[:n])
        x["table"].copy_(torch.from_numpy(r.integers(0, pages, (batch, 12))))
        x["lens"].copy_(torch.from_numpy(r.integers(0, 190, batch)))
        x["cu"].copy_(torch.tensor([0, int(r.integers(0, n)), n]))
        x["t"].copy_(torch.from_numpy(r.choice([0.0, 0.7, 1.0, 1.3], rows)))
        # few and many rows with a nucleus of the whole row: both sides of who takes them
        x["top_k"].copy_(torch.from_numpy(np.where(r.random(rows) < (0.1 if seed % 2 else 0.97), 0, 50)))
        x["top_p"].copy_(torch.from_numpy(r.choice([0.5, 0.95], rows)))
        x["u"].copy_(torch.rand(rows, generator=g, device=DEV))

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        inputs(0)
        step(s.cuda_stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=s):
            step(s.cuda_stream)
            step(s.cuda_stream)
    for seed in range(1, 7):
        inputs(seed)
        torch.cuda.synchronize()
        kept = pools.clone()
        step(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        want = {name: t.clone() for name, t in y.items()}
        pools.copy_(kept)
        for t in y.values():
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for name, t in y.items():
            assert torch.equal(t, want[name]), (seed, name)
        assert cfi.lib().cfi_device_error() == 0
