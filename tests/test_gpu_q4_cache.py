"""The Q4_1 cache (include/cfi_serve.h) against plain implementations in 64 bits: what is stored has to be equal, and the attention
over it near.

Bounds of the attention.  A score is summed as scale times whole numbers and minimum apart: its error is at most EPS_S times the sum of
the magnitudes of all those products, times the scale (EPS_S = 2^-20 covers 128 additions in 32 bits, whose rounding errors do
not all point one way, and operands held to 22 bits).  A softmax weight is then off by that much relative to itself, twice (numerator
and sum), plus 2^-20 for the exponential; an output by this times the largest magnitude of V's parts.  An f16 output adds 2^-11 of
itself."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import q41_pages as q41  # noqa: E402

pytestmark = pytest.mark.gpu
EPS_S = 2.0 ** -20
DEV = "cuda"
Q = cfi.Q4_1


def stream():
    return torch.cuda.current_stream().cuda_stream


def generator(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    return g


def garbage(pages, kv, page, dim, g):
    """A pool of random bytes: NaN, infinities and nonsense among its scales and minima."""
    n = pages * kv * q41.region_bytes(page, dim)
    return torch.randint(0, 256, (n,), generator=g, device=DEV, dtype=torch.int32).to(torch.uint8)


def rows_of(pool, pages, kv, page, dim, of_v):
    return q41.values(pool.cpu().numpy(), pages, kv, page, dim, of_v)


def hard_rows(n, width, dt, g):
    """Rows with what is hard to quantise among ordinary ones."""
    x = torch.randn(n, width, generator=g, device=DEV)
    x[:, ::7] = torch.round(x[:, ::7] * 8) / 8  # grids: quotients on the borders
    for i in range(0, n, 5):
        kind = i // 5 % 9
        b = x[i, 32:64]
        if kind == 0:
            b[:] = 0
        elif kind == 1:
            b[:] = -3.7
        elif kind == 2:
            b[:] = torch.arange(32, device=DEV) * 0.5 - 4  # steps of 15.5 / 15: every border
        elif kind == 3:
            b *= 1e-6  # f16 scales below its normal numbers
        elif kind == 4:
            b += 300
        elif kind == 5:
            b[:] = (torch.arange(32, device=DEV) % 31).float()  # 0 .. 30: all odd ones are ties
        elif kind == 6:
            b *= 1500
        elif kind == 7:
            b[3] = 60000.0
        elif dt == torch.float32:
            b *= 1e-30
    return x.to(dt)


# ---- the cache ----
@pytest.mark.parametrize("src", [cfi.T_F32, cfi.T_F16])
@pytest.mark.parametrize("kv,dim,page,tokens,pad", [(2, 64, 16, 1, 0), (1, 64, 256, 33, 8), (5, 128, 32, 77, 24), (8, 128, 64, 500, 0),
                                                    (3, 64, 16, 700, 16)])
def test_store_and_load(src, kv, dim, page, tokens, pad):
    g = generator(tokens * 7 + dim + src)
    pages = -(-tokens // page) + 3
    kp, vp = (garbage(pages, kv, page, dim, g) for _ in "kv")
    before = [rows_of(x, pages, kv, page, dim, i) for i, x in enumerate((kp, vp))]
    cache = cfi.paged_cache(Q, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    width, dt = kv * dim + pad, torch.float32 if src == cfi.T_F32 else torch.float16
    k, v = hard_rows(tokens, width, dt, g), hard_rows(tokens, width + 8, dt, g)
    slots = torch.randperm(pages * page, generator=g, device=DEV)[:tokens].contiguous()
    if tokens > 4:  # rows that go nowhere
        slots[1], slots[2], slots[3] = -1, pages * page, 1 << 40
    cfi.paged_kv_store(cache, k.data_ptr(), v.data_ptr(), slots.data_ptr(), tokens, src_type=src, k_stride=width, v_stride=width + 8,
                       stream=stream())
    out = torch.full((2, tokens, width), 7.0, dtype=torch.float16, device=DEV)
    cfi.paged_kv_load(cache, slots.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), tokens, k_stride=width, v_stride=width, stream=stream())
    torch.cuda.synchronize()
    sl = slots.cpu().numpy()
    ok = (sl >= 0) & (sl < pages * page)
    for i, (x, pool, was, back) in enumerate(((k, kp, before[0], out[0]), (v, vp, before[1], out[1]))):
        x = x[:, :kv * dim].reshape(tokens, kv, dim).double().cpu().numpy()
        want = q41.quantised(x)
        now = rows_of(pool, pages, kv, page, dim, i)
        np.testing.assert_array_equal(now[sl[ok]], want[ok])
        others = np.setdiff1d(np.arange(pages * page), sl[ok])
        np.testing.assert_array_equal(now[others], was[others])  # NaN equal here
        # and against the values themselves: half a step, and what f16 leaves of scale (15 of them) and minimum
        b, w = x[ok].reshape(-1, 32), want[ok].reshape(-1, 32)
        lo, step = b.min(1, keepdims=True), (b.max(1, keepdims=True) - b.min(1, keepdims=True)) / 15
        assert (np.abs(w - b) <= step * (0.5 + 1e-6 + 15 * 2.0 ** -11) + np.abs(lo) * 2.0 ** -11 + 16 * 2.0 ** -25).all()
        got = back[:, :kv * dim].reshape(tokens, kv, dim).cpu().numpy()
        with np.errstate(over="ignore"):
            np.testing.assert_array_equal(got[ok], want[ok].astype(np.float32).astype(np.float16))
        assert (got[~ok] == 0).all()
        assert (back[:, kv * dim:] == 7.0).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan"), 7e4, -7e4, 3e38])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_bad_block_stays_alone(bad, dim):
    """An infinity, a NaN, a minimum or a scale past f16 make NaN of their block."""
    kv, page, pages = 2, 16, 2
    kp, vp = (torch.zeros(cfi.paged_page_bytes(Q, page, kv, dim) * pages, dtype=torch.uint8, device=DEV) for _ in "kv")
    cache = cfi.paged_cache(Q, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    x = torch.randn(1, kv * dim, generator=generator(dim), device=DEV)
    y = x.clone()
    y[0, 40] = bad
    slots = torch.tensor([19], device=DEV)
    cfi.paged_kv_store(cache, y.data_ptr(), x.data_ptr(), slots.data_ptr(), 1, stream=stream())
    cfi.paged_kv_store(cache, y.data_ptr(), y.data_ptr(), torch.tensor([30], device=DEV).data_ptr(), 1, stream=stream())
    torch.cuda.synchronize()
    plain, spoilt = q41.quantised(x.cpu().numpy().reshape(kv, dim)), q41.quantised(y.cpu().numpy().reshape(kv, dim))
    assert np.isnan(spoilt.reshape(-1)[32:64]).all() == (bad != 7e4)  # 7e4 / 15 is a scale
    k, v = rows_of(kp, pages, kv, page, dim, False), rows_of(vp, pages, kv, page, dim, True)
    np.testing.assert_array_equal(k[19], spoilt)
    np.testing.assert_array_equal(v[19], plain)
    np.testing.assert_array_equal(k[30], spoilt)
    np.testing.assert_array_equal(v[30], spoilt)


def test_many_values_near_borders():
    """A million values within a few units of the last place of a border, in 32 bits, and scales at f16's borders."""
    g = generator(5)
    n, kv, dim, page = 4096, 2, 128, 64
    lo, step = torch.randn(n, kv * dim // 32, 1, generator=g, device=DEV, dtype=torch.float64), torch.rand(
        n, kv * dim // 32, 1, generator=g, device=DEV, dtype=torch.float64) + 0.01
    step[::2] = step[::2].half().double() * (1 + 2.0 ** -11)  # a scale between two f16 numbers
    at = torch.randint(1, 16, (n, kv * dim // 32, 32), generator=g, device=DEV).double() - 0.5
    at[..., 0], at[..., 1] = 0, 15
    x = (lo + at * step).float()
    bits = x.view(torch.int32)
    bits[..., 2:] += torch.randint(-3, 4, (n, kv * dim // 32, 30), generator=g, device=DEV, dtype=torch.int32)
    x = x.reshape(n, kv * dim)
    pages = n // page
    kp, vp = (torch.zeros(cfi.paged_page_bytes(Q, page, kv, dim) * pages, dtype=torch.uint8, device=DEV) for _ in "kv")
    cache = cfi.paged_cache(Q, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    slots = torch.arange(n, device=DEV)
    cfi.paged_kv_store(cache, x.data_ptr(), x.data_ptr(), slots.data_ptr(), n, stream=stream())
    torch.cuda.synchronize()
    want = q41.quantised(x.double().cpu().numpy().reshape(n, kv, dim))
    np.testing.assert_array_equal(rows_of(kp, pages, kv, page, dim, False), want)
    np.testing.assert_array_equal(rows_of(vp, pages, kv, page, dim, True), want)


# ---- one new token ----
def case(heads, kv, dim, page, lens, qt=cfi.T_F32, ot=cfi.T_F32, pad=0, seed=0, amp=1.5, offset=1.0, fill=None, small_v=1.0, scale=None):
    """A cache among garbage and a call over it; fill(k, v): changes the rows [position][kv * dim] that are stored."""
    g = generator(seed + heads * 31 + dim + page)
    need = [max(1, -(-n // page)) for n in lens]
    width, pages, batch = max(need) + 1, sum(need) + 2, len(lens)
    kp, vp = (garbage(pages, kv, page, dim, g) for _ in "kv")
    cache = cfi.paged_cache(Q, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    order = torch.randperm(pages, generator=g, device=DEV).cpu().numpy()
    table = np.full((batch, width), 0x7fffffff, dtype=np.int32)  # what no length reaches is nonsense
    slots, at = [], 0
    for b, n in enumerate(lens):
        own = order[at:at + need[b]]
        table[b, :need[b]] = own
        at += need[b]
        pos = np.arange(max(n, 0))
        slots.append(own[pos // page].astype(np.int64) * page + pos % page)
    total = sum(len(x) for x in slots)
    if total:
        k = torch.randn(total, kv * dim, generator=g, device=DEV) + offset * torch.randn(kv * dim, generator=g, device=DEV)
        v = torch.randn(total, kv * dim, generator=g, device=DEV) * small_v
        if fill:
            fill(k, v)
        sl = torch.from_numpy(np.concatenate(slots)).to(DEV)
        cfi.paged_kv_store(cache, k.data_ptr(), v.data_ptr(), sl.data_ptr(), total, stream=stream())
    q = torch.randn(batch, heads * dim + pad, generator=g, device=DEV) * amp
    q = q.half() if qt == cfi.T_F16 else q
    out = torch.full((batch, heads * dim + 2 * pad), 7.0, dtype=torch.float16 if ot == cfi.T_F16 else torch.float32, device=DEV)
    dt, dl = torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    scale = scale or 1.0 / math.sqrt(dim)

    def call(o=out):
        cfi.paged_attention(cache, q.data_ptr(), o.data_ptr(), dt.data_ptr(), dl.data_ptr(), batch, heads, width, scale, q_type=qt,
                            out_type=ot, q_stride=heads * dim + pad, out_stride=heads * dim + 2 * pad, stream=stream())

    def check(lengths=None):
        torch.cuda.synchronize()
        K, V = rows_of(kp, pages, kv, page, dim, False), rows_of(vp, pages, kv, page, dim, True)
        qq = q[:, :heads * dim].double().cpu().numpy().reshape(batch, heads, dim)
        got = out[:, :heads * dim].double().cpu().numpy().reshape(batch, heads, dim)
        n_g = heads // kv
        for b, n in enumerate(lengths or lens):
            if n <= 0:
                assert (got[b] == 0).all()
                continue
            for h in range(kv):
                kk, vv, mine = K[slots[b][:n], h], V[slots[b][:n], h], qq[b, h * n_g:(h + 1) * n_g]
                s = (mine @ kk.T) * scale
                p = np.exp(s - s.max(-1, keepdims=True))
                want = (p @ vv) / p.sum(-1, keepdims=True)
                # parts of a value: at most its block's minimum and 15 scales, whose magnitudes the block's ends bound
                ends = lambda x: np.repeat((np.abs(x.reshape(len(x), -1, 32)).max(2) * 3), 32, axis=1)  # noqa: E731
                mags = float((np.abs(mine) @ ends(kk).T).max() * scale)
                tol = (2 * EPS_S * mags + 2 * 2.0 ** -20) * ends(vv).max()
                if ot == cfi.T_F16:
                    tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
                err = np.abs(got[b, h * n_g:(h + 1) * n_g] - want)
                assert (err <= tol).all(), (b, h, n, float((err / tol).max()))
        assert (out[:, heads * dim:] == 7.0).all()

    call()
    keep = (kp, vp, q, dt, dl)
    return call, check, out, keep


SHAPES = [(14, 2, 64), (12, 2, 128), (32, 8, 128), (16, 16, 64), (9, 3, 64), (16, 1, 128), (40, 2, 64), (5, 5, 128)]


@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("page", [16, 64])
def test_attention(heads, kv, dim, page):
    case(heads, kv, dim, page, [1, 0, 15, 16, 17, 31, 32, 33, 63, 64, 65, 129, 500, 1023, -3, 2, 255])[1]()


@pytest.mark.parametrize("qt,ot,page,lens,pad", [
    (cfi.T_F16, cfi.T_F16, 32, [700], 8), (cfi.T_F16, cfi.T_F32, 128, [3, 4000], 16), (cfi.T_F32, cfi.T_F16, 256, [257, 1], 0),
    (cfi.T_F32, cfi.T_F32, 16, [20001], 0), (cfi.T_F16, cfi.T_F16, 64, [33333, 5, 12345], 0), (cfi.T_F16, cfi.T_F16, 16, [100] * 70, 0),
    (cfi.T_F32, cfi.T_F32, 16, [0, 0, 0], 0), (cfi.T_F32, cfi.T_F16, 32, [1] * 300, 0)])
@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128)])
def test_attention_types_and_lengths(qt, ot, page, lens, pad, heads, kv, dim):
    case(heads, kv, dim, page, lens, qt, ot, pad)[1]()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("amp,offset,small_v", [(1e-4, 1e3, 1.0), (400.0, 1.0, 1.0), (1.5, 1.0, 1e-4), (1.5, 0.0, 3000.0), (0.0, 1.0, 1.0)])
def test_attention_amplitudes(dim, amp, offset, small_v):
    """Small queries against large keys, sharp scores, values at the ends of f16, equal scores."""
    case(4 * 3, 3, dim, 16, [40, 1000, 5], amp=amp, offset=offset, small_v=small_v)[1]()


@pytest.mark.parametrize("dim", [64, 128])
def test_long_tail_of_small_weights(dim):
    """One key far above many equal ones: the sum of their small weights stays whole."""
    n = 20000

    def fill(k, v):
        k[:] = 0
        k[n // 2] = 1.0  # a block of one value: scale 0 and minimum 1
        v[:, ::2] += 1.0

    call, check, out, keep = case(2, 1, dim, 64, [n], fill=fill, amp=0.0, scale=1.0)
    keep[2][:] = 11.0 / dim  # scores 11 and 0: e^11 is three times the tail
    call()
    check()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("where", ["k", "v", "q"])
def test_what_a_nan_reaches(dim, where):
    """In K all of its kv head's query heads, in V the block's dims of them, in q its head; nothing behind the length."""
    def fill(k, v):
        if where == "k":
            k[70, 5] = float("nan")
        if where == "v":
            v[70, 33] = float("nan")  # block 1 of kv head 0

    heads, kv = 6, 2
    call, check, out, keep = case(heads, kv, dim, 16, [200], fill=fill)
    if where == "q":
        keep[2][0, 2 * dim + 1] = float("nan")
        call()
    torch.cuda.synchronize()
    bad = torch.isnan(out.view(heads, dim)).cpu().numpy()
    want = np.zeros((heads, dim), dtype=bool)
    if where == "k":
        want[:3] = True
    elif where == "v":
        want[:3, 32:64] = True
    else:
        want[2] = True
    np.testing.assert_array_equal(bad, want)
    if where != "q":
        keep[4].fill_(70)  # the length ends before it
        call()
        check([70])


def test_pages_outside_the_pool_and_lengths_past_the_table():
    """A page id outside is the nearest page inside, a length past the table is cut."""
    call, check, out, keep = case(4, 2, 64, 16, [64, 40])  # nine pages
    check()
    want = out.clone()
    table = keep[3]
    table[table == 0] = -5
    table[table == 8] = 1000
    call()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    call2, check2, out2, keep2 = case(4, 2, 64, 16, [48])
    want2 = out2.clone()
    keep2[3][0, 3] = keep2[3][0, 2]  # one more page in the table; the length passes it
    keep2[4][0] = 1 << 30
    call2()
    torch.cuda.synchronize()
    assert bool(torch.isfinite(out2).all()) and not torch.equal(out2, want2)


def test_same_result_again_and_in_company():
    """A sequence's result does not depend on the rest of the batch beyond rounding, and not at all on the run."""
    lens = [2500, 1, 300, 4096, 77]
    call, check, out, keep = case(12, 2, 128, 16, lens)
    check()
    first = out.clone()
    for _ in range(3):
        out.zero_()
        call()
        torch.cuda.synchronize()
        assert torch.equal(out[:, :12 * 128], first[:, :12 * 128])


def test_two_streams_and_a_captured_call():
    a = case(12, 2, 128, 16, [3000, 900, 11], seed=1)
    b = case(14, 2, 64, 32, [2000, 15000], seed=2)
    a[1](), b[1]()
    want = a[2].clone(), b[2].clone()
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for s in (s1, s2):
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        with torch.cuda.stream(s1):
            a[0]()
        with torch.cuda.stream(s2):
            b[0]()
    torch.cuda.synchronize()
    assert torch.equal(a[2], want[0]) and torch.equal(b[2], want[1])
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a[0]()  # the stream's workspace
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        a[0]()
    a[3][4].copy_(torch.tensor([100, 0, 9], dtype=torch.int32))  # other lengths, read when it runs
    graph.replay()
    a[1]([100, 0, 9])


@pytest.mark.parametrize("heads,kv,dim", [(6, 1, 128), (3, 1, 128), (14, 2, 64), (16, 16, 64)])
def test_scales_far_apart(heads, kv, dim):
    """Values whose scales lie 2^20 apart, in one tile, between positions and between blocks of a row, and a large one that comes late."""
    def fill(k, v):
        v[1::3] *= 2.0 ** -12
        v[:, 32:64] *= 2.0 ** -10
        v[-40] *= 2.0 ** 9

    case(heads, kv, dim, 16, [900], fill=fill)[1]()

    def constant(k, v):  # all scales 0 but one, subnormal ones
        v[:] = 0.25
        v[7, :32] = torch.arange(32, device=DEV) * 1e-6

    case(heads, kv, dim, 32, [300], fill=constant)[1]()


@pytest.mark.parametrize("heads,kv,dim", [(6, 1, 128), (3, 1, 128), (14, 2, 64), (16, 16, 64)])
def test_small_blocks_beside_large_ones(heads, kv, dim):
    """A block whose scales are 2^-17 of the others' keeps its own precision: bits of weight times scale end at 2^-39 of the largest,
    2^-22 of this block's, and a sum of a hundred of them that does not cancel is off by less than 2^-20 of the values.  (The block is
    kv head 0's: its query heads are looked at.)"""
    call, check, out, keep = case(heads, kv, dim, 16, [100], fill=lambda k, v: v[:, :32].mul_(2.0 ** -17).add_(2.0 ** -14), amp=0.2)
    check()
    V = rows_of(keep[1], 9, kv, 16, dim, True)
    K = rows_of(keep[0], 9, kv, 16, dim, False)
    table = keep[3][0].cpu().numpy()
    pos = np.arange(100)
    slots = table[pos // 16].astype(np.int64) * 16 + pos % 16
    q = keep[2].double().cpu().numpy().reshape(heads, dim)
    got = out.double().cpu().numpy().reshape(heads, dim)
    for h in range(heads // kv):
        s = K[slots, h * kv // heads] @ q[h] / math.sqrt(dim)
        p = np.exp(s - s.max())
        want = p @ V[slots, h * kv // heads][:, :32] / p.sum()
        mags = float((np.abs(q[h]) @ (np.abs(K[slots, h * kv // heads]) * 3).T).max() / math.sqrt(dim))
        assert (np.abs(got[h, :32] - want) <= (2 * EPS_S * mags + 3 * 2.0 ** -20) * 2.0 ** -14 * 2).all()


@pytest.mark.parametrize("heads,kv,dim,n", [(8, 8, 64, 33000), (12, 2, 64, 80000), (8, 8, 128, 20000), (16, 2, 128, 60000)])
def test_long_sums_keep_their_bits(heads, kv, dim, n):
    """An MMA's result is cut, not rounded, to 24 bits: sums that were kept in one over a sequence would be short by half a unit for each
    of its hundreds of tiles.  Positive values and equal weights: the mean error of a thousand outputs is that of one cut, half of 2^-23, and
    what rounding leaves of either sign."""
    call, check, out, keep = case(heads, kv, dim, 64, [n, n // 2, n], amp=0.0, fill=lambda k, v: v.add_(6.0))
    torch.cuda.synchronize()
    pages = keep[1].numel() // (kv * q41.region_bytes(64, dim))
    V = rows_of(keep[1], pages, kv, 64, dim, True)
    table = keep[3].cpu().numpy()
    rel = []
    for b, m in enumerate((n, n // 2, n)):
        pos = np.arange(m)
        want = V[table[b][pos // 64].astype(np.int64) * 64 + pos % 64].mean(0)  # [kv, dim]
        got = out[b].double().cpu().numpy().reshape(kv, heads // kv, dim)
        rel.append(got / want[:, None] - 1)
    rel = np.concatenate([x.reshape(-1) for x in rel])
    assert abs(rel.mean()) <= 2.0 ** -23 and np.abs(rel).max() <= 2.0 ** -20, (rel.mean() * 2 ** 23, np.abs(rel).max() * 2 ** 23)


@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("amp,offset", [(1.5, 1.0), (0.3, 4.0)])
def test_as_near_as_32_bits(heads, kv, dim, amp, offset):
    """Off from 64 bits by no more than twelve times what the formula on the cached values is in torch's 32 bits.  Operands of 22 bits are
    off by up to four units of the 24th; and the kernel sums a value's parts, scale times whole number and minimum, apart: between -a and
    a these are up to 2 a and a, three times the value's bound, so that what is rounded is up to three times as large."""
    lens = [672, 1500, 77]
    call, check, out, keep = case(heads, kv, dim, 16, lens, amp=amp, offset=offset, seed=9)
    torch.cuda.synchronize()
    pages = keep[1].numel() // (kv * q41.region_bytes(16, dim))
    K, V = (torch.from_numpy(rows_of(keep[i], pages, kv, 16, dim, i == 1)).to(DEV) for i in range(2))
    table = keep[3].cpu().numpy()
    mine, plain, size = 0.0, 0.0, 0.0
    for b, n in enumerate(lens):
        pos = np.arange(n)
        at = torch.from_numpy(table[b][pos // 16].astype(np.int64) * 16 + pos % 16).to(DEV)
        k, v = K[at].repeat_interleave(heads // kv, 1).transpose(0, 1), V[at].repeat_interleave(heads // kv, 1).transpose(0, 1)
        q = keep[2][b].view(heads, 1, dim)

        def formula(t):
            s = (q.to(t) @ k.to(t).transpose(1, 2)) * (1 / math.sqrt(dim))
            p = torch.exp(s - s.amax(-1, keepdim=True))
            return ((p @ v.to(t)) / p.sum(-1, keepdim=True))[:, 0].double()

        want = formula(torch.float64)
        mine += float((out[b].view(heads, dim).double() - want).pow(2).sum())
        plain += float((formula(torch.float32) - want).pow(2).sum())
        size += float(want.pow(2).sum())
    assert math.sqrt(mine) <= 12 * math.sqrt(plain) + 2.0 ** -24 * math.sqrt(size), (math.sqrt(mine / size), math.sqrt(plain / size))


def test_pools_past_31_bits():
    """Pages at the end of pools of 2.3 GB: rows stored, normed into them, read back and attended to."""
    kv, dim, page, pages, n = 8, 128, 256, 14200, 300
    size = cfi.paged_page_bytes(Q, page, kv, dim) * pages
    assert size > 2 ** 31
    kp, vp = (torch.empty(size, dtype=torch.uint8, device=DEV) for _ in "kv")
    cache = cfi.paged_cache(Q, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    g = generator(3)
    k, v = torch.randn(n, kv * dim, generator=g, device=DEV), torch.randn(n, kv * dim, generator=g, device=DEV)
    table = torch.tensor([[pages - 1, pages - 7]], dtype=torch.int32, device=DEV)
    pos = torch.arange(n, device=DEV)
    slots = (table[0].long()[pos // page] * page + pos % page).contiguous()
    cfi.paged_kv_store(cache, k.data_ptr(), v.data_ptr(), slots.data_ptr(), n, stream=stream())
    rows = torch.empty(2, n, kv * dim, dtype=torch.float16, device=DEV)
    cfi.paged_kv_load(cache, slots.data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), n, stream=stream())
    q, out, lens = torch.randn(1, kv * dim, generator=g, device=DEV), torch.empty(1, kv * dim, device=DEV), torch.tensor([n], dtype=torch.int32, device=DEV)
    cfi.paged_attention(cache, q.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(), 1, kv, 2, 0.1, stream=stream())
    torch.cuda.synchronize()
    K, V = (torch.from_numpy(q41.quantised(x.double().cpu().numpy().reshape(n, kv, dim))).to(DEV) for x in (k, v))
    assert torch.equal(rows[0].view(n, kv, dim), K.float().half()) and torch.equal(rows[1].view(n, kv, dim), V.float().half())
    p = torch.softmax(torch.einsum("hd,nhd->hn", q.double().view(kv, dim), K) * 0.1, -1)
    want = torch.einsum("hn,nhd->hd", p, V)
    assert float((out.view(kv, dim) - want).abs().max()) <= 1e-4  # 2^-13: a wrong row is off by tenths
    kp[-1 << 20:] = 0
    made = torch.empty(n, kv * dim, device=DEV)
    cfi.norm_rope(cfi.norm_rope_rows(k.data_ptr(), made.data_ptr(), 0, n, kv, dim, k=k.data_ptr(), v=v.data_ptr(), n_kv_head=kv, n_rot=0,
                                     slots=slots.data_ptr()), cache, stream=stream())
    cfi.paged_kv_load(cache, slots.data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), n, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(rows[0].view(n, kv, dim), K.float().half()) and torch.equal(rows[1].view(n, kv, dim), V.float().half())
    assert torch.equal(made, k)
