"""Serving operators (include/cfi_serve.h) where a bad value lies beside good ones, where values meet borders, angles to their bound, and
in other company, against 64 bits and more.

Bounds of the attention, as in test_gpu_q4_cache.py: a score is off by EPS_S = 2^-20 of the sum of the magnitudes that are added for it, a
weight by twice that and 2^-20, an output by this times the largest magnitude of V's parts."""
import math
from decimal import Decimal, localcontext
from fractions import Fraction

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import q41_pages as q41  # noqa: E402
import test_gpu_q4_cache as q4  # noqa: E402

pytestmark = pytest.mark.gpu
EPS_S = 2.0 ** -20
DEV = "cuda"


def stream():
    return torch.cuda.current_stream().cuda_stream


def q8_values(pool, pages, kv, page, dim):
    """Every slot of a Q8_0 pool in 64 bits: [slot, head, dim]."""
    x = pool.cpu().numpy().reshape(pages, kv, page * dim // 16 * 17)
    q = x[..., :page * dim].view(np.int8).reshape(pages, kv, page, dim).astype(np.float64)
    d = np.ascontiguousarray(x[..., page * dim:]).view(np.float16).astype(np.float64).reshape(pages, kv, page, dim // 32)
    with np.errstate(invalid="ignore"):
        v = q * np.repeat(d, 32, axis=3)
    return v.transpose(0, 2, 1, 3).reshape(pages * page, kv, dim)


# ---- what a bad block of V leaves the other dims ----
@pytest.mark.parametrize("ty", [cfi.Q4_1, cfi.Q8_0])
@pytest.mark.parametrize("heads,kv,dim,blocks", [(3, 1, 64, [1]), (16, 2, 64, [0]), (6, 2, 128, [1]), (6, 2, 128, [0, 1]),
                                                 (7, 1, 128, [0, 1, 3]), (12, 2, 128, [2, 3])])
@pytest.mark.parametrize("at", [0, 70])
@pytest.mark.parametrize("bad", [float("nan"), 1e7])
def test_bad_blocks_of_v_cost_the_other_dims_nothing(ty, heads, kv, dim, blocks, at, bad):
    """Ordinary values of 1e-4 beside blocks whose scales are not finite (1e7 / 127 passes f16, and is an infinity in Q8_0's pages):
    the dims of other blocks are as near to the formula as without it.  (Small queries: the scores' part of the bound is small too.)"""
    page, lens = 16, [80, 3000]
    g = torch.Generator(device=DEV)
    g.manual_seed(heads + dim + at)
    pages = sum(-(-n // page) for n in lens)
    n = cfi.paged_page_bytes(ty, page, kv, dim) * pages
    pools = torch.zeros(2, n, dtype=torch.uint8, device=DEV)
    cache = cfi.paged_cache(ty, pools[0].data_ptr(), pools[1].data_ptr(), pages, page, kv, dim)
    width = max(-(-n // page) for n in lens)
    order = torch.randperm(pages, generator=g, device=DEV)
    table = torch.zeros(2, width, dtype=torch.int32, device=DEV)
    own = (order[:-(-lens[0] // page)], order[-(-lens[0] // page):])
    slots = []
    for b in range(2):
        table[b, :len(own[b])] = own[b]
        pos = torch.arange(lens[b], device=DEV)
        slots.append(own[b][pos // page] * page + pos % page)
    k, v = (torch.randn(sum(lens), kv * dim, generator=g, device=DEV) for _ in "kv")
    v *= 1e-4
    for i in blocks:  # of kv head 0, of both sequences
        v[at, 32 * i + 5] = v[80 + at, 32 * i + 5] = bad
    all_slots = torch.cat(slots).contiguous()
    cfi.paged_kv_store(cache, k.data_ptr(), v.data_ptr(), all_slots.data_ptr(), sum(lens), stream=stream())
    q = torch.randn(2, heads * dim, generator=g, device=DEV) * 0.02
    out, dl = torch.empty(2, heads * dim, device=DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    scale = 1 / math.sqrt(dim)
    cfi.paged_attention(cache, q.data_ptr(), out.data_ptr(), table.data_ptr(), dl.data_ptr(), 2, heads, width, scale, stream=stream())
    torch.cuda.synchronize()
    if ty == cfi.Q4_1:
        K, V = (q41.values(pools[i].cpu().numpy(), pages, kv, page, dim, i == 1) for i in range(2))
    else:
        K, V = (q8_values(pools[i], pages, kv, page, dim) for i in range(2))
    got, qq = out.double().cpu().numpy().reshape(2, heads, dim), q.double().cpu().numpy().reshape(2, heads, dim)
    spoilt = np.concatenate([np.arange(32 * i, 32 * i + 32) for i in blocks])
    clean = np.setdiff1d(np.arange(dim), spoilt)
    for b in range(2):
        sl = slots[b].cpu().numpy()
        for h in range(heads):
            kk, vv = K[sl, h * kv // heads], V[sl, h * kv // heads]
            dims = clean if h * kv // heads == 0 else np.arange(dim)
            assert np.isfinite(got[b, h, spoilt]).any() == (h * kv // heads != 0)
            s = kk @ qq[b, h] * scale
            p = np.exp(s - s.max())
            want = p @ vv[:, dims] / p.sum()
            ends = lambda x: np.repeat(np.abs(x.reshape(len(x), -1, 32)).max(2) * 3, 32, axis=1)  # noqa: E731
            mags = float((np.abs(qq[b, h]) @ ends(kk).T).max() * scale)
            tol = (2 * EPS_S * mags + 2 * 2.0 ** -20) * 3 * np.abs(vv[:, dims]).max()
            err = np.abs(got[b, h][dims] - want).max()
            assert err <= tol, (b, h, err / tol)


# ---- Q4_1 values on borders, beside a minimum far below them ----
def exactly(block):
    """Scale (f16), minimum (f16) and whole numbers of a block, from fractions."""
    x = [Fraction(float(v)) for v in block]
    lo, wide = min(x), max(x) - min(x)
    exact = wide / 15
    if abs(lo) >= 65520 or exact >= 65520:  # past f16
        return math.nan, math.nan, [0] * 32
    near = np.float16(float(exact))
    around = [np.nextafter(near, np.float16(-np.inf)), near, np.nextafter(near, np.float16(np.inf))]
    d = min(around, key=lambda c: (abs(Fraction(float(c)) - exact), int(np.float16(c).view(np.uint16)) & 1))
    return float(d), float(np.float16(block.min())), [int((v - lo) * 15 / wide + Fraction(1, 2)) if wide else 0 for v in x]


def test_scales_and_values_on_borders():
    """Scale and quotients are rounded from their exact values: a minimum that only just is not zero decides where the rest lies on a border,
    with scales among f16's normal numbers, below them and large."""
    blocks = []
    for low in (2.0 ** -100, 2.0 ** -60, 2.0 ** -40, 2.0 ** -30, 1e-38):
        for sign in (-1, 0, 1):
            for step in (1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 2.0 ** -15, 2.0 ** -17 * 1.5, 2.0 ** -20, 2.0 ** -24 * 2.5, 700.0 + 0.25, 61000.0, 5.0):
                b = [(i + 0.5) * step for i in range(15)] + [i * step for i in range(1, 16)] + [15 * step]
                blocks.append([sign * low] + b)
    x = np.array(blocks, dtype=np.float32)
    assert x.shape[1] == 32
    rng = np.random.default_rng(1)
    x = np.concatenate([x, -x, rng.permuted(x, axis=1)])
    x = np.concatenate([x, np.zeros((-len(x) % 4, 32), dtype=np.float32)])
    n, page = len(x) // 4, 16
    pages = -(-n // page)
    rows = torch.from_numpy(x.reshape(n, 128)).to(DEV)
    pools = torch.zeros(2, cfi.paged_page_bytes(cfi.Q4_1, page, 1, 128) * pages, dtype=torch.uint8, device=DEV)
    cache = cfi.paged_cache(cfi.Q4_1, pools[0].data_ptr(), pools[1].data_ptr(), pages, page, 1, 128)
    slots = torch.arange(n, device=DEV)
    cfi.paged_kv_store(cache, rows.data_ptr(), rows.data_ptr(), slots.data_ptr(), n, stream=stream())
    torch.cuda.synchronize()
    want = np.array([[q * d + m for q in qs] for d, m, qs in map(exactly, x)]).reshape(n, 128)
    for i in range(2):
        got = q41.values(pools[i].cpu().numpy(), pages, 1, page, 128, i == 1)[:n, 0]
        np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("dt", [torch.float32, torch.float16])
def test_whole_numbers_of_blocks_of_all_sizes(dt):
    """From f32's least numbers to where a scale passes f16: a block's whole numbers are the exact quotients', values next to borders and blocks
    of one value among them, and scale and minimum the exact ones'."""
    rng = np.random.default_rng(3)
    blocks = []
    for k in range(-148, 17) if dt == torch.float32 else range(-24, 12):
        for offset in (0.0, 1.0, -7.3):
            step = np.ldexp(1 + rng.random(), k)
            at = rng.integers(1, 16, 32) - 0.5
            at[:2] = 0, 15
            b = ((at + offset) * step).astype(np.float32)
            b[2:] = np.where(rng.random(30) < 0.5, b[2:], np.nextafter(b[2:], np.float32(rng.choice([-1, 1]) * 1e38)))
            blocks.append(b)
        blocks.append(np.full(32, np.float32(step)))
    x = np.array(blocks, dtype=np.float32)
    x = x.astype(np.float16).astype(np.float32) if dt == torch.float16 else x
    x = np.concatenate([x, np.zeros((-len(x) % 4, 32), dtype=np.float32)])
    n, page = len(x) // 4, 16
    pages = -(-n // page)
    rows = torch.from_numpy(x.reshape(n, 128)).to(DEV).to(dt)
    pools = torch.zeros(2, cfi.paged_page_bytes(cfi.Q4_1, page, 1, 128) * pages, dtype=torch.uint8, device=DEV)
    cache = cfi.paged_cache(cfi.Q4_1, pools[0].data_ptr(), pools[1].data_ptr(), pages, page, 1, 128)
    slots = torch.arange(n, device=DEV)
    cfi.paged_kv_store(cache, rows.data_ptr(), rows.data_ptr(), slots.data_ptr(), n, src_type=int(dt == torch.float16), stream=stream())
    torch.cuda.synchronize()
    parts = [exactly(b) for b in x]
    q = np.array([p[2] for p in parts]).reshape(n, 128)
    want = np.array([[i * d + m for i in qs] for d, m, qs in parts]).reshape(n, 128)
    for i in range(2):
        np.testing.assert_array_equal(q41.values(pools[i].cpu().numpy(), pages, 1, page, 128, i == 1)[:n, 0], want)
        bare = pools[i].cpu().numpy().reshape(pages, 1280).copy()  # scales of 1 and minima of 0
        bare[:, 1024:].view(np.uint16).reshape(pages, 16, 2, 4)[:] = np.array([0x3c00, 0], dtype=np.uint16)[None, None, :, None]
        np.testing.assert_array_equal(q41.values(bare.reshape(-1), pages, 1, page, 128, i == 1)[:n, 0], q)


# ---- angles ----
PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459230781640628620899862803")


@pytest.mark.parametrize("base,scale,lo,hi", [(1e4, 1.0, 1.0, 4.0), (1e4, 8.0, 1.0, 4.0), (1e4, 1.0, 0.05, 0.2), (5e5, 8.0, 0.05, 0.2),
                                              (1e4, -1.0, 0.5, 1.0), (1e6, 1.0, None, None), (1e4, 8.0, None, None), (0.5, 1.0, None, None),
                                              (1e4, 300.0, None, None), (1.01, 1.0, None, None)])
def test_angles_to_their_bound(base, scale, lo, hi):
    """Pairs of (1, 0) come out as cosine and sine, which are off by a unit of the last place, 2^-23 of themselves: together by 2^-23 rad."""
    g = torch.Generator(device=DEV)
    g.manual_seed(int(base) + int(scale))
    n, dim = 60, 128
    far = (1 << 31) - 1
    pos = torch.randint(1 << 23, 1 << 24, (n,), generator=g, device=DEV).to(torch.int32)
    pos[::3] = torch.randint(far // 2, far, (n // 3,), generator=g, device=DEV).to(torch.int32)
    pos[:5] = torch.tensor([0, 1, far, -far, 4097])
    rows = torch.zeros(n, dim, device=DEV)
    rows[:, :dim // 2] = 1.0
    ff = (lo + (hi - lo) * torch.rand(dim // 2, generator=g, device=DEV)).float() if lo else None
    out = torch.empty(n, dim, device=DEV)
    cfi.norm_rope(cfi.norm_rope_rows(rows.data_ptr(), out.data_ptr(), pos.data_ptr(), n, 1, dim, freq_base=base, freq_scale=scale,
                                     freq_factors=ff.data_ptr() if lo else 0), stream=stream())
    torch.cuda.synchronize()
    got, pos = out.double().cpu().numpy(), pos.tolist()
    factors = ff.double().cpu().tolist() if lo else [1.0] * (dim // 2)
    worst = 0.0
    with localcontext() as c:
        c.prec = 60
        b, s = Decimal(float(np.float32(base))), Decimal(float(np.float32(scale)))
        for i in range(dim // 2):
            rate = s * (b.ln() * Decimal(-2 * i) / dim).exp() / Decimal(factors[i])
            for t in range(n):
                angle = rate * pos[t]
                a = float(angle - (angle / (2 * PI)).to_integral_value() * 2 * PI)
                err = abs(got[t, i + dim // 2] * math.cos(a) - got[t, i] * math.sin(a))
                bound = 1e-7 + abs(pos[t]) * max(1.0, abs(float(rate))) * 2.0 ** (-45 if lo else -53)
                worst = max(worst, err / (bound + 2.0 ** -23))
    assert worst <= 1.0, worst


# ---- what earlier tests leave open ----
@pytest.mark.parametrize("heads,kv,dim", [(12, 2, 128), (14, 2, 64), (8, 2, 128)])
def test_a_sequence_alone_and_in_company(heads, kv, dim):
    """Q4_1: the batch cuts a sequence in other places than it alone is cut; both results are within the bound of the formula."""
    lens = [2500, 1, 300, 4096, 77]
    call, check, out, keep = q4.case(heads, kv, dim, 16, lens)
    check()
    kp, vp, q, table, dl = keep
    pages, width = kp.numel() // cfi.paged_page_bytes(cfi.Q4_1, 16, kv, dim), table.shape[1]
    cache = cfi.paged_cache(cfi.Q4_1, kp.data_ptr(), vp.data_ptr(), pages, 16, kv, dim)
    K, V = (q41.values(x.cpu().numpy(), pages, kv, 16, dim, i) for i, x in enumerate((kp, vp)))
    alone = torch.empty(1, heads * dim, device=DEV)
    for b, n in enumerate(lens):
        own, cut = table[b:b + 1].contiguous(), dl[b:b + 1].clone()
        for w in (width, -(-n // 16)):
            t = own[:, :w].contiguous()
            alone.fill_(7.0)
            cfi.paged_attention(cache, q[b:b + 1].contiguous().data_ptr(), alone.data_ptr(), t.data_ptr(), cut.data_ptr(), 1, heads, w,
                                1 / math.sqrt(dim), stream=stream())
            torch.cuda.synchronize()
            pos = np.arange(n)
            sl = own[0].cpu().numpy()[pos // 16].astype(np.int64) * 16 + pos % 16
            ends = lambda x: np.repeat(np.abs(x.reshape(len(x), kv, -1, 32)).max(3) * 3, 32, axis=2)  # noqa: E731
            qq = np.abs(q[b].double().cpu().numpy().reshape(kv, -1, dim))
            mags = float(np.einsum("hgd,nhd->hgn", qq, ends(K[sl])).max()) / math.sqrt(dim)
            tol = 2 * (2 * EPS_S * mags + 2 * 2.0 ** -20) * ends(V[sl]).max()
            assert float((alone[0] - out[b]).abs().max()) <= tol


@pytest.mark.parametrize("heads,kv,dim", [(14, 2, 64), (12, 2, 128), (32, 8, 128), (9, 3, 64)])
def test_blocks_without_offsets_are_as_near_as_32_bits(heads, kv, dim):
    """Q4_1 blocks whose minimum is zero have one part only: off from 64 bits by no more than four times what torch's 32 bits are, since
    operands of 22 bits are off by up to four units of the 24th."""
    def fill(k, v):
        for x in (k, v):
            x.abs_()
            x[:, ::32] = 0

    lens = [672, 1500, 77]
    call, check, out, keep = q4.case(heads, kv, dim, 16, lens, offset=0.0, fill=fill, seed=9)
    check()
    pages = keep[1].numel() // (kv * q41.region_bytes(16, dim))
    K, V = (torch.from_numpy(q41.values(keep[i].cpu().numpy(), pages, kv, 16, dim, i == 1)).to(DEV) for i in range(2))
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
    assert math.sqrt(mine) <= 4 * math.sqrt(plain) + 2.0 ** -24 * math.sqrt(size), (math.sqrt(mine / size), math.sqrt(plain / size))


@pytest.mark.parametrize("ty", [cfi.T_F16, cfi.Q8_0, cfi.Q4_1])
def test_rows_in_the_cache_do_not_depend_on_what_was_there(ty):
    """cfi_norm_rope writes whole rows: over garbage, over zeros and without rows out beside them the cached values are the same, and slots
    that are not named keep theirs."""
    from test_gpu_norm_rope import make
    heads, kv, dim, page, tokens = 12, 2, 128, 16, 90
    x = make(tokens, heads, kv, dim)
    pages = 8
    n = cfi.paged_page_bytes(ty, page, kv, dim) * pages
    slots = torch.randperm(pages * page, device=DEV)[:tokens].contiguous()
    others = torch.tensor(np.setdiff1d(np.arange(pages * page), slots.cpu().numpy()), device=DEV)
    back = []
    garbage = torch.randint(0, 256, (2, n), device=DEV, dtype=torch.int32).to(torch.uint8)
    for pools, kw in ((garbage, {}), (torch.zeros_like(garbage), {}), (garbage.clone(), dict(k_out=0, v_out=0))):
        pools = pools.clone()
        cache = cfi.paged_cache(ty, pools[0].data_ptr(), pools[1].data_ptr(), pages, page, kv, dim)

        def read(at):
            rows = torch.empty(2, len(at), kv * dim, dtype=torch.float16, device=DEV)
            cfi.paged_kv_load(cache, at.data_ptr(), rows[0].data_ptr(), rows[1].data_ptr(), len(at), stream=stream())
            torch.cuda.synchronize()
            return rows.view(torch.int16)

        before = read(others)
        cfi.norm_rope(x["describe"](slots=slots.data_ptr(), **kw), cache, stream=stream())
        back.append(read(slots))
        assert torch.equal(read(others), before)
    assert torch.equal(back[0], back[1]) and torch.equal(back[0], back[2])


# ---- the driver after a call that failed ----
@pytest.mark.parametrize("tables", ["host", "device"])
def test_a_server_goes_on_after_a_failed_call(monkeypatch, tables):
    """A prompt and a step that raise in the second layer, and again: the same bits as if they had not."""
    import decode
    import serve
    ctx = cfi.Ctx(0)
    cfg = decode.Config(hidden=256, layers=2, n_head=4, n_kv_head=2, head_dim=64, ffn=512, vocab=1024, prompt=8, n_ctx=16)
    m = decode.DecodeModel(torch, ctx, "cuda", cfg, fused=1)
    out = []
    for broken in (False, True):
        fail = []

        def once(real, name):
            def call(*a, **k):
                if fail and fail[0] == name:
                    fail.pop(0)
                    if not fail or fail[0] != name:
                        raise MemoryError(name)
                return real(*a, **k)
            return call

        for name in ("paged_attention", "packed_attention"):
            monkeypatch.setattr(cfi, name, once(getattr(cfi, name), name))
        s = serve.Server(torch, ctx, m, cfi.Q4_1, 16, 20, tables=tables)
        a, b = serve.Sequence([i * 7 % 1024 for i in range(48)]), serve.Sequence([5, 6, 7])
        got = []
        for call, name in ((lambda: s.prefill([a, b]), "packed_attention"), (lambda: s.step([a, b]), "paged_attention"),
                           (lambda: s.step([b, a]), "paged_attention")):
            if broken:
                fail[:] = [name] * 2  # the second layer's
                with pytest.raises(MemoryError):
                    call()
            got.append(call())
            a.tokens.append(11), b.tokens.append(12)
        if tables == "device":
            assert int(s.state.status) == 0 and s.state.cached[[a.row, b.row]].tolist() == [50, 5]
        s.cut([a], [20])
        s.release(a), s.release(b)
        assert (s.n_free if tables == "device" else len(s.free)) == 20
        monkeypatch.undo()
        out.append(got)
    assert all(torch.equal(x, y) for x, y in zip(*out))
    ctx.close()
