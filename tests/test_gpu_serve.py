"""The serving operators (include/cfi_serve.h) against plain implementations in 64 bits.

Bounds.  Scores are sums of D products: their error is at most EPS_S times the sum of the products'
magnitudes times the scale (EPS_S = 2^-20 covers 128 additions in 32 bits, whose rounding errors do not all
point one way, and operands held to 22 bits).  A softmax weight is then off by that much relative to
itself, twice (numerator and sum), plus 2^-20 for the exponential; an output by this times max|V|.  Weights
rounded to f16 (packed prompts) add 2^-11, an f16 output 2^-11 of itself."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402

pytestmark = pytest.mark.gpu
EPS_S = 2.0 ** -20
DEV = "cuda"


def stream():
    return torch.cuda.current_stream().cuda_stream


def region_bytes(ty, page, dim):
    return page * dim * 2 if ty == cfi.T_F16 else page * (dim + dim // 16)


def garbage_pool(ty, pages, kv, page, dim, gen):
    """A pool of random bytes: NaN, infinities and nonsense scales among them."""
    n = pages * kv * region_bytes(ty, page, dim)
    return torch.randint(0, 256, (n,), generator=gen, device=DEV, dtype=torch.int32).to(torch.uint8)


def pool_rows(pool, ty, pages, kv, page, dim):
    """Every slot of a pool in 64 bits: [slot, head, dim]."""
    r = pool.view(pages * kv, region_bytes(ty, page, dim)).cpu().numpy()
    if ty == cfi.T_F16:
        x = r.view(np.float16).astype(np.float64)
    else:
        q = np.ascontiguousarray(r[:, :page * dim]).view(np.int8).astype(np.float64)
        d = np.ascontiguousarray(r[:, page * dim:]).view(np.float16).astype(np.float64)
        x = q * np.repeat(d, 32, axis=1)
    return x.reshape(pages, kv, page, dim).transpose(0, 2, 1, 3).reshape(pages * page, kv, dim)


def quantised(x):
    """Q8_0 values of f32 rows by the definition, in 32-bit arithmetic: q and f16 scales."""
    b = x.astype(np.float32).reshape(-1, 32)
    d = (np.abs(b).max(1, keepdims=True) / np.float32(127)).astype(np.float32)
    inv = np.where(d > 0, np.float32(1) / np.where(d > 0, d, 1), 0).astype(np.float32)
    q = np.clip(np.rint((b * inv).astype(np.float32)), -127, 127)
    return (q * d.astype(np.float16).astype(np.float64)).reshape(x.shape)


# ---- the cache ----
@pytest.mark.parametrize("ty", [cfi.T_F16, cfi.Q8_0])
@pytest.mark.parametrize("src", [cfi.T_F32, cfi.T_F16])
@pytest.mark.parametrize("kv,dim,page,tokens,pad", [(2, 64, 16, 1, 0), (1, 64, 256, 33, 8), (5, 128, 32, 77, 24), (8, 128, 64, 500, 0)])
def test_cache_store_and_load(ty, src, kv, dim, page, tokens, pad):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(tokens * 7 + dim + ty + src)
    pages = -(-tokens // page) + 3
    kp, vp = (garbage_pool(ty, pages, kv, page, dim, gen) for _ in "kv")
    before = [pool_rows(x, ty, pages, kv, page, dim) for x in (kp, vp)]
    cache = cfi.paged_cache(ty, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    width = kv * dim + pad
    dt = torch.float32 if src == cfi.T_F32 else torch.float16
    k = torch.randn(tokens, width, generator=gen, device=DEV).to(dt)
    v = (torch.randn(tokens, width + 8, generator=gen, device=DEV) * 30).to(dt)
    k[0, :32] = 0  # a block of zeros
    slots = torch.randperm(pages * page, generator=gen, device=DEV)[:tokens].contiguous()
    if tokens > 4:  # rows that go nowhere
        slots[1], slots[2], slots[3] = -1, pages * page, 1 << 40
    cfi.paged_kv_store(cache, k.data_ptr(), v.data_ptr(), slots.data_ptr(), tokens, src_type=src, k_stride=width, v_stride=width + 8,
                       stream=stream())
    out = torch.full((2, tokens, width), 7.0, dtype=torch.float16, device=DEV)
    cfi.paged_kv_load(cache, slots.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), tokens, k_stride=width, v_stride=width, stream=stream())
    torch.cuda.synchronize()
    sl = slots.cpu().numpy()
    ok = (sl >= 0) & (sl < pages * page)
    for x, pool, was, back in ((k, kp, before[0], out[0]), (v, vp, before[1], out[1])):
        x = x[:, :kv * dim].reshape(tokens, kv, dim).float().cpu().numpy()
        want = x.astype(np.float16).astype(np.float64) if ty == cfi.T_F16 else quantised(x)
        now = pool_rows(pool, ty, pages, kv, page, dim)
        np.testing.assert_array_equal(now[sl[ok]], want[ok])
        others = np.setdiff1d(np.arange(pages * page), sl[ok])
        np.testing.assert_array_equal(now[others], was[others])  # NaN equal here
        if ty == cfi.Q8_0:  # and against the values themselves: half a step, and the scale's rounding
            d = np.abs(x[ok]).reshape(-1, 32).max(1, keepdims=True) / 127.0
            assert (np.abs(want[ok] - x[ok]).reshape(-1, 32) <= d * (0.5 + 127 * 2.0 ** -11 + 1e-3) + 127 * 2.0 ** -25).all()
        got = back[:, :kv * dim].reshape(tokens, kv, dim).cpu().numpy()
        np.testing.assert_array_equal(got[ok], want[ok].astype(np.float16))
        assert (got[~ok] == 0).all()
        assert (back[:, kv * dim:] == 7.0).all()


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_cache_bad_block_stays_alone(bad):
    kv, dim, page, pages = 2, 64, 16, 2
    kp, vp = (torch.zeros(cfi.paged_page_bytes(cfi.Q8_0, page, kv, dim) * pages, dtype=torch.uint8, device=DEV) for _ in "kv")
    cache = cfi.paged_cache(cfi.Q8_0, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    x = torch.randn(1, kv * dim, device=DEV)
    y = x.clone()
    y[0, 40] = bad
    slots = torch.tensor([19], device=DEV)
    cfi.paged_kv_store(cache, y.data_ptr(), x.data_ptr(), slots.data_ptr(), 1, stream=stream())
    torch.cuda.synchronize()
    got = pool_rows(kp, cfi.Q8_0, pages, kv, page, dim)[19].reshape(-1)
    assert np.isnan(got[32:64]).all()
    want = quantised(x.cpu().numpy().astype(np.float64)).reshape(-1)
    keep = np.r_[0:32, 64:128]
    np.testing.assert_array_equal(got[keep], want[keep])


# ---- one new token ----
def attend(q, k, v, scale):
    s = (q @ k.T) * scale
    p = np.exp(s - s.max(-1, keepdims=True))
    return (p @ v) / p.sum(-1, keepdims=True)


def decode_case(ty, heads, kv, dim, page, lens, qt, ot, pad=0, seed=0, amp=1.5, garbage=True):
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + heads * 31 + dim + page + ty)
    need = [max(1, -(-n // page)) for n in lens]
    width, pages, batch = max(need) + 1, sum(need) + 2, len(lens)
    kp, vp = (garbage_pool(ty, pages, kv, page, dim, gen) if garbage else
              torch.zeros(pages * kv * region_bytes(ty, page, dim), dtype=torch.uint8, device=DEV) for _ in "kv")
    cache = cfi.paged_cache(ty, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    order = torch.randperm(pages, generator=gen, device=DEV).cpu().numpy()
    table = np.full((batch, width), 0x7fffffff, dtype=np.int32)  # what no length reaches is nonsense
    slots, at = [], 0
    for b, n in enumerate(lens):
        own = order[at:at + need[b]]
        table[b, :need[b]] = own
        at += need[b]
        pos = np.arange(n)
        slots.append(own[pos // page].astype(np.int64) * page + pos % page if n > 0 else np.zeros(0, np.int64))
    allslots = np.concatenate(slots)
    total = len(allslots)
    if total:
        k = torch.randn(total, kv * dim, generator=gen, device=DEV)
        v = torch.randn(total, kv * dim, generator=gen, device=DEV)
        sl = torch.from_numpy(allslots).to(DEV)
        cfi.paged_kv_store(cache, k.data_ptr(), v.data_ptr(), sl.data_ptr(), total, stream=stream())
    q = torch.randn(batch, heads * dim + pad, generator=gen, device=DEV) * amp
    q = q.half() if qt == cfi.T_F16 else q
    out = torch.full((batch, heads * dim + 2 * pad), 7.0, dtype=torch.float16 if ot == cfi.T_F16 else torch.float32, device=DEV)
    dt, dl = torch.from_numpy(table).to(DEV), torch.tensor(lens, dtype=torch.int32, device=DEV)
    scale = 1.0 / math.sqrt(dim)

    def call(o=out):
        cfi.paged_attention(cache, q.data_ptr(), o.data_ptr(), dt.data_ptr(), dl.data_ptr(), batch, heads, width, scale, q_type=qt,
                            out_type=ot, q_stride=heads * dim + pad, out_stride=heads * dim + 2 * pad, stream=stream())

    def check():
        torch.cuda.synchronize()
        K, V = pool_rows(kp, ty, pages, kv, page, dim), pool_rows(vp, ty, pages, kv, page, dim)
        Q = q[:, :heads * dim].double().cpu().numpy().reshape(batch, heads, dim)
        got = out[:, :heads * dim].double().cpu().numpy().reshape(batch, heads, dim)
        g = heads // kv
        for b, n in enumerate(lens):
            if n <= 0:
                assert (got[b] == 0).all()
                continue
            for h in range(kv):
                kk, vv, qq = K[slots[b], h], V[slots[b], h], Q[b, h * g:(h + 1) * g]
                want = attend(qq, kk, vv, scale)
                S = float((np.abs(qq) @ np.abs(kk).T).max() * scale)
                tol = (2 * EPS_S * S + 2 * 2.0 ** -20) * np.abs(vv).max()
                if ot == cfi.T_F16:
                    tol = tol + 2.0 ** -11 * np.abs(want) + 2.0 ** -25
                err = np.abs(got[b, h * g:(h + 1) * g] - want)
                assert (err <= tol).all(), (b, h, n, float((err / tol).max()))
        assert (out[:, heads * dim:] == 7.0).all()

    call()
    keep = (kp, vp, q, dt, dl)
    return call, check, out, keep


SHAPES = [(14, 2, 64), (12, 2, 128), (32, 8, 128), (16, 16, 64), (9, 3, 64), (16, 1, 128), (40, 2, 64), (5, 5, 128)]


@pytest.mark.parametrize("ty", [cfi.T_F16, cfi.Q8_0])
@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("page", [16, 64])
def test_paged_attention(ty, heads, kv, dim, page):
    lens = [1, 0, 15, 16, 17, 63, 64, 65, 129, 500, 1023, -3, 2, 255]
    decode_case(ty, heads, kv, dim, page, lens, cfi.T_F32, cfi.T_F32)[1]()


@pytest.mark.parametrize("ty,qt,ot,page,lens,pad", [
    (cfi.T_F16, cfi.T_F16, cfi.T_F16, 32, [700], 8), (cfi.Q8_0, cfi.T_F16, cfi.T_F32, 128, [3, 4000], 16),
    (cfi.T_F16, cfi.T_F32, cfi.T_F16, 256, [257, 1], 0), (cfi.Q8_0, cfi.T_F32, cfi.T_F32, 16, [20001], 0),
    (cfi.T_F16, cfi.T_F16, cfi.T_F32, 64, [33333, 5, 12345], 0), (cfi.Q8_0, cfi.T_F16, cfi.T_F16, 16, [100] * 70, 0)])
def test_paged_attention_types_and_lengths(ty, qt, ot, page, lens, pad):
    for heads, kv, dim in ((14, 2, 64), (12, 2, 128)):
        decode_case(ty, heads, kv, dim, page, lens, qt, ot, pad)[1]()


def test_paged_attention_large_scores():
    decode_case(cfi.T_F16, 14, 2, 64, 16, [1000, 37], cfi.T_F32, cfi.T_F32, amp=40.0)[1]()


def test_paged_attention_is_repeatable_and_graph_replayable():
    call, check, out, keep = decode_case(cfi.Q8_0, 12, 2, 128, 16, [9000, 1, 300], cfi.T_F32, cfi.T_F32)
    torch.cuda.synchronize()
    first = out.clone()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        call()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            call()
            call()
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, torch.where(first == 7.0, torch.zeros_like(first), first))


def test_paged_attention_bad_page_ids_stay_inside():
    """Nonsense ids in reach of a length: the result is of some pages of the pool, nothing is read outside."""
    kv, dim, page, pages = 2, 64, 16, 3
    kp, vp = (torch.zeros(pages * kv * page * dim, dtype=torch.float16, device=DEV) for _ in "kv")
    vp += 1.0
    cache = cfi.paged_cache(cfi.T_F16, kp.data_ptr(), vp.data_ptr(), pages, page, kv, dim)
    table = torch.tensor([[-5, 1 << 30, 2, -(1 << 31)]], dtype=torch.int32, device=DEV)
    lens = torch.tensor([1 << 30], dtype=torch.int32, device=DEV)  # past the table: cut to it
    q, out = torch.randn(1, 4 * dim, device=DEV), torch.zeros(1, 4 * dim, device=DEV)
    cfi.paged_attention(cache, q.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(), 1, 4, 4, 0.125, stream=stream())
    torch.cuda.synchronize()
    assert (out - 1.0).abs().max() <= 2.0 ** -20


# ---- packed prompts ----
def packed_case(heads, kv, dim, nq, nk, causal=True, ot=None, pad=0, seed=0, amp=1.5, poison=False):
    ot = cfi.T_F32 if ot is None else ot
    gen = torch.Generator(device=DEV)
    gen.manual_seed(seed + heads + dim + sum(nq))
    tq, tk = sum(nq), sum(nk)
    wq, wk = heads * dim, kv * dim
    q = (torch.randn(max(tq, 1), wq + pad, generator=gen, device=DEV) * amp).half()
    k = torch.randn(max(tk, 1), wk + pad, generator=gen, device=DEV).half()
    v = torch.randn(max(tk, 1), wk + 2 * pad, generator=gen, device=DEV).half()
    ck, cq = np.cumsum([0] + nk), np.cumsum([0] + nq)
    bad = None
    if poison:  # the second sequence's keys and values are all NaN and infinities
        bad = 1
        k[ck[1]:ck[2]] = float("nan")
        v[ck[1]:ck[2]] = float("inf")
    out = torch.full((max(tq, 1), wq + pad), 7.0, dtype=torch.float16 if ot == cfi.T_F16 else torch.float32, device=DEV)
    cu_q, cu_kv = (torch.from_numpy(c.astype(np.int32)).to(DEV) for c in (cq, ck))
    scale = 1.0 / math.sqrt(dim)
    cfi.packed_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu_q.data_ptr(), cu_kv.data_ptr(), len(nq), tq, tk,
                         heads, kv, dim, scale, causal=causal, out_type=ot, q_stride=wq + pad, k_stride=wk + pad,
                         v_stride=wk + 2 * pad, out_stride=wq + pad, stream=stream())
    torch.cuda.synchronize()
    assert cfi.lib().cfi_device_error() == 0
    g = heads // kv
    for s, (n, m) in enumerate(zip(nq, nk)):
        if s == bad or n == 0:
            continue
        Q = q[cq[s]:cq[s + 1], :wq].double().reshape(n, kv, g, dim).permute(1, 2, 0, 3)
        K = k[ck[s]:ck[s + 1], :wk].double().reshape(m, kv, dim).permute(1, 0, 2)[:, None]
        V = v[ck[s]:ck[s + 1], :wk].double().reshape(m, kv, dim).permute(1, 0, 2)[:, None]
        got = out[cq[s]:cq[s + 1], :wq].double().reshape(n, kv, g, dim).permute(1, 2, 0, 3)
        if m == 0:
            assert (got == 0).all()
            continue
        x = (Q @ K.transpose(2, 3)) * scale
        blind = torch.zeros(n, dtype=torch.bool, device=DEV)
        if causal:
            seen = torch.arange(m, device=DEV)[None] <= torch.arange(n, device=DEV)[:, None] + (m - n)
            x = x.masked_fill(~seen, -math.inf)
            blind = ~seen.any(1)
        p = torch.softmax(x, -1)
        p[:, :, blind] = 0
        want = p @ V
        S = float((Q.abs() @ K.abs().transpose(2, 3)).max() * scale)
        tol = (2 * EPS_S * S + 2 * 2.0 ** -20 + 2.0 ** -11) * float(V.abs().max())
        if ot == cfi.T_F16:
            tol = tol + 2.0 ** -11 * want.abs() + 2.0 ** -25
        err = (got - want).abs()
        assert bool((err <= tol).all()), (s, n, m, float((err / tol).max()))
        assert (got[:, :, blind] == 0).all()
    assert (out[:, wq:] == 7.0).all()
    return out


@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention(heads, kv, dim, causal):
    nq = [1, 0, 17, 128, 129, 300, 2, 64]
    packed_case(heads, kv, dim, nq, nq, causal)


@pytest.mark.parametrize("heads,kv,dim", SHAPES[:4])
@pytest.mark.parametrize("causal", [True, False])
def test_packed_attention_context(heads, kv, dim, causal):
    """More keys than queries (an earlier context), and fewer: the first queries then see none."""
    nq = [5, 130, 1, 40, 70, 3, 0, 9]
    nk = [300, 131, 1000, 17, 70, 0, 50, 2049]
    packed_case(heads, kv, dim, nq, nk, causal, ot=cfi.T_F16, pad=8)


@pytest.mark.parametrize("n", [1, 2, 127, 255, 256, 257, 631, 2100])
def test_packed_attention_one_sequence(n):
    packed_case(14, 2, 64, [n], [n])
    packed_case(12, 2, 128, [n], [n], ot=cfi.T_F16)


@pytest.mark.parametrize("heads", [1, 3, 7, 48, 64, 100, 128])
def test_packed_attention_group_sizes(heads):
    packed_case(heads, 1, 64, [50, 3, 200], [50, 3, 260])


def test_packed_attention_hundreds_of_short_sequences():
    rng = np.random.default_rng(5)
    nq = [int(x) for x in rng.integers(0, 40, 300)]
    packed_case(4, 2, 64, nq, nq)


def test_packed_attention_large_scores():
    packed_case(12, 2, 128, [300, 20], [400, 20], amp=30.0)


def test_packed_attention_bad_neighbour():
    """NaN keys and infinite values of one sequence leave the others as they are, beside it in a tile or not."""
    for heads, kv, dim in ((14, 2, 64), (12, 2, 128)):
        packed_case(heads, kv, dim, [40, 50, 60], [40, 50, 60], poison=True)
        packed_case(heads, kv, dim, [200, 3, 130], [333, 3, 140], poison=True)


@pytest.mark.parametrize("heads,kv,dim,n", [(12, 2, 128, 2048), (14, 2, 64, 1500), (2, 2, 64, 9000), (16, 16, 64, 3000),
                                             (40, 2, 64, 1500), (32, 8, 128, 1500)])
def test_packed_attention_every_tile_writes_its_own_rows(heads, kv, dim, n):
    """More single tiles than SMs, of which the short ones end long before their neighbours: each row is written by
    its own tile only, in both output types, with and without the mask."""
    for causal in (True, False):
        for ot in (cfi.T_F32, cfi.T_F16):
            packed_case(heads, kv, dim, [n], [n] if causal else [130], causal, ot=ot, seed=n)


@pytest.mark.parametrize("heads,kv,dim", [(12, 2, 128), (14, 2, 64), (8, 8, 128), (64, 1, 64)])
@pytest.mark.parametrize("n", [3, 40, 130])
def test_packed_attention_many_sequences(heads, kv, dim, n):
    """Sequences of all lengths in no order, empty ones, contexts, more queries than keys: few tiles and many."""
    rng = np.random.default_rng(n + heads)
    nq = [int(x) for x in rng.integers(0, 260, n)]
    nk = [max(0, q + int(x)) for q, x in zip(nq, rng.choice([0, 0, 0, 500, -60], n))]
    for causal in (True, False):
        packed_case(heads, kv, dim, nq, nk, causal, ot=cfi.T_F16, seed=n)


@pytest.mark.parametrize("heads,kv,dim", [(12, 2, 128), (14, 2, 64), (40, 2, 64)])
@pytest.mark.parametrize("n", [400, 2000])
def test_packed_attention_tiles_without_a_key(heads, kv, dim, n):
    """Far more queries than keys: tiles that see none, alone and beside one that sees some, are zeros, on every run."""
    for m in (1, 10, 45, 130):
        for ot in (cfi.T_F32, cfi.T_F16):
            packed_case(heads, kv, dim, [n, 5, n], [m, 9, m + 3], True, ot=ot, seed=m)


def test_packed_attention_ranges_are_cut():
    """Ends past the tensors are cut to them: nothing outside is read or written."""
    heads, kv, dim, n = 4, 2, 64, 100
    q, k, v = (torch.randn(n, h * dim, device=DEV).half() for h in (heads, kv, kv))
    out = torch.full((n + 50, heads * dim), 7.0, device=DEV)
    cu = torch.tensor([0, 60, 5000], dtype=torch.int32, device=DEV)
    cfi.packed_attention(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), cu.data_ptr(), cu.data_ptr(), 2, n, n, heads, kv, dim,
                         0.125, stream=stream())
    torch.cuda.synchronize()
    assert (out[n:] == 7.0).all() and torch.isfinite(out).all() and not (out[:n] == 7.0).any()


# ---- sampling ----
def sample(z, u, temperature=None, top_k=None, top_p=None, min_p=None):
    rows, vocab = z.shape
    dev = lambda x, t: None if x is None else torch.tensor(x, dtype=t, device=DEV)  # noqa: E731
    a = [dev(temperature, torch.float32), dev(top_k, torch.int32), dev(top_p, torch.float32), dev(min_p, torch.float32)]
    ud = dev(u, torch.float32)
    token = torch.full((rows,), -9, dtype=torch.int32, device=DEV)
    lp = torch.full((rows,), 7.0, device=DEV)
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    cfi.sample(z.data_ptr(), ud.data_ptr(), token.data_ptr(), rows, vocab, ptr(a[0]), ptr(a[1]), ptr(a[2]), ptr(a[3]), lp.data_ptr(),
               row_stride=z.stride(0), stream=stream())
    torch.cuda.synchronize()
    return token.cpu().numpy(), lp.double().cpu().numpy()


SLACK = 1e-6  # of the whole weight: expf's error, a weight's cut to 2^-40 and the logits' division


def fits(zrow, u, token, lp, t=1.0, k=0, p=1.0, m=0.0):
    """Whether the token is one that the definition allows, in 64 bits, with SLACK at every border."""
    z = zrow.astype(np.float64)
    z = np.where(np.isnan(z), -np.inf, z)
    best = int(np.argmax(z))
    if t <= 0:
        return token == best and lp == 0
    z = z / t
    order = np.argsort(-z, kind="stable")
    e = np.exp(z - z[best])
    eo = e[order]
    if k > 0:
        eo = np.where(np.arange(len(eo)) < k, eo, 0)
    before = np.cumsum(eo) - eo
    lo = (before < (p - SLACK) * eo.sum()) & (eo >= m * (1 + SLACK))   # surely kept
    hi = ((before < (p + SLACK) * eo.sum()) if p < 1 else np.ones(len(eo), bool)) & (eo >= m * (1 - SLACK))
    if p >= 1:
        lo = eo >= m * (1 + SLACK)
    lo[0] = hi[0] = True
    if k > 0:
        lo[k:] = hi[k:] = False
    n_lo, n_hi = int(lo.sum()), int(hi.sum())
    assert n_hi - n_lo <= 2 or eo[n_lo:n_hi].sum() < 4 * SLACK * eo.sum()
    for n in {n_lo, n_hi}:
        kept = np.sort(order[:n])
        cum = np.cumsum(e[kept])
        at = np.searchsorted(kept, token)
        if at < len(kept) and kept[at] == token:
            x = float(np.float32(u)) * cum[-1]
            if cum[at] - e[token] - SLACK * cum[-1] <= x <= cum[at] + SLACK * cum[-1] and \
                    abs(lp - (np.log(e[token]) - np.log(cum[-1]))) <= 4e-6 * max(1.0, abs(np.log(e[token])), abs(lp)):
                return True
    return False


@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 32001, 151936, 400000])
def test_sample(vocab):
    rng = np.random.default_rng(vocab)
    rows = 24
    z = (rng.normal(size=(rows, vocab)) * 2.5).astype(np.float32)
    for r in range(rows):
        top = rng.integers(0, vocab, min(40, vocab))
        z[r, top] += rng.random(len(top)).astype(np.float32) * 10
    t = [0.7, 1.0, 0.0, 1.5, 0.3, 1.0][:6] * 4
    k = [0, 40, 0, 1000, 1, 7, 0, 300][:8] * 3
    p = [1.0, 0.9, 0.5][:3] * 8
    m = [0.0, 0.0, 0.05, 0.0][:4] * 6
    u = rng.random(rows).astype(np.float32)
    u[0], u[1] = 0.0, np.float32(1) - np.float32(2.0 ** -24)
    d = torch.from_numpy(z).to(DEV)
    token, lp = sample(d, u, t, k, p, m)
    for r in range(rows):
        assert fits(z[r], u[r], token[r], lp[r], t[r], k[r], p[r], m[r]), (r, token[r], lp[r], t[r], k[r], p[r], m[r])
    again, lp2 = sample(d[5:6], u[5:6], t[5:6], k[5:6], p[5:6], m[5:6])  # alone: the same token
    assert again[0] == token[5] and lp2[0] == lp[5]


def test_sample_defaults_and_stride():
    rng = np.random.default_rng(3)
    z = rng.normal(size=(5, 1100)).astype(np.float32)
    d = torch.from_numpy(z).to(DEV)[:, 3:1004]
    u = rng.random(5).astype(np.float32)
    token, lp = sample(d, u)
    for r in range(5):
        assert fits(z[r, 3:1004], u[r], token[r], lp[r])


def test_sample_every_uniform_number():
    """Across u, each token comes as often as its share: the ends of the shares are hit exactly."""
    z = torch.log(torch.tensor([[0.125, 0.5, 0.25, 0.125]], device=DEV)).expand(4096, 4).contiguous()
    u = (np.arange(4096) + 0.5) / 4096
    token, _ = sample(z, u.tolist())
    assert np.abs(np.bincount(token, minlength=4) - 4096 * np.array([0.125, 0.5, 0.25, 0.125])).max() <= 1


@pytest.mark.parametrize("vocab", [700, 151936])
def test_sample_ties(vocab):
    z = np.zeros((9, vocab), np.float32)
    z[4] = np.round(np.random.default_rng(1).normal(size=vocab) * 2) / 2  # few distinct values
    z[5] = z[4]
    z[6] = np.random.default_rng(2).normal(size=vocab) * 1e-8  # differ in the last bits of z only
    z[7] = z[6]
    z[8, ::2] = -0.0  # equal to 0
    u = [0.0, 0.999, 0.5, 0.7, 0.3, 0.9, 0.6, 0.6, 0.99]
    t, k, p = [1, 1, 0, 1, 1, 1, 1, 1, 1.0], [5, 5, 0, 0, 333, 0, 333, 0, 400], [1, 1, 1, 0.25, 1, 0.8, 1, 0.4, 1.0]
    token, lp = sample(torch.from_numpy(z).to(DEV), u, t, k, p)
    assert token[0] == 0 and token[1] == 4 and token[2] == 0
    assert token[3] == int(0.7 * math.ceil(vocab / 4))
    assert token[8] == 396
    assert abs(lp[0] + math.log(5)) <= 1e-6
    for r in (4, 5, 6, 7):
        assert fits(z[r], u[r], token[r], lp[r], 1.0, k[r], p[r]), r


def test_sample_infinities_and_nan():
    inf, nan = math.inf, math.nan
    z = np.full((6, 500), -inf, np.float32)
    z[1, 7] = 2.0
    z[2] = nan
    z[2, 11] = -3.0
    z[3, [5, 9]] = inf
    z[4] = 1.0
    z[4, :250] = nan
    z[5] = np.finfo(np.float32).min
    for k, p in ((0, 1.0), (10, 0.9), (0, 0.5)):
        token, lp = sample(torch.from_numpy(z).to(DEV), [0.937] * 6, None, [k] * 6, [p] * 6)
        assert token[0] == -1 and lp[0] == -inf
        assert token[1] == 7 and lp[1] == 0
        assert token[2] == 11
        assert token[3] == (9 if p > 0.5 else 5)
        assert token[4] == 250 + int(0.937 * (250 if k == 0 else 10) * p)
        assert token[5] == int(0.937 * (500 if k == 0 else 10) * p)


def test_sample_top_p_zero_and_top_k_one():
    z = torch.randn(2, 5000, device=DEV)
    token, lp = sample(z, [0.99, 0.99], None, [0, 1], [0.0, 1.0])
    assert (token == z.argmax(1).cpu().numpy()).all() and (lp == 0).all()


@pytest.mark.parametrize("vocab", [1, 33, 1000, 2049, 5001, 65536, 151936, 400000])
@pytest.mark.parametrize("whole", [2, 60])
def test_sample_many_rows(vocab, whole):
    """Many rows in one call, of which few or most have a nucleus of the whole row or a long top-k, give what each
    row gives in a small call: every sum is a whole number, so token and log probability are the same."""
    rng = np.random.default_rng(vocab + whole)
    rows, wide = 76, vocab + 5
    z = (rng.normal(size=(rows, wide)) * 2.5).astype(np.float32)
    z[:, 3:][np.arange(rows), rng.integers(0, vocab, rows)] += 12
    z[3] = 0.0
    z[4] = np.round(z[4] * 2) / 2   # long runs of equal logits
    z[5, ::2] = -np.inf
    z[6] = -np.inf
    z[7, :vocab // 2] = np.nan
    z[8, 3] = np.inf
    z[9] = np.finfo(np.float32).min
    z[10] *= 1e-3                   # flat
    z[11] *= np.float32(1e-38)      # products that underflow
    z[12] *= 1000.0
    t = np.array([0.7, 1.0, 0.0, 1.3, 2.5, 1e-3, 1e20], np.float32)[np.arange(rows) % 7]
    k = np.array([40, 1000, 5, 1, 1024, 300], np.int32)[np.arange(rows) % 6]
    k[20:30] = 0
    p = np.array([1.0, 0.9, 0.5, 0.999], np.float32)[np.arange(rows) % 4]
    m = np.array([0.0, 0.0, 0.05], np.float32)[np.arange(rows) % 3]
    p[20:30] = 1.0                  # no filter
    for r in range(30 if whole > 2 else 74, 76):
        k[r], p[r] = (0, [0.95, 0.3, 0.9999][r % 3]) if r % 4 else (min(vocab, 3000), 0.9)
    k[3:13], p[3:13] = (0, 0.9) if whole > 2 else (50, 0.8)
    u = rng.random(rows).astype(np.float32)
    d = torch.from_numpy(z).to(DEV)[:, 3:3 + vocab]
    token, lp = sample(d, u, t, k, p, m)
    for at in range(0, rows, 30):
        one = slice(at, at + 30)
        alone, lp2 = sample(d[one], u[one], t[one], k[one], p[one], m[one])
        assert (token[one] == alone).all(), (at, token[one], alone)
        assert ((lp[one] == lp2) | ((lp[one] != lp[one]) & (lp2 != lp2))).all()
    for r in (0, 1, 13, 21, 40, 41, 75):
        assert fits(z[r, 3:3 + vocab], u[r], token[r], lp[r], t[r], k[r], p[r], m[r]), r


# ---- streams ----
def test_two_streams_do_not_share():
    """The operators on two streams at once give what each gives alone."""
    cases = [decode_case(cfi.T_F16, 14, 2, 64, 16, [5000, 77, 1], cfi.T_F32, cfi.T_F32, seed=1),
             decode_case(cfi.Q8_0, 12, 2, 128, 32, [8000, 3], cfi.T_F32, cfi.T_F32, seed=2)]
    torch.cuda.synchronize()
    want = [c[2].clone() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(10):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                c[2].zero_()
                c[0]()
    torch.cuda.synchronize()
    for c, w in zip(cases, want):
        assert torch.equal(c[2], torch.where(w == 7.0, torch.zeros_like(w), w))
