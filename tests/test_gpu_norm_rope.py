"""cfi_norm_rope (include/cfi_serve.h) against its formula in 64 bits.

Bounds.  The norm's sum of up to 128 squares, its quotient, root and the two products leave at most 2^-20 of a value; bias, the angle
(1e-7 rad), its sine and cosine (2^-23) and the two products of the rotation at most 2^-21 of the two values it joins.  An f16
output adds 2^-11 of itself (2^-25 below its normal numbers)."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import q41_pages as q41  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def stream():
    return torch.cuda.current_stream().cuda_stream


def formula(x, bias, norm, eps, pos, n_rot, base, scale, ff):
    """[token][head][dim] rows, and how far from it 32 bits may be."""
    x = x.double()
    if bias is not None:
        x = x + bias.double().view(x.shape[1:])
    if norm is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * norm.double()
    tol = x.abs() * 2.0 ** -20
    if n_rot:
        i = torch.arange(n_rot // 2, dtype=torch.float64, device=DEV)
        angle = pos.double()[:, None] * scale * torch.pow(torch.tensor(base, dtype=torch.float64, device=DEV), -2 * i / n_rot)
        angle = (angle / ff.double() if ff is not None else angle)[:, None]
        a, b = x[..., :n_rot // 2], x[..., n_rot // 2:n_rot]
        reach = (a.abs() + b.abs()) * (2.0 ** -20 + 2.0 ** -21)
        tol = torch.cat([reach, reach, tol[..., n_rot:]], -1)
        x = torch.cat([a * angle.cos() - b * angle.sin(), a * angle.sin() + b * angle.cos(), x[..., n_rot:]], -1)
    return x, tol


def near(got, want, tol):
    g = got.double()
    if got.dtype == torch.float16:
        tol = tol + want.abs() * 2.0 ** -11 + 2.0 ** -25
    worst = float(((g - want).abs() / (tol + 1e-300)).max())
    assert worst <= 1.0, worst


def make(tokens, heads, kv, dim, in_type=cfi.T_F32, q_type=cfi.T_F32, kv_type=cfi.T_F32, n_rot=None, bias=True, norm=True, ff=False, base=1e6,
         scale=1.0, far=5000, pad=0, seed=0, parts="qkv", amp=1.0):
    """Stacked rows and the description of a call that writes rows of all parts."""
    g = torch.Generator(device=DEV)
    g.manual_seed(seed + tokens + heads + dim)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    n_rot = dim if n_rot is None else n_rot
    base, scale = float(np.float32(base)), float(np.float32(scale))  # as the call takes them
    dt = lambda t: torch.float32 if t == cfi.T_F32 else torch.float16  # noqa: E731
    nq, nkv = heads * dim, kv * dim
    width = nq + 2 * nkv + pad
    x = dict(rows=(rand(tokens, width) * amp).to(dt(in_type)), bias=rand(nq + 2 * nkv) * 0.5 if bias else None,
             q_norm=1 + 0.2 * rand(dim) if norm else None, k_norm=1 + 0.2 * rand(dim) if norm else None,
             ff=1 + 3 * torch.rand(max(1, n_rot // 2), generator=g, device=DEV) if ff else None,
             pos=torch.randint(0, far, (tokens,), generator=g, device=DEV).to(torch.int32),
             q_out=torch.full((tokens, nq + 8), 7.0, dtype=dt(q_type), device=DEV),
             k_out=torch.full((tokens, nkv + 16), 7.0, dtype=dt(kv_type), device=DEV),
             v_out=torch.full((tokens, nkv), 7.0, dtype=dt(kv_type), device=DEV))
    p = lambda t, off=0: t.data_ptr() + off * t.element_size() if t is not None else 0  # noqa: E731
    args = dict(k=p(x["rows"], nq), v=p(x["rows"], nq + nkv), n_kv_head=kv, k_out=p(x["k_out"]), v_out=p(x["v_out"]), in_type=in_type,
                q_out_type=q_type, kv_out_type=kv_type, q_bias=p(x["bias"]), k_bias=p(x["bias"], nq), v_bias=p(x["bias"], nq + nkv),
                q_norm=p(x["q_norm"]), k_norm=p(x["k_norm"]), eps=1e-6, n_rot=n_rot, freq_base=base, freq_scale=scale,
                freq_factors=p(x["ff"]), q_stride=width, k_stride=width, v_stride=width, q_out_stride=nq + 8, k_out_stride=nkv + 16,
                v_out_stride=nkv)
    if not bias:
        args.update(k_bias=0, v_bias=0)
    if "k" not in parts:
        args.update(k=0, k_out=0)
    if "v" not in parts:
        args.update(v=0, v_out=0)
    x["args"] = args
    x["describe"] = lambda **kw: cfi.norm_rope_rows(p(x["rows"]), p(x["q_out"]), p(x["pos"]), tokens, heads, dim, **{**args, **kw})

    def want():
        r = x["rows"][:, :nq + 2 * nkv].reshape(tokens, -1, dim)
        b = x["bias"].view(-1, dim) if bias else None
        turn = (x["pos"], n_rot, base, scale, x["ff"])
        return [formula(r[:, :heads], b[:heads] if bias else None, x["q_norm"], 1e-6, *turn),
                formula(r[:, heads:heads + kv], b[heads:heads + kv] if bias else None, x["k_norm"], 1e-6, *turn),
                formula(r[:, heads + kv:], b[heads + kv:] if bias else None, None, 1e-6, x["pos"], 0, base, scale, None)]

    def check(parts=parts):
        torch.cuda.synchronize()
        for name, heads_of, (w, tol) in zip("qkv", (heads, kv, kv), want()):
            out = x[name + "_out"]
            if name not in parts:
                assert bool((out == 7.0).all())
                continue
            near(out[:, :heads_of * dim].reshape(tokens, heads_of, dim), w, tol)
            assert bool((out[:, heads_of * dim:] == 7.0).all())

    x["want"], x["check"] = want, check
    return x


SHAPES = [(14, 2, 64), (12, 2, 128), (32, 8, 128), (9, 3, 64), (16, 1, 128), (1, 1, 64), (5, 5, 128)]


@pytest.mark.parametrize("heads,kv,dim", SHAPES)
@pytest.mark.parametrize("tokens", [1, 3, 64, 333])
def test_rows(heads, kv, dim, tokens):
    x = make(tokens, heads, kv, dim)
    cfi.norm_rope(x["describe"](), stream=stream())
    x["check"]()


@pytest.mark.parametrize("in_type", [cfi.T_F32, cfi.T_F16])
@pytest.mark.parametrize("q_type,kv_type", [(cfi.T_F32, cfi.T_F16), (cfi.T_F16, cfi.T_F32), (cfi.T_F16, cfi.T_F16)])
@pytest.mark.parametrize("bias,norm", [(False, True), (True, False), (False, False)])
def test_types_and_parts(in_type, q_type, kv_type, bias, norm):
    for parts in ("qkv", "q", "qk", "qv"):
        for dim in (64, 128):
            x = make(37, 6, 2, dim, in_type, q_type, kv_type, bias=bias, norm=norm, pad=24, parts=parts)
            cfi.norm_rope(x["describe"](), stream=stream())
            x["check"]()


@pytest.mark.parametrize("dim,n_rot", [(64, 0), (64, 8), (64, 24), (64, 32), (64, 56), (128, 8), (128, 64), (128, 96), (128, 120), (128, 0)])
def test_parts_of_heads_turned(dim, n_rot):
    for norm in (False, True):
        x = make(21, 7, 2, dim, n_rot=n_rot, norm=norm)
        cfi.norm_rope(x["describe"](), stream=stream())
        x["check"]()


@pytest.mark.parametrize("tokens,heads,kv,dim", [(2500, 14, 2, 64), (4001, 32, 8, 128), (9000, 3, 1, 128)])
def test_many_rows(tokens, heads, kv, dim):
    """Sizes at which a thread takes several heads."""
    for in_type in (cfi.T_F32, cfi.T_F16):
        x = make(tokens, heads, kv, dim, in_type=in_type, q_type=cfi.T_F16, far=100000)
        cfi.norm_rope(x["describe"](), stream=stream())
        x["check"]()


@pytest.mark.parametrize("base,scale,ff", [(1e4, 1.0, False), (1e6, 0.25, False), (5e5, 1.0, True), (1e4, 8.0, True), (1.0, 1.0, False),
                                           (1e4, -1.0, False), (1e4, -1.0, True), (1e4, -0.01, True)])
def test_angles_of_far_positions(base, scale, ff):
    """The angles' errors do not grow with the positions (a formula in 64 bits is itself off by 2^-53 of the angle)."""
    far = (1 << 24) - 1 if ff else (1 << 31) - 1
    x = make(200, 2, 1, 128, base=base, scale=scale, ff=ff, norm=False, bias=False, far=far)
    x["pos"][0], x["pos"][1], x["pos"][2] = 0, far, 1
    if not ff:
        x["pos"][3], x["pos"][4] = -1, -(1 << 31)
    cfi.norm_rope(x["describe"](), stream=stream())
    x["check"]()


def test_in_place():
    for dim in (64, 128):
        x = make(50, 6, 2, dim)
        want = x["want"]()
        rows, width, nq, nkv = x["rows"], x["rows"].shape[1], 6 * dim, 2 * dim
        at = rows.data_ptr()
        args = dict(x["args"], k_out=at + 4 * nq, v_out=at + 4 * (nq + nkv), q_out_stride=width, k_out_stride=width, v_out_stride=width)
        cfi.norm_rope(cfi.norm_rope_rows(at, at, x["pos"].data_ptr(), 50, 6, dim, **args), stream=stream())
        torch.cuda.synchronize()
        got = rows[:, :nq + 2 * nkv].view(50, -1, dim)
        for (w, tol), part in zip(want, (got[:, :6], got[:, 6:8], got[:, 8:])):
            near(part, w, tol)


@pytest.mark.parametrize("ty", [cfi.T_F16, cfi.Q8_0, cfi.Q4_1])
@pytest.mark.parametrize("heads,kv,dim,page,tokens,n_rot", [(14, 2, 64, 16, 48, 64), (12, 2, 128, 64, 333, 64), (9, 3, 64, 32, 1, 24),
                                                            (32, 8, 128, 16, 2100, 128)])
def test_the_cache_gets_what_a_store_of_the_rows_puts_there(ty, heads, kv, dim, page, tokens, n_rot):
    """Bit for bit, and slots outside the pool get nothing."""
    x = make(tokens, heads, kv, dim, n_rot=n_rot)
    pages = -(-tokens // page) + 2
    n = cfi.paged_page_bytes(ty, page, kv, dim) * pages
    pools = torch.randint(0, 256, (4, n), device=DEV, dtype=torch.int32).to(torch.uint8)
    pools[2:] = pools[:2]
    fused, apart = (cfi.paged_cache(ty, pools[i].data_ptr(), pools[i + 1].data_ptr(), pages, page, kv, dim) for i in (0, 2))
    slots = torch.randperm(pages * page, device=DEV)[:tokens].contiguous()
    if tokens > 3:
        slots[1], slots[2] = -1, pages * page
    cfi.norm_rope(x["describe"](slots=slots.data_ptr()), fused, stream=stream())
    x["check"]()
    nkv = kv * dim
    cfi.paged_kv_store(apart, x["k_out"].data_ptr(), x["v_out"].data_ptr(), slots.data_ptr(), tokens, k_stride=nkv + 16, v_stride=nkv,
                       stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    again = pools[:2].clone()  # and without rows of k and v
    pools[:2] = 0
    cfi.norm_rope(x["describe"](slots=slots.data_ptr()), fused, stream=stream())
    whole = pools[:2].clone()
    pools[:2] = 0
    cfi.norm_rope(x["describe"](slots=slots.data_ptr(), k_out=0, v_out=0), fused, stream=stream())
    torch.cuda.synchronize()
    assert torch.equal(pools[:2], whole) and again.shape == whole.shape


def test_rows_of_zeros_and_of_bad_values():
    x = make(8, 4, 2, 64, bias=False)
    x["rows"][0] = 0
    x["rows"][1, 3] = float("nan")  # head 0 of q
    x["rows"][2, 4 * 64 + 5] = float("inf")  # head 0 of k
    cfi.norm_rope(x["describe"](), stream=stream())
    torch.cuda.synchronize()
    q, k, v = (x[n + "_out"][:, :m * 64].view(8, m, 64) for n, m in (("q", 4), ("k", 2), ("v", 2)))
    assert bool((q[0] == 0).all() and (k[0] == 0).all() and (v[0] == 0).all())
    assert bool(torch.isnan(q[1, 0]).all()) and bool(torch.isfinite(q[1, 1:]).all())
    assert not bool(torch.isfinite(k[2, 0]).all()) and bool(torch.isfinite(k[2, 1]).all())
    assert bool(torch.isfinite(q[3:]).all() and torch.isfinite(k[3:]).all() and torch.isfinite(v).all())


def test_captured():
    """Positions, slots and rows are read when the graph runs."""
    x = make(40, 12, 2, 128)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.graph(graph, stream=side):
        cfi.norm_rope(x["describe"](), stream=torch.cuda.current_stream().cuda_stream)
    for i in range(3):
        x["rows"].normal_()
        x["pos"].copy_(torch.arange(40) * 37 + 1000 * i)
        graph.replay()
        x["check"]()


def test_against_the_norm_and_rotation_that_are_there():
    """rms_norm and rope_neox one after the other, near positions (their angles are in 32 bits: off by 2^-22 of a turn's angle there)."""
    ctx = cfi.Ctx(0)
    g = cfi.GgmlCaller(ctx, "all")
    tokens, heads, dim = 60, 6, 64
    x = make(tokens, heads, 1, dim, bias=False, far=100, parts="q")
    rows = x["rows"][:, :heads * dim].contiguous()
    a, b = torch.empty_like(rows), torch.empty_like(rows)
    g.rms_norm(rows.data_ptr(), a.data_ptr(), dim, tokens * heads, mul=x["q_norm"].data_ptr(), eps=1e-6, stream=stream())
    g.rope_neox(a.data_ptr(), b.data_ptr(), dim, heads, tokens, dim, x["pos"].data_ptr(), freq_base=1e6, stream=stream())
    cfi.norm_rope(x["describe"](), stream=stream())
    torch.cuda.synchronize()
    err = (x["q_out"][:, :heads * dim] - b).abs().max()
    ctx.close()
    assert float(err) <= 100 * 2.0 ** -22 * 2 * float(a.abs().max())


def test_quantised_rows_are_the_definitions():
    """What the Q4_1 cache holds against the blocks of the rows that come out beside it."""
    x = make(64, 4, 2, 128)
    pools = torch.zeros(2, cfi.paged_page_bytes(cfi.Q4_1, 16, 2, 128) * 4, dtype=torch.uint8, device=DEV)
    cache = cfi.paged_cache(cfi.Q4_1, pools[0].data_ptr(), pools[1].data_ptr(), 4, 16, 2, 128)
    slots = torch.arange(64, device=DEV)
    cfi.norm_rope(x["describe"](slots=slots.data_ptr()), cache, stream=stream())
    torch.cuda.synchronize()
    for i, name in enumerate("kv"):
        got = q41.values(pools[i].cpu().numpy(), 4, 2, 16, 128, i == 1)
        np.testing.assert_array_equal(got, q41.quantised(x[name + "_out"][:, :256].reshape(64, 2, 128).double().cpu().numpy()))
