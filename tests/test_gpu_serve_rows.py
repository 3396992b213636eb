"""Q4_1 caches, fused rows and device page tables together: as the serving driver runs them, and as a captured step.

Bounds of the driver's logits as in test_gpu_serve_model.py: every activation passes Q8_1 rounding several times a layer, and chained
logits are held to 5e-2 relative L2.  A Q4_1 cache is off by half a step, 1/30 of its blocks' ranges, which a comparison of its own
with another type would have to bound; here it is compared with itself."""
import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import decode  # noqa: E402
import q41_pages as q41  # noqa: E402
import serve  # noqa: E402

pytestmark = pytest.mark.gpu
REL = 5e-2
DEV = "cuda"


@pytest.fixture(scope="module", params=[64, 128])
def model(request):
    ctx = cfi.Ctx(0)
    cfg = decode.Config(hidden=256, layers=2, n_head=4, n_kv_head=2, head_dim=request.param, ffn=512, vocab=1024, prompt=8, n_ctx=16)
    yield ctx, decode.DecodeModel(torch, ctx, "cuda", cfg, fused=1)
    ctx.close()


def tokens(n, seed):
    return torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


def norms_of(model, seed=1):
    gen = torch.Generator().manual_seed(seed)
    return [(1 + 0.3 * torch.randn(2, model.cfg.head_dim, generator=gen)).cuda() for _ in model.layers]


@pytest.mark.parametrize("ty", [cfi.T_F16, cfi.Q8_0, cfi.Q4_1])
def test_fused_rows_are_the_separate_ones(model, ty):
    ctx, m = model
    out = [serve.Server(torch, ctx, m, ty, 16, 64, fused=f).prefill([serve.Sequence(tokens(n, n)) for n in (75, 3)]) for f in (False, True)]
    assert rel(out[1], out[0]) <= REL


@pytest.mark.parametrize("page", [16, 64])
@pytest.mark.parametrize("tables", ["host", "device"])
def test_prompts_steps_and_chunks_agree_on_q4_1(model, page, tables):
    ctx, m = model
    s = serve.Server(torch, ctx, m, cfi.Q4_1, page, 64, tables=tables, norms=norms_of(m))
    text = tokens(75, 1)
    whole = s.prefill([serve.Sequence(text)])
    chunked = serve.Sequence(text)
    s.prefill([chunked], [33])
    assert rel(s.prefill([chunked]), whole) <= REL
    stepped = serve.Sequence(text[:70])
    s.prefill([stepped])
    for x in text[70:]:
        stepped.tokens.append(x)
        logits = s.step([stepped])
    assert rel(logits, whole) <= REL


def test_norms_of_the_heads(model):
    """Against torch's own norm of the rows before the separate rope and store."""
    ctx, m = model
    norms = norms_of(m, 3)

    class Apart(serve.Server):
        def _rope(self, x, heads, pos):
            c = self.c
            y = x.view(-1, heads, c.head_dim)
            layer, which = divmod(self.at, 2)
            self.at += 1
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + c.eps) * norms[layer][which]
            return super()._rope(y.reshape(x.shape).contiguous(), heads, pos)

    apart = Apart(torch, ctx, m, cfi.T_F16, 16, 64)
    apart.at = 0
    want = apart.prefill([serve.Sequence(tokens(60, 8))])
    got = serve.Server(torch, ctx, m, cfi.T_F16, 16, 64, norms=norms).prefill([serve.Sequence(tokens(60, 8))])
    without = serve.Server(torch, ctx, m, cfi.T_F16, 16, 64).prefill([serve.Sequence(tokens(60, 8))])
    assert rel(got, want) <= REL and rel(without, want) > 2 * rel(got, want)


def test_device_tables_take_the_hosts_pages(model):
    """Prompts are placed where the host would place them, and run to the same bits."""
    ctx, m = model
    a, b = (serve.Server(torch, ctx, m, cfi.Q4_1, 16, 40, tables=t) for t in ("host", "device"))
    mine = [[serve.Sequence(tokens(n, n)) for n in (50, 1, 33)] for _ in "ab"]
    assert torch.equal(a.prefill(mine[0]), b.prefill(mine[1]))
    for x, y in zip(*mine):
        assert b.state.table[y.row, :len(x.pages)].tolist() == x.pages
    for s, q in ((a, mine[0]), (b, mine[1])):
        s.cut(q[:2], [17, 1])
        s.release(q[2])
        for z in q[:2]:
            z.tokens += tokens(30, 5)
    assert torch.equal(a.prefill(mine[0][:2]), b.prefill(mine[1][:2]))
    n = int(b.state.n_free)
    assert n == b.n_free == len(a.free) and b.state.free[:n].tolist() == a.free
    assert torch.equal(a.pools, b.pools) and int(b.state.status) == 0
    for x, y in zip(mine[0][:2], mine[1][:2]):
        x.tokens.append(7), y.tokens.append(7)
    # the table's width chooses how the attention is cut: rounding of 32 bits, and of Q8_1 behind it
    assert rel(b.step(mine[1][:2]), a.step(mine[0][:2])) <= REL


@pytest.mark.parametrize("tables", ["host", "device"])
def test_generate(model, tables):
    ctx, m = model
    out = []
    for _ in range(2):
        s = serve.Server(torch, ctx, m, cfi.Q4_1, 32, 64, seed=7, tables=tables)
        seqs = [serve.Sequence(tokens(n, n), temperature=t, top_k=20, top_p=0.9) for n, t in ((5, 0.0), (33, 0.9), (64, 1.2))]
        out.append(s.generate(seqs, 6))
        for q in seqs:
            s.release(q)
        assert (s.n_free if tables == "device" else len(s.free)) == 64
    assert out[0] == out[1]
    assert all(len(x) == 6 and all(0 <= i < 1024 for i in x) for x in out[0])


def test_drafts_that_are_not_taken(model):
    """A step after drafted tokens were cut away is the step without them, bit for bit."""
    ctx, m = model
    s = serve.Server(torch, ctx, m, cfi.Q4_1, 16, 64, tables="device")
    text = tokens(46, 9)
    plain, drafted = serve.Sequence(text), serve.Sequence(text)
    s.prefill([plain])
    s.prefill([drafted])
    drafted.tokens += tokens(20, 10)
    s.prefill([drafted])
    s.cut([drafted], [46])
    assert drafted.tokens == plain.tokens and drafted.cached == 46
    plain.tokens.append(3), drafted.tokens.append(3)
    assert torch.equal(s.step([plain]), s.step([drafted]))


@pytest.mark.parametrize("heads,kv,dim", [(6, 2, 128), (4, 1, 64), (14, 2, 64)])
def test_a_captured_step_of_all_of_them(heads, kv, dim):
    """Place, norm and rotate into the cache, attend: one graph, replayed for forty tokens of three sequences that cross pages, with other
    rows each time; then drafts of a second graph are cut away again.  The last outputs against the formula over what the cache holds."""
    page, pages, width, n, cap = 16, 40, 12, 3, 5
    nq, nkv = heads * dim, kv * dim
    g = torch.Generator(device=DEV)
    g.manual_seed(heads)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    zeros = lambda k, t=torch.int32: torch.zeros(k, dtype=t, device=DEV)  # noqa: E731
    table, cached, free, n_free = zeros(4 * width), i32([0] * 4), i32(list(range(pages))[::-1]), i32([pages])
    t = cfi.page_table(table.data_ptr(), cached.data_ptr(), free.data_ptr(), n_free.data_ptr(), 4, width, page, pages)
    pools = torch.randint(0, 256, (2, cfi.paged_page_bytes(cfi.Q4_1, page, kv, dim) * pages), device=DEV, dtype=torch.int32).to(torch.uint8)
    cache = cfi.paged_cache(cfi.Q4_1, pools[0].data_ptr(), pools[1].data_ptr(), pages, page, kv, dim)
    rows, new, keep = i32([2, 0, 3]), i32([1] * n), i32([0] * n)
    lens, batch_table, cu_q, cu_kv, positions, status = zeros(n), zeros(n * width), zeros(n + 1), zeros(n + 1), zeros(cap), zeros(2)
    slots = zeros(cap, torch.int64)
    batch = cfi.page_batch(rows.data_ptr(), new.data_ptr(), n, lens.data_ptr(), batch_table.data_ptr(), cu_q.data_ptr(), cu_kv.data_ptr(),
                           slots.data_ptr(), positions.data_ptr(), cap, status.data_ptr())
    qkv, q, out = torch.zeros(cap, nq + 2 * nkv, device=DEV), torch.zeros(cap, nq, device=DEV), torch.zeros(n, nq, device=DEV)
    weights = 1 + 0.2 * torch.randn(2, dim, generator=g, device=DEV)
    at = qkv.data_ptr()
    made = cfi.norm_rope_rows(at, q.data_ptr(), positions.data_ptr(), cap, heads, dim, k=at + 4 * nq, v=at + 4 * (nq + nkv), n_kv_head=kv,
                              slots=slots.data_ptr(), q_norm=weights[0].data_ptr(), k_norm=weights[1].data_ptr(), freq_base=1e4,
                              q_stride=nq + 2 * nkv, k_stride=nq + 2 * nkv, v_stride=nq + 2 * nkv)
    scale = 1 / math.sqrt(dim)

    def step():
        s = torch.cuda.current_stream().cuda_stream
        cfi.paged_place(t, batch, stream=s)
        cfi.norm_rope(made, cache, stream=s)
        cfi.paged_attention(cache, q.data_ptr(), out.data_ptr(), batch_table.data_ptr(), lens.data_ptr(), n, heads, width, scale, stream=s)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()  # the stream's workspace
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        step()
    for i in range(40):
        qkv.copy_(torch.randn(cap, nq + 2 * nkv, generator=g, device=DEV))
        if i == 25:
            new.copy_(i32([1, 0, 1]))  # one waits
        if i == 30:
            new.fill_(1)
        graph.replay()
        assert status.tolist() == [0, 0]
    want_len = [41, 36, 41]
    assert lens.tolist() == want_len and cached.tolist() == [36, 0, 41, 41] and int(n_free) == pages - 9
    held = [q41.values(pools[x].cpu().numpy(), pages, kv, page, dim, x == 1) for x in range(2)]
    bt = batch_table.view(n, width).cpu().numpy()
    got, qq = out.double().cpu().numpy().reshape(n, heads, dim), q[:n].double().cpu().numpy().reshape(n, heads, dim)
    for s in range(n):
        pos = np.arange(want_len[s])
        where = bt[s, pos // page].astype(np.int64) * page + pos % page
        for h in range(heads):
            K, V = held[0][where, h * kv // heads], held[1][where, h * kv // heads]
            x = K @ qq[s, h] * scale
            p = np.exp(x - x.max())
            want = p @ V / p.sum()
            mags = float((np.abs(qq[s, h]) @ (np.abs(K) + np.abs(K).max()).T).max() * scale)
            tol = (2 * 2.0 ** -20 * 3 * mags + 2 * 2.0 ** -20) * 3 * np.abs(V).max()
            assert (np.abs(got[s, h] - want) <= tol).all()
    # drafts: three more tokens each, cut away
    keep.copy_(lens)
    before = free[:int(n_free)].tolist()
    new.copy_(i32([1, 3, 1]))
    graph.replay()
    cfi.paged_trim(t, rows.data_ptr(), keep.data_ptr(), n, status.data_ptr() + 4, stream=torch.cuda.current_stream().cuda_stream)
    assert status.tolist() == [0, 0] and cached.tolist() == [36, 0, 41, 41] and free[:int(n_free)].tolist() == before
    # and a step that cannot be placed stores nothing
    new.fill_(1 << 20)
    was = pools.clone()
    graph.replay()
    assert int(status[0]) == cfi.PLACE_TOO_LONG and torch.equal(pools, was) and not bool(out.any())
