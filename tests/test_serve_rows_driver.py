"""The serving driver's Q4_1 caches, fused rows and device page tables (serve.py) without a GPU: its tensors on the CPU, the library's
calls recorded.  What they compute is tested in test_gpu_serve_rows.py."""
import ctypes as C
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import serve  # noqa: E402
from test_serve_driver import Stream, Torch  # noqa: E402


def word(p, n=1):
    return (C.c_int32 * n).from_address(p)


@pytest.fixture
def rig(monkeypatch):
    """build(**kw): a server on a tiny model.  calls: (function, stream); rows: of each norm_rope; status: what the calls on page tables
    answer next; drawn tokens are 1."""
    r = SimpleNamespace(t=Torch(), calls=[], rows=[], status=[], kept=[])

    def record(name):
        return lambda *a, stream=None, **k: r.calls.append((name, stream))

    def placed(table, batch, stream=None):
        r.calls.append(("paged_place", stream))
        r.batch = batch
        word(batch.status)[0] = r.status.pop(0) if r.status else 0

    def trimmed(table, rows, keep, n, status, stream=None):
        r.calls.append(("paged_trim", stream))
        r.trimmed = list(zip(word(rows, n), word(keep, n)))
        word(status)[0] = r.status.pop(0) if r.status else 0

    def rotated(rows, cache=None, stream=None):
        r.calls.append(("norm_rope", stream))
        r.rows.append(rows)

    def draw(logits, u, token, n, *a, stream=None):
        r.calls.append(("sample", stream))
        word(token, n)[:] = [1] * n

    for name in ("paged_kv_store", "paged_kv_load", "paged_attention", "packed_attention"):
        monkeypatch.setattr(cfi, name, record(name))
    monkeypatch.setattr(cfi, "paged_place", placed)
    monkeypatch.setattr(cfi, "paged_trim", trimmed)
    monkeypatch.setattr(cfi, "norm_rope", rotated)
    monkeypatch.setattr(cfi, "sample", draw)
    monkeypatch.setattr(cfi, "device_error", lambda: 0)
    monkeypatch.setattr(cfi, "GgmlCaller", lambda ctx, switch: SimpleNamespace(
        **{name: record(name) for name in ("quantize_mmq", "mmq", "rms_norm", "rope_neox")}))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda x, s: r.kept.append((x.data_ptr(), s)))
    c = SimpleNamespace(hidden=128, layers=2, n_head=4, n_kv_head=2, head_dim=64, ffn=128, vocab=64, eps=1e-6, theta=1e6)
    u8, f = lambda n: torch.zeros(n, dtype=torch.uint8), torch.zeros  # noqa: E731
    layer = lambda: dict(wqkv=u8(1), bqkv=f(512), attn_norm=f(128), wo=u8(1), wgu=u8(1), ffn_norm=f(128), wd=u8(1))  # noqa: E731
    r.model = SimpleNamespace(cfg=c, dev="cpu", layers=[layer() for _ in range(2)], embd=u8(64 * 4 * 34), head=u8(1), out_norm=f(128))
    r.build = lambda ty=cfi.Q8_0, pages=32, **kw: serve.Server(r.t, None, r.model, ty, 16, pages, **kw)
    r.names = lambda: [n for n, _ in r.calls]
    return r


def test_which_rows_are_fused(rig):
    norms = [(torch.ones(64), torch.ones(64)) for _ in range(2)]
    for kw, fused in ((dict(), False), (dict(ty=cfi.T_F16), False), (dict(ty=cfi.Q4_1), True), (dict(norms=norms), True), (dict(fused=True), True),
                      (dict(ty=cfi.Q4_1, fused=False), False)):
        del rig.calls[:], rig.rows[:]
        s = rig.build(**kw)
        s.prefill([serve.Sequence([1, 2, 3])])
        assert ("norm_rope" in rig.names()) == fused and ("rope_neox" in rig.names()) == (not fused)
        assert ("paged_kv_store" in rig.names()) == (not fused)
        for i, x in enumerate(rig.rows):
            assert (x.q_norm, x.k_norm) == ((norms[i][0].data_ptr(), norms[i][1].data_ptr()) if "norms" in kw else (None, None))
            assert x.q_bias == rig.model.layers[i]["bqkv"].data_ptr() and x.n_tokens == 3 and x.q_out_type == cfi.T_F16
    with pytest.raises(ValueError):
        rig.build(norms=norms[:1])
    with pytest.raises(ValueError):
        rig.build(norms=norms, fused=False)
    with pytest.raises(ValueError):
        rig.build(tables="elsewhere")


def test_work_goes_to_the_stream_of_the_call(rig):
    """Also of the calls on page tables, whose state is kept until they are done."""
    s = rig.build(cfi.Q4_1, tables="device")
    seqs = [serve.Sequence([1, 2, 3]), serve.Sequence([4])]
    logits = s.prefill(seqs)
    first = rig.t.now
    assert {x for _, x in rig.calls} == {100} and "paged_place" in rig.names()
    at = first
    for handle, call in ((200, lambda: s.sample(seqs, logits)), (300, lambda: s.step(seqs)), (200, lambda: s.cut(seqs, [2, 1])),
                         (100, lambda: s.release(seqs[0]))):
        del rig.calls[:], rig.kept[:]
        rig.t.now = Stream(handle)
        call()
        assert {x for _, x in rig.calls} == {handle}
        assert at in rig.t.now.waited_for
        for x in s.held:
            assert (x.data_ptr(), rig.t.now) in rig.kept
        at = rig.t.now


@pytest.mark.parametrize("tables", ["host", "device"])
def test_pages_are_counted(rig, tables):
    s = rig.build(pages=8, tables=tables)
    free = lambda: s.n_free if tables == "device" else len(s.free)  # noqa: E731
    a, b = serve.Sequence(list(range(40))), serve.Sequence(list(range(17)))
    s.prefill([a, b])
    assert free() == 8 - 3 - 2
    with pytest.raises(serve.OutOfPages):
        s.prefill([serve.Sequence(range(49))])
    assert free() == 3 and "paged_place" not in rig.names()[-3:]
    s.cut([a, b], [16, 90])
    assert (a.cached, len(a.tokens), a.prompt, b.cached, len(b.tokens), free()) == (16, 16, 16, 17, 17, 5)
    if tables == "device":
        assert sorted(rig.trimmed) == sorted([(a.row, 16), (b.row, 17)])
    a.tokens.append(5)
    s.step([a])
    assert free() == 4 and a.cached == 17
    s.release(a)
    assert free() == 6 and a.cached == 0 and len(a.tokens) == 17 and a.row is None
    s.cut([b], [-3])
    assert free() == 8 and b.tokens == [] and b.cached == 0
    with pytest.raises(ValueError):
        s.cut([a, a], [1, 1])


def test_rows_of_the_table_are_counted(rig):
    s = rig.build(tables="device", rows=2)
    seqs = [serve.Sequence([1]), serve.Sequence([2])]
    s.prefill(seqs)
    with pytest.raises(serve.OutOfPages):
        s.prefill([serve.Sequence([3])])
    s.release(seqs[1])
    s.prefill([serve.Sequence([3])])
    s.release(serve.Sequence([9]))  # one that never ran
    assert len(s.rows) == 0


def test_a_refused_page_table_is_seen(rig):
    s = rig.build(tables="device")
    seqs = [serve.Sequence([1, 2])]
    logits = s.prefill(seqs)
    rig.status[:] = [cfi.PLACE_NO_PAGES]
    s.sample(seqs, logits)
    logits = s.step(seqs)
    with pytest.raises(RuntimeError, match="refused"):
        s.sample(seqs, logits)
    assert seqs[0].tokens == [1, 2, 1]


@pytest.mark.parametrize("tables", ["host", "device"])
def test_generate(rig, tables):
    seqs = [serve.Sequence([1, 2]), serve.Sequence([3])]
    assert rig.build(cfi.Q4_1, tables=tables).generate(seqs, 3) == [[1] * 3] * 2
    assert [q.cached for q in seqs] == [4, 3]
