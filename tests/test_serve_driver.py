"""The serving driver (serve.py) without a GPU: its tensors on the CPU, the library's calls recorded.  What it computes is
tested in test_gpu_serve_model.py."""
import ctypes as C
from types import SimpleNamespace

import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import serve  # noqa: E402


class Stream:
    def __init__(self, handle):
        self.cuda_stream, self.waited_for = handle, []

    def wait_stream(self, other):
        self.waited_for.append(other)


class Torch:
    """torch with streams of this test's."""

    def __init__(self):
        self.now = Stream(100)
        self.cuda = SimpleNamespace(current_stream=lambda *a: self.now)

    def __getattr__(self, name):
        return getattr(torch, name)


@pytest.fixture
def rig(monkeypatch):
    """A server on a tiny model.  calls: (function, stream) of each of the library's calls; drawn: the tokens that sample()
    gives next; kept: (tensor's address, stream) of each record_stream."""
    r = SimpleNamespace(t=Torch(), calls=[], drawn=[], kept=[])

    def record(name):
        return lambda *a, stream=None, **k: r.calls.append((name, stream))

    def draw(logits, u, token, n, *a, stream=None):
        r.calls.append(("sample", stream))
        (C.c_int32 * n).from_address(token)[:] = [r.drawn.pop(0) if r.drawn else 1 for _ in range(n)]

    for name in ("paged_kv_store", "paged_kv_load", "paged_attention", "packed_attention"):
        monkeypatch.setattr(cfi, name, record(name))
    monkeypatch.setattr(cfi, "sample", draw)
    monkeypatch.setattr(cfi, "GgmlCaller", lambda ctx, switch: SimpleNamespace(
        **{name: record(name) for name in ("quantize_mmq", "mmq", "rms_norm", "rope_neox")}))
    monkeypatch.setattr(torch.Tensor, "record_stream", lambda x, s: r.kept.append((x.data_ptr(), s)))
    c = SimpleNamespace(hidden=128, layers=2, n_head=4, n_kv_head=2, head_dim=64, ffn=128, vocab=64, eps=1e-6, theta=1e6)
    u8, f = lambda n: torch.zeros(n, dtype=torch.uint8), torch.zeros  # noqa: E731
    layer = lambda: dict(wqkv=u8(1), bqkv=f(512), attn_norm=f(128), wo=u8(1), wgu=u8(1), ffn_norm=f(128), wd=u8(1))  # noqa: E731
    model = SimpleNamespace(cfg=c, dev="cpu", layers=[layer() for _ in range(2)], embd=u8(64 * 4 * 34), head=u8(1), out_norm=f(128))
    r.server = serve.Server(r.t, None, model, cfi.Q8_0, 16, 32)
    return r


def test_work_goes_to_the_stream_of_the_call(rig):
    """Each call's kernels go where torch's work of the same call goes, after what the server did before on another stream, and
    what it holds and is given is kept until they are done."""
    s, first = rig.server, rig.t.now
    seqs = [serve.Sequence([1, 2, 3]), serve.Sequence([4])]
    logits = s.prefill(seqs)
    assert {x for _, x in rig.calls} == {100} and len(rig.calls) > 20
    at = first
    for handle, call, given in ((200, lambda: s.sample(seqs, logits), [logits]), (300, lambda: s.step(seqs), []),
                                (200, lambda: s.generate([serve.Sequence([5, 6])], 2), []), (100, lambda: s.prefill([serve.Sequence([7])]), [])):
        del rig.calls[:], rig.kept[:]
        rig.t.now = Stream(handle)
        call()
        assert {x for _, x in rig.calls} == {handle}
        assert at in rig.t.now.waited_for
        for x in [s.pools] + given:
            assert (x.data_ptr(), rig.t.now) in rig.kept
        at = rig.t.now
    again = len(at.waited_for)
    s.sample([serve.Sequence([8])], logits)
    assert len(at.waited_for) == again  # the same stream: nothing to wait for
    assert (logits.data_ptr(), at) in rig.kept  # but these are another's


def test_a_row_without_a_token_is_an_error(rig):
    """-1 (no logit that can be taken) is not appended, nor is anything else of that call: the next step would read the
    embedding of the last token of the vocabulary."""
    s = rig.server
    seqs = [serve.Sequence([1, 2]), serve.Sequence([3])]
    logits = s.prefill(seqs)
    rig.drawn[:] = [5, -1]
    with pytest.raises(serve.NoToken, match="1"):
        s.sample(seqs, logits)
    assert [q.tokens for q in seqs] == [[1, 2], [3]]
    s.sample(seqs[:1], logits[:1])  # the other goes on
    s.step(seqs[:1])
    assert seqs[0].tokens == [1, 2, 1]


def test_a_wait_that_ran_out_is_seen(rig, monkeypatch):
    """What a kernel records when a bounded wait runs out makes the results void: sample(), which waits for them, raises."""
    s = rig.server
    seqs = [serve.Sequence([1, 2])]
    logits = s.prefill(seqs)
    words = [0xfb200]
    monkeypatch.setattr(cfi, "device_error", lambda: words.pop() if words else 0)
    with pytest.raises(RuntimeError, match="0xfb200"):
        s.sample(seqs, logits)
    assert seqs[0].tokens == [1, 2]
    s.sample(seqs, logits)
    assert seqs[0].tokens == [1, 2, 1]


@pytest.mark.parametrize("new", [0, 1, 3])
def test_generate_gives_as_many_tokens_as_asked(rig, new):
    seqs = [serve.Sequence([1, 2]), serve.Sequence([3])]
    assert rig.server.generate(seqs, new) == [[1] * new] * 2
    assert [q.cached for q in seqs] == [2 + max(0, new - 1), 1 + max(0, new - 1)]
