"""The serving driver (serve.py) on a small model: prompts packed, in chunks, stepped token by token and
in company give the same logits. (The operators themselves are held to 64 bits in test_gpu_serve.py.)

Bounds.  Every activation passes Q8_1 rounding several times a layer, and a difference in the last bits of
its input flips some of those roundings by one step of 1/127 of the block's maximum; attention differs
between the paths by the f16 rounding of q and the weights.  The decode driver's own test measures 5e-4
relative L2 after an attention and 2e-3 after the FFN per layer and holds chained logits to 5e-2; so does this one."""
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import decode  # noqa: E402
import serve  # noqa: E402

pytestmark = pytest.mark.gpu
REL = 5e-2


@pytest.fixture(scope="module")
def model():
    ctx = cfi.Ctx(0)
    cfg = decode.Config(hidden=256, layers=2, n_head=4, n_kv_head=2, head_dim=64, ffn=512, vocab=1024, prompt=8, n_ctx=16)
    yield ctx, decode.DecodeModel(torch, ctx, "cuda", cfg, fused=1)
    ctx.close()


def tokens(n, seed):
    return torch.randint(0, 1024, (n,), generator=torch.Generator().manual_seed(seed)).tolist()


def rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("ty", [cfi.T_F16, cfi.Q8_0])
@pytest.mark.parametrize("page", [16, 64])
def test_prompt_steps_and_chunks_agree(model, ty, page):
    ctx, m = model
    s = serve.Server(torch, ctx, m, ty, page, 64)
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


def test_company_does_not_matter(model):
    ctx, m = model
    s = serve.Server(torch, ctx, m, cfi.Q8_0, 16, 64)
    alone = s.prefill([serve.Sequence(tokens(40, 2))])
    many = [serve.Sequence(tokens(n, 2 if n == 40 else n)) for n in (1, 17, 40, 130)]
    assert rel(s.prefill(many)[2:3], alone) <= REL
    step = serve.Sequence(tokens(41, 2))
    step.tokens[:40] = tokens(40, 2)
    s.prefill([step], [40])
    for q in many:
        q.tokens.append(step.tokens[40])
    assert rel(s.step(many)[2:3], s.step([step])) <= REL


def test_f16_and_q8_0_caches_are_near(model):
    """Half a step of a Q8_0 block is 1/254 of its maximum: logits stay within a few of those."""
    ctx, m = model
    a, b = (serve.Server(torch, ctx, m, ty, 16, 16).prefill([serve.Sequence(tokens(90, 3))]) for ty in (cfi.T_F16, cfi.Q8_0))
    assert rel(b, a) <= REL


def test_pages_are_shared_and_reused(model):
    ctx, m = model
    s = serve.Server(torch, ctx, m, cfi.T_F16, 16, 8)
    first = [serve.Sequence(tokens(50, 4)), serve.Sequence(tokens(60, 5))]
    want = s.prefill(first)
    assert len(s.free) == 0
    with pytest.raises(serve.OutOfPages):
        s.prefill([serve.Sequence([1])])
    for q in first:
        s.release(q)
    assert len(s.free) == 8
    again = [serve.Sequence(tokens(60, 5)), serve.Sequence(tokens(50, 4))]  # other pages than before
    got = s.prefill(again)
    assert torch.equal(got[1], want[0]) and torch.equal(got[0], want[1])
    with pytest.raises(ValueError):
        s.step(again)  # nothing was sampled yet
    with pytest.raises(ValueError):
        s.prefill(again)  # nothing is left to run


def test_generate(model):
    ctx, m = model
    out = []
    for _ in range(2):
        s = serve.Server(torch, ctx, m, cfi.Q8_0, 32, 64, seed=7)
        out.append(s.generate([serve.Sequence(tokens(n, n), temperature=t, top_k=20, top_p=0.9) for n, t in ((5, 0.0), (33, 0.9), (64, 1.2))], 6))
    assert out[0] == out[1]  # the uniform numbers come from the seed
    assert all(len(x) == 6 and all(0 <= i < 1024 for i in x) for x in out[0])
    s = serve.Server(torch, ctx, m, cfi.Q8_0, 32, 64)
    greedy = serve.Sequence(tokens(5, 5), temperature=0.0)
    logits = s.prefill([greedy])
    s.sample([greedy], logits)
    assert greedy.tokens[-1] == int(logits.argmax())


def test_other_streams_than_the_one_it_was_built_on(model):
    """Prompts, steps and samples on streams of the caller's give what one stream gives."""
    ctx, m = model
    out = []
    for many in (False, True):
        s = serve.Server(torch, ctx, m, cfi.Q8_0, 16, 64, seed=9)
        seqs = [serve.Sequence(tokens(n, n), temperature=0.9, top_k=30) for n in (70, 3)]
        streams = [torch.cuda.Stream() for _ in range(3)] if many else [torch.cuda.current_stream()]
        if many:
            for x in streams:
                x.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(streams[0]):
            logits = s.prefill(seqs)
        for i in range(8):
            with torch.cuda.stream(streams[(i + 1) % len(streams)]):
                s.sample(seqs, logits)
            with torch.cuda.stream(streams[(i + 2) % len(streams)]):
                logits = s.step(seqs)
        torch.cuda.synchronize()
        out.append(([q.tokens for q in seqs], logits.clone()))
    assert out[0][0] == out[1][0] and torch.equal(out[0][1], out[1][1])
