"""Synthetic serving driver: many sequences at once on the weights of a decode.DecodeModel (Qwen2
architecture, Q8_0; random, or those of a GGUF file through decode.load_gguf).

A prompt of any length goes through the stack packed with the others of its batch, one token of each
running sequence steps together, and tokens are sampled on the device (include/cfi_serve.h): the rows
of K and V go into the pages of one cache per layer, in f16 or quantised to Q8_0 as they are written;
a prompt reads its whole context back as f16 rows and attends causally; a step attends over the pages.
Products run through the substituted quantize_mmq_q8_1 and mul_mat_q, norms and rope through rms_norm
and rope_neox; biases, SwiGLU, residuals and the embedding rows are torch's.

    python serve.py [--cache f16|q8_0] [--batch 8] [--new 32] [--layers 4] [--file model.gguf]
"""
import math

import cfi_b200 as cfi


class OutOfPages(RuntimeError):
    pass


class NoToken(RuntimeError):
    """Logits of which none can be taken: all are -inf or NaN."""


class Sequence:
    """One request: its tokens so far, the pages that hold its context, how many positions they hold."""

    def __init__(self, tokens, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
        self.tokens = [int(t) for t in tokens]
        self.prompt = len(self.tokens)
        self.pages = []
        self.cached = 0
        self.temperature, self.top_k, self.top_p, self.min_p = temperature, top_k, top_p, min_p


class Server:
    """`model`: a DecodeModel (its weights are used, its own caches are not); `pages` pages of
    `page_size` positions are shared by all sequences; cache_type cfi.T_F16 or cfi.Q8_0.  Each call works on the
    stream that is torch's current one then, after what the calls before it did on theirs."""

    def __init__(self, torch, ctx, model, cache_type=cfi.T_F16, page_size=16, pages=256, seed=0):
        self.t, self.m, self.c = torch, model, model.cfg
        self.dev = model.dev
        self.g = cfi.GgmlCaller(ctx, "all")
        self.page_size, self.pages, self.cache_type = page_size, pages, cache_type
        c = self.c
        n = cfi.paged_page_bytes(cache_type, page_size, c.n_kv_head, c.head_dim)
        if n == 0:
            raise ValueError("no paged cache of type %d with pages of %d and heads of %d" % (cache_type, page_size, c.head_dim))
        # the pools, [layer][K or V][page]: a program keeps the description of each beside them
        self.pools = torch.zeros(c.layers, 2, pages * n, dtype=torch.uint8, device=self.dev)
        self.caches = [cfi.paged_cache(cache_type, p[0].data_ptr(), p[1].data_ptr(), pages, page_size, c.n_kv_head, c.head_dim)
                       for p in self.pools]
        self.free = list(range(pages))[::-1]
        self.gen = torch.Generator(device=self.dev)
        self.gen.manual_seed(seed)
        self.last = torch.cuda.current_stream()  # that of the last call
        self.stream = self.last.cuda_stream

    def _begin(self, *given):
        """A call begins: its stream, which waits for the last call's where that was another; what it reads is kept from the
        allocator until it has."""
        now = self.t.cuda.current_stream()
        if now != self.last:
            now.wait_stream(self.last)
            self.pools.record_stream(now)
            self.last, self.stream = now, now.cuda_stream
        for x in given:
            x.record_stream(now)

    # ---- pages ----
    def _grow(self, seqs, lengths):
        """Pages for the sequences' positions below `lengths`: all of them, or none are taken."""
        need = [-(-n // self.page_size) - len(s.pages) for s, n in zip(seqs, lengths)]
        if sum(x for x in need if x > 0) > len(self.free):
            raise OutOfPages("%d pages are free" % len(self.free))
        for s, x in zip(seqs, need):
            s.pages += [self.free.pop() for _ in range(x)]

    def release(self, seq):
        """The sequence's pages go back; its tokens stay."""
        self.free += seq.pages[::-1]
        seq.pages, seq.cached = [], 0

    def _slots(self, seq, first, end):
        p = self.page_size
        return [seq.pages[i // p] * p + i % p for i in range(first, end)]

    def _int(self, values, dtype=None):
        return self.t.tensor(values, dtype=dtype or self.t.int32, device=self.dev)

    # ---- the layers ----
    def _product(self, w, x, rows):
        """x [tokens][k] f32 times the Q8_0 matrix w [rows][k]."""
        n, k = x.shape
        q = self.t.empty(n * k // 128 * 144, dtype=self.t.uint8, device=self.dev)
        out = self.t.empty(n, rows, device=self.dev)
        self.g.quantize_mmq(0, x.data_ptr(), q.data_ptr(), k, k, n, stream=self.stream)
        self.g.mmq(cfi.Q8_0, w.data_ptr(), q.data_ptr(), out.data_ptr(), k, rows, n, stream=self.stream)
        return out

    def _norm(self, x, w):
        out = self.t.empty_like(x)
        self.g.rms_norm(x.data_ptr(), out.data_ptr(), x.shape[1], x.shape[0], mul=w.data_ptr(), eps=self.c.eps, stream=self.stream)
        return out

    def _rope(self, x, heads, pos):
        out = self.t.empty_like(x)
        self.g.rope_neox(x.data_ptr(), out.data_ptr(), self.c.head_dim, heads, x.shape[0], self.c.head_dim, pos.data_ptr(),
                         freq_base=self.c.theta, stream=self.stream)
        return out

    def _embed(self, tokens):
        b = self.m.embd.view(self.c.vocab, self.c.hidden // 32, 34)[self._int(tokens, self.t.int64)]
        d = b[..., :2].contiguous().view(self.t.float16).float()
        return (b[..., 2:].contiguous().view(self.t.int8).float() * d).reshape(len(tokens), self.c.hidden)

    def _run(self, tokens, positions, new_slots, attend, last):
        """The layers over packed tokens; attend(layer, q) after the layer's rows are stored.  Logits of
        the rows `last`."""
        t, c = self.t, self.c
        nq, nkv = c.n_head * c.head_dim, c.n_kv_head * c.head_dim
        width = nq + 2 * nkv
        x = self._embed(tokens)
        pos = self._int(positions)
        slots = self._int(new_slots, t.int64)
        for i, lay in enumerate(self.m.layers):
            qkv = self._product(lay["wqkv"], self._norm(x, lay["attn_norm"]), width) + lay["bqkv"]
            q = self._rope(qkv[:, :nq].contiguous(), c.n_head, pos)
            k = self._rope(qkv[:, nq:nq + nkv].contiguous(), c.n_kv_head, pos)
            # V is read in place, a slice of the stacked rows
            cfi.paged_kv_store(self.caches[i], k.data_ptr(), qkv.data_ptr() + 4 * (nq + nkv), slots.data_ptr(), len(tokens),
                               v_stride=width, stream=self.stream)
            x = x + self._product(lay["wo"], attend(i, q), c.hidden)
            gu = self._product(lay["wgu"], self._norm(x, lay["ffn_norm"]), 2 * c.ffn)
            x = x + self._product(lay["wd"], t.nn.functional.silu(gu[:, :c.ffn]) * gu[:, c.ffn:], c.hidden)
        x = x[self._int(last, t.int64)].contiguous()
        return self._product(self.m.head, self._norm(x, self.m.out_norm), c.vocab)

    def prefill(self, seqs, upto=None):
        """Runs the sequences' tokens that are not cached yet (of each the first upto[i] at most), all packed,
        after what is; logits of each one's last."""
        self._begin()
        t, c = self.t, self.c
        ends = [len(s.tokens) if upto is None else min(upto[i], len(s.tokens)) for i, s in enumerate(seqs)]
        if any(e <= s.cached for s, e in zip(seqs, ends)):
            raise ValueError("a sequence has no token to run")
        self._grow(seqs, ends)
        tokens, positions, new, context, cu_q, cu_k = [], [], [], [], [0], [0]
        for s, e in zip(seqs, ends):
            tokens += s.tokens[s.cached:e]
            positions += range(s.cached, e)
            new += self._slots(s, s.cached, e)
            context += self._slots(s, 0, e)
            cu_q.append(len(tokens))
            cu_k.append(len(context))
        dq, dk, slots = self._int(cu_q), self._int(cu_k), self._int(context, t.int64)
        kv = t.empty(2, len(context), c.n_kv_head * c.head_dim, dtype=t.float16, device=self.dev)
        out = t.empty(len(tokens), c.n_head * c.head_dim, device=self.dev)

        def attend(i, q):
            q16 = q.half()
            cfi.paged_kv_load(self.caches[i], slots.data_ptr(), kv[0].data_ptr(), kv[1].data_ptr(), len(context), stream=self.stream)
            cfi.packed_attention(q16.data_ptr(), kv[0].data_ptr(), kv[1].data_ptr(), out.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                                 len(seqs), len(tokens), len(context), c.n_head, c.n_kv_head, c.head_dim, 1.0 / math.sqrt(c.head_dim),
                                 stream=self.stream)
            return out

        logits = self._run(tokens, positions, new, attend, [x - 1 for x in cu_q[1:]])
        for s, e in zip(seqs, ends):
            s.cached = e
        return logits

    def step(self, seqs):
        """One token of each sequence, its last, over its pages; logits."""
        self._begin()
        t, c = self.t, self.c
        if any(s.cached != len(s.tokens) - 1 for s in seqs):
            raise ValueError("a step runs exactly the last token of each sequence")
        self._grow(seqs, [len(s.tokens) for s in seqs])
        width = max(len(s.pages) for s in seqs)
        table = self._int([s.pages + [0] * (width - len(s.pages)) for s in seqs])
        lens = self._int([len(s.tokens) for s in seqs])
        out = t.empty(len(seqs), c.n_head * c.head_dim, device=self.dev)

        def attend(i, q):
            cfi.paged_attention(self.caches[i], q.data_ptr(), out.data_ptr(), table.data_ptr(), lens.data_ptr(), len(seqs), c.n_head,
                                width, 1.0 / math.sqrt(c.head_dim), stream=self.stream)
            return out

        new = [self._slots(s, s.cached, s.cached + 1)[0] for s in seqs]
        logits = self._run([s.tokens[-1] for s in seqs], [s.cached for s in seqs], new, attend, range(len(seqs)))
        for s in seqs:
            s.cached += 1
        return logits

    def sample(self, seqs, logits):
        """Draws each sequence's next token and appends it; the drawn tokens' log probabilities.  NoToken, and no sequence is
        longer, where one has no logit that can be taken; RuntimeError where a kernel since the last call has given up a wait."""
        self._begin(logits)
        t, n = self.t, len(seqs)
        f = lambda v: t.tensor(v, dtype=t.float32, device=self.dev)  # noqa: E731
        temperature, top_p, min_p = f([s.temperature for s in seqs]), f([s.top_p for s in seqs]), f([s.min_p for s in seqs])
        top_k = self._int([s.top_k for s in seqs])
        u = t.rand(n, generator=self.gen, device=self.dev)
        token, logprob = t.empty(n, dtype=t.int32, device=self.dev), t.empty(n, device=self.dev)
        cfi.sample(logits.data_ptr(), u.data_ptr(), token.data_ptr(), n, self.c.vocab, temperature.data_ptr(), top_k.data_ptr(),
                   top_p.data_ptr(), min_p.data_ptr(), logprob.data_ptr(), stream=self.stream)
        drawn = token.tolist()
        error = cfi.device_error()
        if error:
            raise RuntimeError("a kernel's wait ran out (0x%x): the logits and what was cached since the last tokens are void" % error)
        if min(drawn, default=0) < 0:
            raise NoToken("no token for the sequences at %s of the batch" % [i for i, x in enumerate(drawn) if x < 0])
        for s, x in zip(seqs, drawn):
            s.tokens.append(x)
        return logprob

    def generate(self, seqs, new):
        """Prompts, then `new` tokens of each sequence."""
        logits = self.prefill(seqs)
        for i in range(new):
            self.sample(seqs, logits if i == 0 else self.step(seqs))
        return [s.tokens[s.prompt:] for s in seqs]


def main():
    import argparse
    import time

    import torch

    import decode

    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--cache", choices=("f16", "q8_0"), default="q8_0")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--file", help="a qwen2 GGUF file instead of random weights")
    a = ap.parse_args()
    torch.cuda.set_device(0)
    ctx = cfi.Ctx(0, const_weights=True)
    small = dict(prompt=8, n_ctx=16)  # of the model's own caches, which a server does not use
    m = (decode.load_gguf(torch, ctx, "cuda", a.file, fused=1, **small) if a.file else
         decode.DecodeModel(torch, ctx, "cuda", decode.Config(layers=a.layers, **small), fused=1))
    gen = torch.Generator().manual_seed(1)
    lengths = [int(x) for x in torch.randint(1, 600, (a.batch,), generator=gen)]
    seqs = [Sequence(torch.randint(0, m.cfg.vocab, (n,), generator=gen).tolist(), temperature=0.8, top_k=50, top_p=0.95) for n in lengths]
    pages = sum(-(-(n + a.new) // 16) for n in lengths)
    s = Server(torch, ctx, m, cfi.Q8_0 if a.cache == "q8_0" else cfi.T_F16, 16, pages)
    begin = time.perf_counter()
    tokens = s.generate(seqs, a.new)
    torch.cuda.synchronize()
    took = time.perf_counter() - begin
    print("%d prompts of %d to %d tokens, %d new tokens each in %.3f s" % (a.batch, min(lengths), max(lengths), a.new, took))
    for n, x in zip(lengths, tokens):
        print("prompt %4d: %s" % (n, x[:8]))


if __name__ == "__main__":
    main()
