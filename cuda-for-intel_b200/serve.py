"""Synthetic serving driver: many sequences at once on the weights of a decode.DecodeModel (Qwen2
architecture, Q8_0; random, or those of a GGUF file through decode.load_gguf).

A prompt of any length goes through the stack packed with the others of its batch, one token of each
running sequence steps together, and tokens are sampled on the device (include/cfi_serve.h): the rows
of K and V go into the pages of one cache per layer, in f16 or quantised to Q8_0 or Q4_1 as they are
written; a prompt reads its whole context back as f16 rows and attends causally; a step attends over the pages.
Products run through the substituted quantize_mmq_q8_1 and mul_mat_q, norms and rope through rms_norm
and rope_neox, or biases, norms of the heads, rope and the cache's rows through one cfi_norm_rope; who owns
which page is kept on the host or, by cfi_paged_place, on the device; SwiGLU, residuals and the embedding
rows are torch's.

    python serve.py [--cache f16|q8_0|q4_1] [--batch 8] [--new 32] [--layers 4] [--file model.gguf] [--fused] [--norms]
                    [--tables host|device]
"""
import math
from types import SimpleNamespace

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
        self.pages = []  # where the tables are the host's
        self.row = None  # of the device's table
        self.placed = 0  # positions that the row may hold: more than are cached where a call did not come to its end
        self.cached = 0
        self.sure = 0  # of these, what was there at the last tokens: where the table is the device's
        self.temperature, self.top_k, self.top_p, self.min_p = temperature, top_k, top_p, min_p


class Server:
    """`model`: a DecodeModel (its weights are used, its own caches are not); `pages` pages of
    `page_size` positions are shared by all sequences; cache_type cfi.T_F16, cfi.Q8_0 or cfi.Q4_1.  Each call works on the
    stream that is torch's current one then, after what the calls before it did on theirs.

    fused: biases, rope and the rows into the cache by one cfi_norm_rope a layer (its angles are right at any position; those of
    rope_neox are in 32 bits).  None: where the cache is Q4_1 or there are norms.  norms: of each layer the weights (f32, head_dim,
    on the model's device) that the heads of q and of k are normed with, for models that have them.
    tables: "host", or "device" for page tables that cfi_paged_place keeps, for up to `rows` sequences at a time; a step's attention is then given
    a table as wide as the pool, for which it is cut as for long sequences (one of 768 takes 7.4 us instead of 5.5).
    A call that raises leaves what was cached before it; it can be made again."""

    def __init__(self, torch, ctx, model, cache_type=cfi.T_F16, page_size=16, pages=256, seed=0, fused=None, norms=None, tables="host",
                 rows=64):
        self.t, self.m, self.c = torch, model, model.cfg
        self.dev = model.dev
        self.g = cfi.GgmlCaller(ctx, "all")
        self.page_size, self.pages, self.cache_type = page_size, pages, cache_type
        c = self.c
        n = cfi.paged_page_bytes(cache_type, page_size, c.n_kv_head, c.head_dim)
        if n == 0:
            raise ValueError("no paged cache of type %d with pages of %d and heads of %d" % (cache_type, page_size, c.head_dim))
        if norms is not None and (len(norms) != len(model.layers) or fused is False):
            raise ValueError("norms are two vectors for each layer of a fused server")
        if tables not in ("host", "device"):
            raise ValueError("tables are the host's or the device's")
        self.norms = [tuple(pair) for pair in norms] if norms is not None else None
        self.fused = cache_type == cfi.Q4_1 or norms is not None if fused is None else fused
        # the pools, [layer][K or V][page]: a program keeps the description of each beside them
        self.pools = torch.zeros(c.layers, 2, pages * n, dtype=torch.uint8, device=self.dev)
        self.caches = [cfi.paged_cache(cache_type, p[0].data_ptr(), p[1].data_ptr(), pages, page_size, c.n_kv_head, c.head_dim)
                       for p in self.pools]
        for pair in self.norms or ():  # the kernels are given their addresses
            if len(pair) != 2 or not all(torch.is_tensor(w) and w.dtype == torch.float32 and w.shape == (c.head_dim,) and w.is_contiguous() and
                                         w.device == self.pools.device and w.data_ptr() % 16 == 0 for w in pair):
                raise ValueError("norms are two contiguous f32 vectors of %d on %s for each layer" % (c.head_dim, self.pools.device))
        self.free = list(range(pages))[::-1]  # where the tables are the host's
        self.held = [self.pools]
        self.on_device = tables == "device"
        if self.on_device:
            self.n_free, self.rows = pages, list(range(rows))[::-1]  # of which the host keeps count alone
            self.owner = {}  # the sequence of a row
            state = dict(table=torch.zeros(rows, pages, dtype=torch.int32, device=self.dev), cached=self._int([0] * rows),
                         free=self._int(self.free), n_free=self._int([pages]), status=self._int([0]))
            self.state = SimpleNamespace(**state)
            self.held += state.values()
            self.table = cfi.page_table(*(state[x].data_ptr() for x in ("table", "cached", "free", "n_free")), rows, pages, page_size, pages)
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
            for x in self.held:
                x.record_stream(now)
            self.last, self.stream = now, now.cuda_stream
        for x in given:
            x.record_stream(now)

    # ---- pages ----
    def _pages(self, positions):
        return -(-positions // self.page_size)

    def _once(self, seqs):
        if len({id(s) for s in seqs}) < len(seqs):
            raise ValueError("a sequence is named twice")

    def _grow(self, seqs, lengths):
        """Pages for the sequences' positions below `lengths`: all of them, or none are taken."""
        if self.on_device:
            self._once(seqs)
            left = [s for s in seqs if s.placed > s.cached]
            self._trim(left, [s.cached for s in left])
            need = sum(self._pages(n) - self._pages(s.placed) for s, n in zip(seqs, lengths))
            if need > self.n_free:
                raise OutOfPages("%d pages are free" % self.n_free)
            fresh = [s for s in seqs if s.row is None]
            if len(fresh) > len(self.rows):
                raise OutOfPages("%d rows of the page table are free" % len(self.rows))
            for s in fresh:
                s.row = self.rows.pop()
                s.sure, self.owner[s.row] = 0, s
            # before the device's table has them: what a call that fails from here on leaves behind is cut back by the next
            self.n_free -= need
            for s, n in zip(seqs, lengths):
                s.placed = n
            return
        need = [self._pages(n) - len(s.pages) for s, n in zip(seqs, lengths)]
        if sum(x for x in need if x > 0) > len(self.free):
            raise OutOfPages("%d pages are free" % len(self.free))
        for s, x in zip(seqs, need):
            s.pages += [self.free.pop() for _ in range(x)]

    def _trim(self, seqs, lengths):
        """The device's table keeps the sequences' first lengths[i] positions."""
        if not seqs:
            return
        rows, keep, status = self._int([s.row for s in seqs]), self._int(lengths), self._int([0])
        cfi.paged_trim(self.table, rows.data_ptr(), keep.data_ptr(), len(seqs), status.data_ptr(), stream=self.stream)
        self.n_free += sum(self._pages(s.placed) - self._pages(n) for s, n in zip(seqs, lengths))
        for s, n in zip(seqs, lengths):
            s.placed = n
        self.state.status |= status

    def _shrink(self, seqs, lengths):
        """The pages behind the sequences' first lengths[i] positions go back."""
        lengths = [min(s.cached, max(n, 0)) for s, n in zip(seqs, lengths)]
        if self.on_device:
            mine = [(s, n) for s, n in zip(seqs, lengths) if s.row is not None]
            self._trim([s for s, _ in mine], [n for _, n in mine])
        else:
            for s, n in zip(seqs[::-1], lengths[::-1]):
                while len(s.pages) > self._pages(n):
                    self.free.append(s.pages.pop())
        for s, n in zip(seqs, lengths):
            s.cached, s.sure = n, min(s.sure, n)

    def _told(self):
        """The page table's status, which is then clear.  Where calls were refused, the sequences have again what they had when it was last
        clear, and the host's counts are the device's."""
        status = int(self.state.status)
        if status == 0:
            for s in self.owner.values():
                s.sure = s.cached
            return 0
        self.state.status.zero_()
        held = self.state.cached.tolist()
        left = [r for r in self.rows if held[r]]  # of sequences that are released
        if left:
            rows, keep = self._int(left), self._int([0] * len(left))
            cfi.paged_trim(self.table, rows.data_ptr(), keep.data_ptr(), len(left), self.state.status.data_ptr(), stream=self.stream)
        self.n_free = int(self.state.n_free)
        for r, s in self.owner.items():
            s.placed = held[r]
            s.cached = s.sure = min(s.sure, held[r])
        return status

    def cut(self, seqs, lengths):
        """The sequences keep their first lengths[i] tokens and what is cached of them: the pages behind go back."""
        self._once(seqs)
        self._begin()
        self._shrink(seqs, lengths)
        for s, n in zip(seqs, lengths):
            del s.tokens[max(n, 0):]
            s.prompt = min(s.prompt, len(s.tokens))

    def release(self, seq):
        """The sequence's pages go back; its tokens stay."""
        if not self.on_device:
            self.free += seq.pages[::-1]
            seq.pages, seq.cached = [], 0
            return
        self._begin()
        self._shrink([seq], [0])
        if seq.row is not None:
            del self.owner[seq.row]
            self.rows.append(seq.row)
            seq.row = None

    def _placed(self, seqs, ends, with_context):
        """Where the sequences' tokens from what is cached to `ends` go: slots and positions of the new ones, lengths and pages, and, for
        prompts, the packed offsets and the slots of whole contexts."""
        t, n = self.t, len(seqs)
        self._grow(seqs, ends)
        p = SimpleNamespace(tokens=sum(e - s.cached for s, e in zip(seqs, ends)), positions=sum(ends), width=max(map(self._pages, ends), default=0))
        if self.on_device:
            i32 = lambda k: t.empty(k, dtype=t.int32, device=self.dev)  # noqa: E731
            p.width = self.pages
            p.rows, p.new = self._int([s.row for s in seqs]), self._int([e - s.cached for s, e in zip(seqs, ends)])
            p.lens, p.table, p.cu_q, p.cu_k, p.pos, status = i32(n), i32(n * self.pages), i32(n + 1), i32(n + 1), i32(p.tokens), i32(1)
            p.slots = t.empty(p.tokens, dtype=t.int64, device=self.dev)
            p.context = t.empty(p.positions if with_context else 0, dtype=t.int64, device=self.dev)
            batch = cfi.page_batch(p.rows.data_ptr(), p.new.data_ptr(), n, p.lens.data_ptr(), p.table.data_ptr(), p.cu_q.data_ptr(),
                                   p.cu_k.data_ptr(), p.slots.data_ptr(), p.pos.data_ptr(), p.tokens, status.data_ptr(),
                                   context=p.context.data_ptr() if with_context else 0, max_context=p.positions if with_context else 0)
            cfi.paged_place(self.table, batch, stream=self.stream)
            self.state.status |= status
            return p
        slots, positions, context, cu_q, cu_k = [], [], [], [0], [0]
        for s, e in zip(seqs, ends):
            slots += self._slots(s, s.cached, e)
            positions += range(s.cached, e)
            cu_q.append(len(slots))
            if with_context:
                context += self._slots(s, 0, e)
                cu_k.append(len(context))
        p.slots, p.pos = self._int(slots, t.int64), self._int(positions)
        if with_context:
            p.cu_q, p.cu_k, p.context = self._int(cu_q), self._int(cu_k), self._int(context, t.int64)
        else:
            p.table = self._int([s.pages + [0] * (p.width - len(s.pages)) for s in seqs])
            p.lens = self._int(ends)
        return p

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

    def _rows(self, i, lay, x, placed, q_type):
        """Layer i's rows of q, and those of k and v in its cache."""
        t, c = self.t, self.c
        nq, nkv, n = c.n_head * c.head_dim, c.n_kv_head * c.head_dim, x.shape[0]
        width = nq + 2 * nkv
        qkv = self._product(lay["wqkv"], self._norm(x, lay["attn_norm"]), width)
        if self.fused:
            out = t.empty(n, nq, dtype=t.float16 if q_type == cfi.T_F16 else t.float32, device=self.dev)
            at, bias = qkv.data_ptr(), lay["bqkv"].data_ptr()
            norm = [w.data_ptr() for w in self.norms[i]] if self.norms else [0, 0]
            cfi.norm_rope(cfi.norm_rope_rows(at, out.data_ptr(), placed.pos.data_ptr(), n, c.n_head, c.head_dim, k=at + 4 * nq, v=at + 4 * (nq + nkv),
                                             n_kv_head=c.n_kv_head, slots=placed.slots.data_ptr(), q_out_type=q_type, q_bias=bias,
                                             k_bias=bias + 4 * nq, v_bias=bias + 4 * (nq + nkv), q_norm=norm[0], k_norm=norm[1], eps=c.eps,
                                             freq_base=c.theta, q_stride=width, k_stride=width, v_stride=width), self.caches[i], stream=self.stream)
            return out
        qkv = qkv + lay["bqkv"]
        q = self._rope(qkv[:, :nq].contiguous(), c.n_head, placed.pos)
        k = self._rope(qkv[:, nq:nq + nkv].contiguous(), c.n_kv_head, placed.pos)
        # V is read in place, a slice of the stacked rows
        cfi.paged_kv_store(self.caches[i], k.data_ptr(), qkv.data_ptr() + 4 * (nq + nkv), placed.slots.data_ptr(), n, v_stride=width,
                           stream=self.stream)
        return q.half() if q_type == cfi.T_F16 else q

    def _run(self, tokens, placed, q_type, attend, last):
        """The layers over packed tokens; attend(layer, q) after the layer's rows are stored.  Logits of
        the rows `last`."""
        t, c = self.t, self.c
        x = self._embed(tokens)
        for i, lay in enumerate(self.m.layers):
            x = x + self._product(lay["wo"], attend(i, self._rows(i, lay, x, placed, q_type)), c.hidden)
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
        p = self._placed(seqs, ends, True)
        tokens, last = [], []
        for s, e in zip(seqs, ends):
            tokens += s.tokens[s.cached:e]
            last.append(len(tokens) - 1)
        kv = t.empty(2, p.positions, c.n_kv_head * c.head_dim, dtype=t.float16, device=self.dev)
        out = t.empty(len(tokens), c.n_head * c.head_dim, device=self.dev)

        def attend(i, q):
            cfi.paged_kv_load(self.caches[i], p.context.data_ptr(), kv[0].data_ptr(), kv[1].data_ptr(), p.positions, stream=self.stream)
            cfi.packed_attention(q.data_ptr(), kv[0].data_ptr(), kv[1].data_ptr(), out.data_ptr(), p.cu_q.data_ptr(), p.cu_k.data_ptr(),
                                 len(seqs), len(tokens), p.positions, c.n_head, c.n_kv_head, c.head_dim, 1.0 / math.sqrt(c.head_dim),
                                 stream=self.stream)
            return out

        logits = self._run(tokens, p, cfi.T_F16, attend, last)
        for s, e in zip(seqs, ends):
            s.cached = e
        return logits

    def step(self, seqs):
        """One token of each sequence, its last, over its pages; logits."""
        self._begin()
        t, c = self.t, self.c
        if any(s.cached != len(s.tokens) - 1 for s in seqs):
            raise ValueError("a step runs exactly the last token of each sequence")
        p = self._placed(seqs, [len(s.tokens) for s in seqs], False)
        out = t.empty(len(seqs), c.n_head * c.head_dim, device=self.dev)

        def attend(i, q):
            cfi.paged_attention(self.caches[i], q.data_ptr(), out.data_ptr(), p.table.data_ptr(), p.lens.data_ptr(), len(seqs), c.n_head,
                                p.width, 1.0 / math.sqrt(c.head_dim), stream=self.stream)
            return out

        logits = self._run([s.tokens[-1] for s in seqs], p, cfi.T_F32, attend, range(len(seqs)))
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
        refused = self._told() if self.on_device else 0
        if refused:
            raise RuntimeError("the page table's calls were refused (%d): what was cached since the last tokens is void" % refused)
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
    ap.add_argument("--cache", choices=("f16", "q8_0", "q4_1"), default="q8_0")
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--new", type=int, default=32)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--file", help="a qwen2 GGUF file instead of random weights")
    ap.add_argument("--fused", action="store_true", help="biases, rope and the cache's rows in one kernel")
    ap.add_argument("--norms", action="store_true", help="norms of the heads of q and k (random weights)")
    ap.add_argument("--tables", choices=("host", "device"), default="host")
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
    norms = [(1 + 0.1 * torch.randn(2, m.cfg.head_dim, generator=gen)).cuda() for _ in m.layers] if a.norms else None
    s = Server(torch, ctx, m, dict(f16=cfi.T_F16, q8_0=cfi.Q8_0, q4_1=cfi.Q4_1)[a.cache], 16, pages, fused=True if a.fused else None,
               norms=norms, tables=a.tables, rows=a.batch)
    begin = time.perf_counter()
    tokens = s.generate(seqs, a.new)
    torch.cuda.synchronize()
    took = time.perf_counter() - begin
    print("%d prompts of %d to %d tokens, %d new tokens each in %.3f s" % (a.batch, min(lengths), max(lengths), a.new, took))
    for n, x in zip(lengths, tokens):
        print("prompt %4d: %s" % (n, x[:8]))


if __name__ == "__main__":
    main()
