"""Cases of the serving operators: the paged key-value cache (quantised as it is written, and read
back), the attention of one new token over it, the causal attention of packed prompts, and sampling.

A case names its operator in "op":
  cache   new rows of K and V go into the pages of a cache; a Q8_0 cache is then read back as f16
          rows (what a prompt that continues an earlier context does), an F16 cache is the output
  decode  one new token for each sequence attends to the sequence's pages
  prompt  packed sequences attend causally to their own keys, which may begin with an earlier context
  sample  one token for each row of logits: temperature, top-k, top-p, min-p, a given uniform number

Head counts and widths are those of the decode configurations (14 query and 2 key-value heads of 64,
12 and 2 of 128) and a generic 32 and 8 of 128; the vocabulary is theirs, 151936.
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

F32, F16, Q8_0 = 0, 1, 8
UNIT = 2.0 ** 40  # sampling weights are whole multiples of 2^-40 of the largest: sums of them have no order
DEV = "cuda"


def listed():
    return [
        # one decode step of 48 sequences writes a row each: latency
        dict(name="cache step f16", op="cache", type=F16, src=F32, tokens=48, context=0, heads_kv=2, dim=64, page=16, spare=464),
        # a short odd chunk after a short context
        dict(name="cache chunk q8", op="cache", type=Q8_0, src=F32, tokens=333, context=298, heads_kv=2, dim=128, page=32, spare=7),
        # a chunk of a long prompt after a long context
        dict(name="cache long q8", op="cache", type=Q8_0, src=F16, tokens=8192, context=57345, heads_kv=8, dim=128, page=64, spare=100),
        # a single user's token: latency
        dict(name="decode one f16", op="decode", type=F16, heads=14, heads_kv=2, dim=64, page=16, batch=1, lo=672, hi=672, lens=1),
        # a batch of chats whose lengths differ
        dict(name="decode batch q8", op="decode", type=Q8_0, heads=12, heads_kv=2, dim=128, page=16, batch=64, lo=16, hi=4096, lens=2),
        # a few long documents
        dict(name="decode long f16", op="decode", type=F16, heads=32, heads_kv=8, dim=128, page=64, batch=8, lo=9000, hi=65000, lens=3),
        # one prompt of 631 tokens
        dict(name="prompt one", op="prompt", heads=14, heads_kv=2, dim=64, batch=1, lo=631, hi=631, ctx=0, lens=4),
        # prompts of one token to 2048 in one call
        dict(name="prompt packed", op="prompt", heads=12, heads_kv=2, dim=128, batch=16, lo=1, hi=2048, ctx=0, lens=5),
        # chunks of four prompts, each after its earlier context
        dict(name="prompt chunks", op="prompt", heads=14, heads_kv=2, dim=64, batch=4, lo=300, hi=800, ctx=7000, lens=6),
        # one long document
        dict(name="prompt long", op="prompt", heads=12, heads_kv=2, dim=128, batch=1, lo=16384, hi=16384, ctx=0, lens=7),
        # a single user's token
        dict(name="sample one", op="sample", rows=1, vocab=151936, mix="nucleus"),
        # a large batch in which every request has its own settings
        dict(name="sample batch", op="sample", rows=256, vocab=151936, mix="all"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache", "decode", "prompt", "sample"])
    heads, kv, dim = rng.choice([(14, 2, 64), (12, 2, 128), (32, 8, 128), (16, 16, 64), (9, 3, 64), (16, 1, 128)])
    page, spread = rng.choice([16, 32, 64, 128]), rng.randrange(1, 1 << 20)
    if op == "cache":
        context = rng.choice([0, _log(rng, 1, 40000)])
        return dict(op=op, type=rng.choice([F16, Q8_0]), src=rng.choice([F32, F16]), tokens=_log(rng, 1, 16000), context=context,
                    heads_kv=min(kv, 8), dim=dim, page=page, spare=rng.randrange(1, 200))
    if op == "decode":
        batch = _log(rng, 1, 128)
        most = max(1, min(65000, 450_000_000 // (batch * kv * dim)))
        hi = _log(rng, 1, most)
        return dict(op=op, type=rng.choice([F16, Q8_0]), heads=heads, heads_kv=kv, dim=dim, page=page, batch=batch,
                    lo=_log(rng, 1, hi), hi=hi, lens=spread)
    if op == "prompt":
        batch = _log(rng, 1, 16)
        hi = _log(rng, 1, int(min(8192, math.sqrt(1.6e9 / (batch * heads)))))
        most = min(16000, 1_600_000_000 // (batch * heads * hi) - hi)
        ctx = rng.choice([0, _log(rng, 1, most)]) if most >= 1 else 0
        return dict(op=op, heads=heads, heads_kv=kv, dim=dim, batch=batch, lo=_log(rng, 1, hi), hi=hi, ctx=ctx, lens=spread)
    return dict(op=op, rows=_log(rng, 1, 250), vocab=_log(rng, 1000, 151936), mix=rng.choice(["all", "nucleus", "plain"]))


def _lengths(case):
    """The sequences' lengths: spread over the logarithm of lo..hi, one of them the longest."""
    r = random.Random(case["lens"])
    n = [_log(r, case["lo"], case["hi"]) for _ in range(case["batch"])]
    n[r.randrange(case["batch"])] = case["hi"]
    return n


def _contexts(case):
    """How many earlier keys each packed sequence has."""
    r = random.Random(case["lens"] + 1)
    return [r.randrange(case["ctx"] // 2, case["ctx"] + 1) for _ in range(case["batch"])]


def work(case):
    op = case["op"]
    if op == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * 4 + 28), "flops": case["rows"] * case["vocab"] * 4}
    dim = case["dim"]
    row = case["heads_kv"] * dim * 2  # values of K and V of one position
    held = (2 if case.get("type") == F16 else 34 / 32) * row
    if op == "cache":
        n = case["tokens"] * (row * (4 if case["src"] == F32 else 2) + held + 8)
        if case["type"] == Q8_0:
            n += (case["tokens"] + case["context"]) * (row * 2 + 8) + case["context"] * held
        return {"bytes": n, "flops": 4 * case["tokens"] * row}
    lens = _lengths(case)
    if op == "decode":
        q = case["batch"] * case["heads"] * dim * 2
        return {"bytes": sum(lens) * held + 2 * q + sum(4 * -(-n // case["page"]) + 4 for n in lens),
                "flops": 4 * sum(lens) * case["heads"] * dim}
    pairs = sum(n * c + n * (n + 1) // 2 for n, c in zip(lens, _contexts(case)))
    return {"bytes": sum(lens) * case["heads"] * dim * 4 + (sum(lens) + sum(_contexts(case))) * row * 2,
            "flops": 4 * pairs * case["heads"] * dim}


# ---- inputs ----
def _fill_pool(values, kind, dim):
    """[page, head, slot, dim] values as a pool's bytes: f16 rows, or int8 rows and behind them the f16 scales of their blocks."""
    if kind == F16:
        return values.half()
    n, h, p, _ = values.shape
    q, d = _q8_0(values)
    return torch.cat([q.to(torch.int8).view(n, h, p * dim).view(torch.uint8), d.half().view(n, h, p * dim // 32).view(torch.uint8)], 2)


def _pool(case, pages, g):
    v = torch.randn(pages, case["heads_kv"], case["page"], case["dim"], generator=g, device=DEV)
    return _fill_pool(v, case["type"], case["dim"])


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    op = case["op"]
    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a language model's logits: a broad normal floor and a few hundred candidates well above it
        z = rand(rows, vocab) * 2.0
        top = torch.randint(0, vocab, (rows, min(300, vocab)), generator=g, device=DEV)
        z.scatter_add_(1, top, torch.rand(rows, top.shape[1], generator=g, device=DEV) ** 2 * 14.0)
        u = torch.rand(rows, generator=g, device=DEV)
        r = torch.arange(rows, device=DEV)
        on = {"all": [0.7, 1.0, 0.0, 1.3], "nucleus": [0.8] * 4, "plain": [1.0] * 4}[case["mix"]]
        s.update(logits=z, u=u, temperature=torch.tensor(on, device=DEV)[r % 4].contiguous(),
                 token=torch.empty(rows, dtype=torch.int32, device=DEV), logprob=torch.empty(rows, device=DEV))
        mixed = case["mix"] == "all"
        plain = case["mix"] == "plain"
        pick = lambda a, t: torch.tensor(a, dtype=t, device=DEV)[(r // 4) % len(a)].contiguous()  # noqa: E731
        s["top_k"] = pick([0, 40, 1000, 1, 5] if mixed else [0] if plain else [50], torch.int32)
        s["top_p"] = pick([1.0, 0.95, 0.5] if mixed else [1.0] if plain else [0.9], torch.float32)
        s["min_p"] = pick([0.0, 0.05] if mixed else [0.0] if plain else [0.02], torch.float32)
        return _bind(s)
    dim, kv = case["dim"], case["heads_kv"]
    if op == "cache":
        n = case["tokens"] + case["context"]
        pages = -(-n // case["page"]) + case["spare"]
        s["k_pool"], s["v_pool"] = _pool(case, pages, g), _pool(case, pages, g)
        order = torch.randperm(pages, generator=g, device=DEV)
        pos = torch.arange(n, device=DEV)
        s["slots"] = (order[pos // case["page"]] * case["page"] + pos % case["page"]).contiguous()
        s["new"] = s["slots"][case["context"]:].contiguous()
        t = torch.float32 if case["src"] == F32 else torch.float16
        s["k"], s["v"] = rand(case["tokens"], kv, dim).to(t), rand(case["tokens"], kv, dim).to(t)
        if case["type"] == Q8_0:
            s["k_rows"], s["v_rows"] = (torch.empty(n, kv, dim, dtype=torch.float16, device=DEV) for _ in "kv")
        s["pages"] = pages
        return _bind(s)
    lens = _lengths(case)
    if op == "decode":
        need = [-(-n // case["page"]) for n in lens]
        width = max(need)
        pages = sum(need) + 3
        s["k_pool"], s["v_pool"] = _pool(case, pages, g), _pool(case, pages, g)
        order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
        start = torch.tensor([0] + need, device=DEV).cumsum(0)[:-1]
        at = torch.arange(width, device=DEV)[None] + start[:, None]
        s["table"] = torch.where(torch.arange(width, device=DEV)[None] < torch.tensor(need, device=DEV)[:, None],
                                 order[at.clamp_max(pages - 1)], 0).to(torch.int32).contiguous()
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["q"] = (rand(case["batch"], case["heads"], dim) * 1.5).half()
        s["out"] = torch.empty_like(s["q"])
        s.update(pages=pages, width=width, scale=1.0 / math.sqrt(dim))
        return _bind(s)
    klens = [n + c for n, c in zip(lens, _contexts(case))]
    s.update(tq=sum(lens), tk=sum(klens), lq=max(lens), lk=max(klens), scale=1.0 / math.sqrt(dim))
    s["cu_q"] = torch.tensor([0] + lens, device=DEV).cumsum(0).to(torch.int32)
    s["cu_k"] = torch.tensor([0] + klens, device=DEV).cumsum(0).to(torch.int32)
    s["q"] = (rand(s["tq"], case["heads"], dim) * 1.5).half()
    s["k"], s["v"] = rand(s["tk"], kv, dim).half(), rand(s["tk"], kv, dim).half()
    s["out"] = torch.empty_like(s["q"])
    return _bind(s)


def _bind(s):
    """The cache's description that a program keeps beside its pools."""
    if own and "pages" in s:
        c = s["case"]
        s["cache"] = _cfi().paged_cache(c["type"], s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), s["pages"], c["page"],
                                        c["heads_kv"], c["dim"])
    return s


def _cfi():
    at = os.path.join(os.getcwd(), "cuda-for-intel_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import cfi_b200
    return cfi_b200


# ---- one pass ----
def run(s):
    return (_run_own if own else _run_plain)[s["case"]["op"]](s)


def _own_cache(s):
    cfi, c, st = _cfi(), s["case"], s["stream"]
    cfi.paged_kv_store(s["cache"], s["k"].data_ptr(), s["v"].data_ptr(), s["new"].data_ptr(), c["tokens"], src_type=c["src"], stream=st)
    if c["type"] == F16:
        return s["k_pool"], s["v_pool"]
    cfi.paged_kv_load(s["cache"], s["slots"].data_ptr(), s["k_rows"].data_ptr(), s["v_rows"].data_ptr(),
                      c["tokens"] + c["context"], stream=st)
    return s["k_rows"], s["v_rows"]


def _own_decode(s):
    c = s["case"]
    _cfi().paged_attention(s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(),
                           c["batch"], c["heads"], s["width"], s["scale"], q_type=F16, out_type=F16, stream=s["stream"])
    return s["out"]


def _own_prompt(s):
    c = s["case"]
    _cfi().packed_attention(s["q"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), s["out"].data_ptr(), s["cu_q"].data_ptr(),
                            s["cu_k"].data_ptr(), c["batch"], s["tq"], s["tk"], c["heads"], c["heads_kv"], c["dim"], s["scale"],
                            causal=True, out_type=F16, stream=s["stream"])
    return s["out"]


def _own_sample(s):
    c = s["case"]
    _cfi().sample(s["logits"].data_ptr(), s["u"].data_ptr(), s["token"].data_ptr(), c["rows"], c["vocab"],
                  temperature=s["temperature"].data_ptr(), top_k=s["top_k"].data_ptr(), top_p=s["top_p"].data_ptr(),
                  min_p=s["min_p"].data_ptr(), logprob=s["logprob"].data_ptr(), stream=s["stream"])
    return s["token"], s["logprob"]


_run_own = {"cache": _own_cache, "decode": _own_decode, "prompt": _own_prompt, "sample": _own_sample}


def _q8_0(x):
    """Blocks of 32 along the last axis: whole numbers of at most 127 and the block's scale, rounded to f16."""
    b = x.float().unflatten(-1, (-1, 32))
    d = b.abs().amax(-1, keepdim=True) / 127.0
    q = torch.where(d > 0, b * (1.0 / d), 0.0).round().clamp(-127, 127)
    return q.flatten(-2), d.half().squeeze(-1)


def _rows(pool, kind, dim, page):
    """A pool, or pages of it, as f32 [..., head, slot, dim]."""
    if kind == F16:
        return pool.float()
    q = pool[..., : page * dim].view(torch.int8).unflatten(-1, (page, dim // 32, 32)).float()
    d = pool[..., page * dim:].view(torch.float16).unflatten(-1, (page, dim // 32, 1)).float()
    return (q * d).flatten(-2)


def _plain_cache(s):
    c = s["case"]
    dim, page = c["dim"], c["page"]
    at, off = s["new"] // page, s["new"] % page
    for_both = []
    for new, pool in ((s["k"], s["k_pool"]), (s["v"], s["v_pool"])):  # K and V
        if c["type"] == F16:
            pool[at, :, off] = new.half()
            for_both.append(pool)
            continue
        q, d = _q8_0(new)
        quants = pool[..., : page * dim].view(torch.int8).unflatten(-1, (page, dim))
        scales = pool[..., page * dim:].view(torch.float16).unflatten(-1, (page, dim // 32))
        quants[at, :, off] = q.to(torch.int8)
        scales[at, :, off] = d
        p, o = s["slots"] // page, s["slots"] % page
        for_both.append((quants[p, :, o].unflatten(-1, (-1, 32)).float() * scales[p, :, o].float()[..., None]).flatten(-2).half())
    return tuple(for_both)


def _plain_decode(s):
    c = s["case"]
    dim, page, kv = c["dim"], c["page"], c["heads_kv"]
    t = s["table"].long()
    k = _rows(s["k_pool"][t], c["type"], dim, page).transpose(1, 2).flatten(2, 3)  # [batch, head, position, dim]
    q = s["q"].float().unflatten(1, (kv, -1))
    x = (q @ k.transpose(2, 3)) * s["scale"]
    del k
    live = (torch.arange(x.shape[-1], device=DEV)[None] < s["lens"][:, None])[:, None, None]
    x = torch.where(live, x, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    v = _rows(s["v_pool"][t], c["type"], dim, page).transpose(1, 2).flatten(2, 3)
    return ((p @ v) / p.sum(-1, keepdim=True)).flatten(1, 2).half()


def _padded(x, cu, longest, heads):
    """Packed [token, head, dim] as f32 [sequence, head, position, dim]; what is past a sequence's end is another's."""
    at = (cu[:-1, None].long() + torch.arange(longest, device=DEV)[None]).clamp_max(x.shape[0] - 1)
    return x[at].float().transpose(1, 2)


def _plain_prompt(s):
    c = s["case"]
    kv, lq, lk = c["heads_kv"], s["lq"], s["lk"]
    nq, nk = s["cu_q"].diff().long(), s["cu_k"].diff().long()
    q = _padded(s["q"], s["cu_q"], lq, c["heads"]).unflatten(1, (kv, -1)).flatten(2, 3)
    k = _padded(s["k"], s["cu_k"], lk, kv)
    x = ((q * s["scale"]) @ k.transpose(2, 3)).unflatten(2, (-1, lq))  # [sequence, kv head, head, query, key]
    i, j = torch.arange(lq, device=DEV), torch.arange(lk, device=DEV)
    seen = (j[None, None] <= i[None, :, None] + (nk - nq)[:, None, None])[:, None, None]
    x.masked_fill_(~seen, float("-inf"))
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    o = (x.flatten(2, 3) @ _padded(s["v"], s["cu_k"], lk, kv)).unflatten(2, (-1, lq)) / x.sum(-1, keepdim=True)
    token = torch.arange(s["tq"], device=DEV)
    seq = torch.searchsorted(s["cu_q"][1:].long(), token, right=True)
    o = o.flatten(1, 2)[seq, :, token - s["cu_q"].long()[seq]]
    return o.half()


def _plain_sample(s):
    t = s["temperature"][:, None]
    greedy = t <= 0
    z = s["logits"] / torch.where(greedy, 1.0, t)
    zs, order = z.sort(dim=1, descending=True, stable=True)
    e = torch.exp(zs - zs[:, :1])
    w = (e * UNIT).long()
    rank = torch.arange(z.shape[1], device=DEV)[None]
    k = torch.where(s["top_k"] > 0, s["top_k"], z.shape[1])[:, None]
    w = torch.where((rank < k) & ~(greedy & (rank > 0)), w, 0)
    before = w.cumsum(1) - w
    keep = (before.double() < s["top_p"].double()[:, None] * w.sum(1, keepdim=True).double()) & (e >= s["min_p"][:, None])
    w = torch.where(keep | (rank == 0), w, 0)
    total = w.sum(1)
    w = torch.zeros_like(w).scatter_(1, order, w)
    target = (s["u"].double() * total.double()).long()
    token = (w.cumsum(1) <= target[:, None]).sum(1)
    logprob = (z.gather(1, token[:, None]) - zs[:, :1])[:, 0] - torch.log((total.double() / UNIT).float())
    return token.int(), logprob


_run_plain = {"cache": _plain_cache, "decode": _plain_decode, "prompt": _plain_prompt, "sample": _plain_sample}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "sample":
        return None, _exact_logprob(s)
    if op == "cache":
        return _exact_cache(s)
    return (_exact_decode if op == "decode" else _exact_prompt)(s)


def _exact_blocks(x):
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    d = b.abs().max(-1, keepdim=True).values / 127
    return ((b / d).round() * d.half().double()).reshape(x.shape)


def _exact_pool(pool, case):
    """Every slot's row in 64 bits: [slot, head, dim]."""
    dim, page, kv = case["dim"], case["page"], case["heads_kv"]
    if case["type"] == F16:
        x = pool.double()
    else:
        flat = pool.reshape(-1, pool.shape[-1])
        q = flat[:, : page * dim].contiguous().view(torch.int8).double()
        d = flat[:, page * dim:].contiguous().view(torch.float16).double()
        x = (q * d.repeat_interleave(32, 1)).reshape(-1, kv, page, dim)
    return x.permute(0, 2, 1, 3).reshape(-1, kv, dim)


def _exact_cache(s):
    case, out = s["case"], []
    for new, pool in ((s["k"], s["k_pool"]), (s["v"], s["v_pool"])):
        rows = _exact_pool(pool, case)
        rows[s["new"]] = new.double() if case["type"] == F16 else _exact_blocks(new)
        if case["type"] == F16:
            out.append(rows.reshape(s["pages"], case["page"], case["heads_kv"], case["dim"]).permute(0, 2, 1, 3).contiguous())
        else:
            out.append(rows[s["slots"]])
    return tuple(out)


def _attend(q, k, v, scale, first=None):
    """softmax(scale q k') v for [query, dim] and [key, dim] in 64 bits; query i sees the keys up to first + i."""
    x = (q @ k.T) * scale
    if first is not None:
        x += torch.full_like(x, -math.inf).triu(first + 1)
    return torch.softmax(x, -1) @ v


def _exact_decode(s):
    case = s["case"]
    group = case["heads"] // case["heads_kv"]
    out = torch.zeros(case["batch"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    k, v = _exact_pool(s["k_pool"], case), _exact_pool(s["v_pool"], case)
    for b, n in enumerate(_lengths(case)):
        pos = torch.arange(n, device=DEV)
        slot = s["table"][b].long()[pos // case["page"]] * case["page"] + pos % case["page"]
        for h in range(case["heads_kv"]):
            mine = slice(h * group, (h + 1) * group)
            out[b, mine] = _attend(s["q"][b, mine].double(), k[slot, h], v[slot, h], s["scale"])
    return out


def _exact_prompt(s):
    case = s["case"]
    group = case["heads"] // case["heads_kv"]
    out = torch.zeros(s["tq"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    a, b = 0, 0
    for n, c in zip(_lengths(case), _contexts(case)):
        for h in range(case["heads"]):
            k, v = (s[x][b:b + n + c, h // group].double() for x in "kv")
            for i in range(0, n, 4096):
                m = min(n, i + 4096)
                out[a + i:a + m, h] = _attend(s["q"][a + i:a + m, h].double(), k[:c + m], v[:c + m], s["scale"], c + i)
        a, b = a + n, b + n + c
    return out


def _exact_logprob(s):
    """The log probability of the token that the definition takes, for each row."""
    t = s["temperature"].double().cpu().numpy()
    out = np.zeros(len(t))
    for r, u in enumerate(s["u"].double().cpu().numpy()):
        z = s["logits"][r].double().cpu().numpy()
        best = int(z.argmax())
        if t[r] <= 0:
            continue
        z = z / t[r]
        order = np.argsort(-z, kind="stable")
        k = int(s["top_k"][r])
        order = order[:k] if k > 0 else order
        e = np.exp(z[order] - z[best])
        before = np.cumsum(e) - e
        keep = (before < float(s["top_p"][r]) * e.sum()) & (e >= float(s["min_p"][r]))
        keep[0] = True
        order = np.sort(order[keep])
        e = np.exp(z[order] - z[best])
        at = min(int((np.cumsum(e) <= u * e.sum()).sum()), len(order) - 1)
        out[r] = np.log(e[at]) - np.log(e.sum())
    return torch.from_numpy(out)
