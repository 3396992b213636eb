"""Cases of the operators beside the paged cache: a cache held in 4 bits with the attention that reads
it, the rows' bias, norm and rotation on their way into a cache, and page tables built on the GPU.

A case names its operator in "op":
  cache4   new rows of K and V go into a Q4_1 cache, and a context is read back from it as f16 rows
  decode4  one new token for each sequence attends to the sequence's pages of a Q4_1 cache
  rotate   a product's rows of q, k and v: bias, norm of each head, rotation; q comes out, k and v go into a cache's slots
  place    a batch's new tokens get pages, slots and positions; then the sequences are cut back to
           where they were, as after drafted tokens that were not taken

Head counts and widths are those of the decode configurations (14 query and 2 key-value heads of 64,
12 and 2 of 128) and a generic 32 and 8 of 128.
"""
import math
import os
import random
import sys

import torch

own = False

F32, F16, Q4_1 = 0, 1, 3
DEV = "cuda"


def listed():
    return [
        # one decode step of 48 sequences: latency
        dict(name="cache4 step", op="cache4", src=F32, tokens=48, context=0, heads_kv=2, dim=64, page=16, spare=464),
        # a short odd chunk after a short context
        dict(name="cache4 chunk", op="cache4", src=F32, tokens=333, context=298, heads_kv=2, dim=128, page=32, spare=7),
        # a chunk of a long prompt after a long context
        dict(name="cache4 long", op="cache4", src=F16, tokens=8192, context=57345, heads_kv=8, dim=128, page=64, spare=100),
        # a single user's token: latency
        dict(name="decode4 one", op="decode4", q=F32, heads=14, heads_kv=2, dim=64, page=16, batch=1, lo=672, hi=672, lens=1),
        # a batch of chats whose lengths differ
        dict(name="decode4 batch", op="decode4", q=F32, heads=12, heads_kv=2, dim=128, page=16, batch=64, lo=16, hi=4096, lens=2),
        # a few long documents
        dict(name="decode4 long", op="decode4", q=F16, heads=32, heads_kv=8, dim=128, page=64, batch=8, lo=9000, hi=65000, lens=3),
        # a decode step of 48 sequences with biases
        dict(name="rotate step", op="rotate", src=F32, out=F32, tokens=48, seqs=48, heads=14, heads_kv=2, dim=64, turned=64, norm=False,
             bias=True, far=4096, page=16, spare=100),
        # a prompt of 631 tokens, normed
        dict(name="rotate prompt", op="rotate", src=F32, out=F16, tokens=631, seqs=1, heads=12, heads_kv=2, dim=128, turned=128, norm=True,
             bias=False, far=1, page=16, spare=9),
        # a chunk of 8191 tokens of long documents, normed, half of each head turned
        dict(name="rotate long", op="rotate", src=F32, out=F16, tokens=8191, seqs=4, heads=32, heads_kv=8, dim=128, turned=64, norm=True,
             bias=True, far=100000, page=64, spare=50),
        # the next token of 64 sequences of 100, in a batch padded to 72 tokens
        dict(name="place step", op="place", batch=64, rows=100, page=16, width=256, lo=16, hi=4000, new_lo=1, new_hi=1, pad=8, context=False,
             lens=4),
        # sixteen prompts' chunks, some after an earlier context
        dict(name="place prompts", op="place", batch=16, rows=40, page=32, width=300, lo=1, hi=5000, new_lo=1, new_hi=2048, pad=0, context=True,
             lens=5),
        # chunks of a large batch with the slots of all its contexts
        dict(name="place large", op="place", batch=1024, rows=2000, page=16, width=700, lo=100, hi=8000, new_lo=1, new_hi=200, pad=100,
             context=True, lens=6),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["cache4", "decode4", "rotate", "place"])
    heads, kv, dim = rng.choice([(14, 2, 64), (12, 2, 128), (32, 8, 128), (16, 16, 64), (9, 3, 64), (16, 1, 128)])
    page, spread = rng.choice([16, 32, 64, 128]), rng.randrange(1, 1 << 20)
    if op == "cache4":
        return dict(op=op, src=rng.choice([F32, F16]), tokens=_log(rng, 1, 8000), context=rng.choice([0, _log(rng, 1, 40000)]),
                    heads_kv=min(kv, 8), dim=dim, page=page, spare=rng.randrange(1, 200))
    if op == "decode4":
        batch = _log(rng, 1, 128)
        hi = _log(rng, 1, max(1, min(65000, 220_000_000 // (batch * kv * dim))))
        return dict(op=op, q=rng.choice([F32, F16]), heads=heads, heads_kv=kv, dim=dim, page=page, batch=batch, lo=_log(rng, 1, hi), hi=hi,
                    lens=spread)
    if op == "rotate":
        tokens = _log(rng, 1, 8191 * 48 * 128 // ((heads + 2 * kv) * dim))
        return dict(op=op, src=rng.choice([F32, F16]), out=rng.choice([F32, F16]), tokens=tokens, seqs=_log(rng, 1, min(tokens, 64)),
                    heads=heads, heads_kv=kv, dim=dim, turned=rng.choice([dim, dim, dim // 2]), norm=rng.random() < 0.6,
                    bias=rng.random() < 0.5, far=_log(rng, 1, 130000), page=page, spare=rng.randrange(1, 60))
    batch = _log(rng, 1, 1024)
    hi = _log(rng, 1, min(8000, 1_800_000 // batch))
    new = rng.choice([1, _log(rng, 1, max(1, 36_000 // batch))])
    return dict(op=op, batch=batch, rows=batch + rng.randrange(1, 200), page=page, width=(hi + new) // page + rng.randrange(1, 60),
                lo=_log(rng, 1, hi), hi=hi, new_lo=_log(rng, 1, new), new_hi=new, pad=rng.choice([0, rng.randrange(1, 100)]),
                context=rng.random() < 0.5, lens=spread)


def _spread(case, lo, hi, n, salt=0):
    """n numbers over the logarithm of lo..hi, one of them hi."""
    r = random.Random(case["lens"] + salt)
    x = [_log(r, lo, hi) for _ in range(n)]
    x[r.randrange(n)] = hi
    return x


def _place_sizes(case):
    """What each row of the table holds, which rows are in the batch, and how many tokens each gets."""
    r = random.Random(case["lens"] + 2)
    held = [h if r.random() < 0.9 else 0 for h in _spread(case, case["lo"], case["hi"], case["rows"])]
    rows = r.sample(range(case["rows"]), case["batch"])
    return held, rows, _spread(case, case["new_lo"], case["new_hi"], case["batch"], 1)


def work(case):
    op = case["op"]
    if op == "place":
        held, rows, new = _place_sizes(case)
        page, after = case["page"], [held[r] + n for r, n in zip(rows, new)]
        tokens, pages = sum(new) + case["pad"], sum(-(-a // page) for a in after)
        n = 16 * case["batch"] + 4 * pages + 4 * pages + 12 * tokens + 8 * (sum(after) if case["context"] else 0)
        return {"bytes": n, "flops": 4 * tokens + 2 * case["batch"]}
    dim = case["dim"]
    row = case["heads_kv"] * dim * 2  # values of K and V of one position
    held = row * 5 / 8
    if op == "cache4":
        n = case["tokens"] * (row * (4 if case["src"] == F32 else 2) + held + 8)
        n += (case["tokens"] + case["context"]) * (row * 2 + 8) + case["context"] * held
        return {"bytes": n, "flops": 6 * case["tokens"] * row}
    if op == "rotate":
        q = case["heads"] * dim
        n = case["tokens"] * ((q + row) * (4 if case["src"] == F32 else 2) + q * (4 if case["out"] == F32 else 2) + row * 2 + 12)
        return {"bytes": n, "flops": case["tokens"] * 8 * (q + row // 2)}
    lens = _spread(case, case["lo"], case["hi"], case["batch"])
    q = case["batch"] * case["heads"] * dim * (4 if case["q"] == F32 else 2)
    return {"bytes": sum(lens) * held + 2 * q + sum(4 * -(-n // case["page"]) + 4 for n in lens),
            "flops": 4 * sum(lens) * case["heads"] * dim}


# ---- a Q4_1 pool: [page][kv head][tile of 16 positions][nibbles of 16 rows, then 16 rows of f16 scales and minima] ----
def _places(dim, of_v):
    """Where byte n of each of a tile's rows (dims 2n and 2n + 1) lies among the tile's nibbles: [16, dim / 2]."""
    n = torch.arange(dim // 2, device=DEV)
    block, at = n // 16, n % 16
    row = torch.arange(16, device=DEV)[:, None]
    if not of_v:  # four groups, of each block 8 dims
        inside = (at // 4) * (dim // 8) + 4 * block + at % 4
        return row * (dim // 2) + inside[None]
    group = (at // 2)[None].expand(16, -1)  # eight groups, of each block 4 dims
    if dim == 128:
        group = group ^ (4 * (row >> 1 & 1))
    return row * (dim // 2) + group * (dim // 16) + (2 * block + at % 2)[None]


def _pack(q, d, m, of_v):
    """Whole numbers [..., position, dim] and f16 scales and minima [..., position, block] as the bytes of tiles."""
    dim = q.shape[-1]
    both = q.to(torch.uint8).unflatten(-1, (-1, 2))
    both = (both[..., 0] | both[..., 1] << 4).unflatten(-2, (-1, 16)).flatten(-2)
    nibbles = torch.empty_like(both)
    nibbles[..., _places(dim, of_v).flatten()] = both
    params = torch.cat([d, m], -1).unflatten(-2, (-1, 16)).flatten(-2).contiguous().view(torch.uint8)
    return torch.cat([nibbles, params], -1).flatten(-2)


def _unpack(pool, dim, of_v):
    """Pages of a pool as q (uint8) [..., position, dim] and f16 scales and minima [..., position, block]."""
    tiles = pool.unflatten(-1, (-1, dim * 10))
    both = tiles[..., :dim * 8].index_select(-1, _places(dim, of_v).flatten())
    q = torch.stack([both & 15, both >> 4], -1).flatten(-2).unflatten(-1, (16, dim)).flatten(-3, -2)
    params = tiles[..., dim * 8:].contiguous().view(torch.float16).unflatten(-1, (16, dim // 16)).flatten(-3, -2)
    return q, params[..., :dim // 32], params[..., dim // 32:]


def _half(x):
    """64-bit numbers rounded once to f16."""
    e = torch.frexp(x)[1]
    ulp = torch.ldexp(torch.ones_like(x), torch.clamp_min(e - 11, -24))
    return ((x / ulp).round() * ulp).half()


def _q4_1(x):
    """Blocks of 32 along the last axis: q of 0..15, scale and minimum rounded to f16."""
    b = x.double().unflatten(-1, (-1, 32))
    lo, hi = b.amin(-1, keepdim=True), b.amax(-1, keepdim=True)
    q = torch.where(hi > lo, (b - lo) * 15.0 / (hi - lo) + 0.5, 0.0).floor()
    return q.flatten(-2), _half((hi - lo) / 15.0).squeeze(-1), _half(lo).squeeze(-1)


def _values(q, d, m):
    return (q.float().unflatten(-1, (-1, 32)) * d.float()[..., None] + m.float()[..., None]).flatten(-2)


# ---- inputs ----
def _pool4(case, pages, g, of_v):
    """Pages of random rows; those of K about an offset of each channel's own."""
    out = []
    for n in range(0, pages, 2048):
        x = torch.randn(min(2048, pages - n), case["heads_kv"], case["page"], case["dim"], generator=g, device=DEV)
        if not of_v:
            gc = torch.Generator(device=DEV)
            gc.manual_seed(case["heads_kv"])
            x += torch.randn(case["heads_kv"], 1, case["dim"], generator=gc, device=DEV)
        out.append(_pack(*_q4_1(x), of_v))
    return torch.cat(out)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV)  # noqa: E731
    op = case["op"]
    s = {"case": case, "stream": torch.cuda.current_stream().cuda_stream}
    if op == "place":
        return _prepare_place(s, case, g)
    dim, kv = case["dim"], case["heads_kv"]
    if op == "cache4":
        n = case["tokens"] + case["context"]
        pages = -(-n // case["page"]) + case["spare"]
        s["k_pool"], s["v_pool"] = _pool4(case, pages, g, False), _pool4(case, pages, g, True)
        order = torch.randperm(pages, generator=g, device=DEV)
        pos = torch.arange(n, device=DEV)
        s["slots"] = (order[pos // case["page"]] * case["page"] + pos % case["page"]).contiguous()
        s["new"] = s["slots"][case["context"]:].contiguous()
        t = torch.float32 if case["src"] == F32 else torch.float16
        s["k"], s["v"] = rand(case["tokens"], kv, dim).to(t), rand(case["tokens"], kv, dim).to(t)
        s["k_rows"], s["v_rows"] = (torch.empty(n, kv, dim, dtype=torch.float16, device=DEV) for _ in "kv")
        s["pages"] = pages
        return _bind(s)
    if op == "rotate":
        n, heads = case["tokens"], case["heads"]
        t = torch.float32 if case["src"] == F32 else torch.float16
        s["qkv"] = (rand(n, (heads + 2 * kv) * dim) * 2.0).to(t)
        s["bias"] = rand((heads + 2 * kv) * dim) * 0.5 if case["bias"] else None
        s["norm"] = [1.0 + 0.2 * rand(dim), 1.0 + 0.2 * rand(dim)] if case["norm"] else None
        begin = torch.randint(0, case["far"], (case["seqs"],), generator=g, device=DEV)
        token = torch.arange(n, device=DEV)
        each = -(-n // case["seqs"])
        s["pos"] = (begin[token // each] + token % each).to(torch.int32)
        pages = -(-n // case["page"]) + case["spare"]
        s["slots"] = torch.randperm(pages * case["page"], generator=g, device=DEV)[:n].contiguous()
        s["k_pool"], s["v_pool"] = (rand(pages, kv, case["page"], dim).half() for _ in "kv")
        s["q_out"] = torch.empty(n, heads, dim, dtype=torch.float32 if case["out"] == F32 else torch.float16, device=DEV)
        s.update(pages=pages, eps=1e-6, base=1e6)
        return _bind(s)
    lens = _spread(case, case["lo"], case["hi"], case["batch"])
    need = [-(-n // case["page"]) for n in lens]
    width, pages = max(need), sum(need) + 3
    s["k_pool"], s["v_pool"] = _pool4(case, pages, g, False), _pool4(case, pages, g, True)
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    start = torch.tensor([0] + need, device=DEV).cumsum(0)[:-1]
    at = torch.arange(width, device=DEV)[None] + start[:, None]
    s["table"] = torch.where(torch.arange(width, device=DEV)[None] < torch.tensor(need, device=DEV)[:, None],
                             order[at.clamp_max(pages - 1)], 0).to(torch.int32).contiguous()
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    s["q"] = (rand(case["batch"], case["heads"], dim) * 1.5).to(torch.float32 if case["q"] == F32 else torch.float16)
    s["out"] = torch.empty_like(s["q"])
    s.update(pages=pages, width=width, scale=1.0 / math.sqrt(dim))
    return _bind(s)


def _prepare_place(s, case, g):
    held, rows, new = _place_sizes(case)
    page, width = case["page"], case["width"]
    need = [-(-h // page) for h in held]
    more = sum(-(-(held[r] + n) // page) - need[r] for r, n in zip(rows, new))
    pages = sum(need) + more + 5
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    nt = i32(need).long()
    start = nt.cumsum(0) - nt
    at = torch.arange(width, device=DEV)[None] + start[:, None]
    s["table"] = torch.where(torch.arange(width, device=DEV)[None] < nt[:, None], order[at.clamp_max(pages - 1)], 0).to(torch.int32).contiguous()
    s["free"] = torch.zeros(pages, dtype=torch.int32, device=DEV)
    s["free"][:pages - sum(need)] = order[sum(need):]
    s["n_free"] = i32([pages - sum(need)])
    s["cached"], s["rows"], s["new"] = i32(held), i32(rows), i32(new)
    s["before"] = s["cached"][s["rows"].long()].contiguous()
    b, tokens = case["batch"], sum(new) + case["pad"]
    context = sum(held[r] + n for r, n in zip(rows, new)) if case["context"] else 0
    zeros = lambda n, t=torch.int32: torch.zeros(n, dtype=t, device=DEV)  # noqa: E731
    s.update(lens_out=zeros(b), batch_table=torch.zeros(b, width, dtype=torch.int32, device=DEV), cu_q=zeros(b + 1), cu_kv=zeros(b + 1),
             slots=zeros(tokens, torch.int64), positions=zeros(tokens), context=zeros(context, torch.int64), status=zeros(2),
             pages=pages, tokens=tokens, n_context=context)
    if own:
        s["held"] = _cfi().page_table(s["table"].data_ptr(), s["cached"].data_ptr(), s["free"].data_ptr(), s["n_free"].data_ptr(),
                                      case["rows"], width, page, pages)
        s["described"] = _cfi().page_batch(s["rows"].data_ptr(), s["new"].data_ptr(), b, s["lens_out"].data_ptr(),
                                           s["batch_table"].data_ptr(), s["cu_q"].data_ptr(), s["cu_kv"].data_ptr(), s["slots"].data_ptr(),
                                           s["positions"].data_ptr(), tokens, s["status"].data_ptr(),
                                           context=s["context"].data_ptr() if context else 0, max_context=context)
    return s


def _bind(s):
    """The descriptions of its cache and rows that a program keeps beside their buffers."""
    if not own:
        return s
    cfi, c = _cfi(), s["case"]
    s["cache"] = cfi.paged_cache(F16 if c["op"] == "rotate" else Q4_1, s["k_pool"].data_ptr(), s["v_pool"].data_ptr(), s["pages"],
                                 c["page"], c["heads_kv"], c["dim"])
    if c["op"] == "rotate":
        size = s["qkv"].element_size()
        nq, nkv = c["heads"] * c["dim"], c["heads_kv"] * c["dim"]
        width, q = nq + 2 * nkv, s["qkv"].data_ptr()
        b = s["bias"].data_ptr() if c["bias"] else 0
        s["described"] = cfi.norm_rope_rows(
            q, s["q_out"].data_ptr(), s["pos"].data_ptr(), c["tokens"], c["heads"], c["dim"], k=q + nq * size, v=q + (nq + nkv) * size,
            n_kv_head=c["heads_kv"], slots=s["slots"].data_ptr(), in_type=c["src"], q_out_type=c["out"], q_bias=b,
            k_bias=b + 4 * nq if b else 0, v_bias=b + 4 * (nq + nkv) if b else 0, q_norm=s["norm"][0].data_ptr() if c["norm"] else 0,
            k_norm=s["norm"][1].data_ptr() if c["norm"] else 0, eps=s["eps"], n_rot=c["turned"], freq_base=s["base"], q_stride=width,
            k_stride=width, v_stride=width)
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


def _own_cache4(s):
    cfi, c, st = _cfi(), s["case"], s["stream"]
    cfi.paged_kv_store(s["cache"], s["k"].data_ptr(), s["v"].data_ptr(), s["new"].data_ptr(), c["tokens"], src_type=c["src"], stream=st)
    cfi.paged_kv_load(s["cache"], s["slots"].data_ptr(), s["k_rows"].data_ptr(), s["v_rows"].data_ptr(),
                      c["tokens"] + c["context"], stream=st)
    return s["k_rows"], s["v_rows"]


def _own_decode4(s):
    c = s["case"]
    _cfi().paged_attention(s["cache"], s["q"].data_ptr(), s["out"].data_ptr(), s["table"].data_ptr(), s["lens"].data_ptr(),
                           c["batch"], c["heads"], s["width"], s["scale"], q_type=c["q"], out_type=c["q"], stream=s["stream"])
    return s["out"]


def _own_rotate(s):
    _cfi().norm_rope(s["described"], s["cache"], stream=s["stream"])
    return s["q_out"], s["k_pool"], s["v_pool"]


def _place_outputs(s):
    return (s["status"], s["lens_out"], s["cu_q"], s["cu_kv"], s["batch_table"], s["slots"], s["positions"], s["context"], s["table"],
            s["cached"], s["free"], s["n_free"])


def _own_place(s):
    cfi, c, st = _cfi(), s["case"], s["stream"]
    cfi.paged_place(s["held"], s["described"], stream=st)
    cfi.paged_trim(s["held"], s["rows"].data_ptr(), s["before"].data_ptr(), c["batch"], s["status"].data_ptr() + 4, stream=st)
    return _place_outputs(s)


_run_own = {"cache4": _own_cache4, "decode4": _own_decode4, "rotate": _own_rotate, "place": _own_place}


def _plain_cache4(s):
    c = s["case"]
    dim, page, out = c["dim"], c["page"], []
    at, off = s["new"] // page, s["new"] % page
    p, o = s["slots"] // page, s["slots"] % page
    for new, pool, of_v in ((s["k"], s["k_pool"], False), (s["v"], s["v_pool"], True)):
        tiles = pool.view(*pool.shape[:2], page // 16, dim * 10)
        places = _places(dim, of_v)
        q, d, m = _q4_1(new)
        both = q.to(torch.uint8).unflatten(-1, (-1, 2))
        both = both[..., 0] | both[..., 1] << 4
        head = torch.arange(c["heads_kv"], device=DEV)[None, :, None]
        tiles[at[:, None, None], head, (off // 16)[:, None, None], places[off % 16][:, None]] = both
        params = torch.cat([d, m], -1).contiguous().view(torch.uint8)
        behind = dim * 8 + (off % 16)[:, None] * (dim // 8) + torch.arange(dim // 8, device=DEV)[None]
        tiles[at[:, None, None], head, (off // 16)[:, None, None], behind[:, None]] = params
        both = tiles[p[:, None, None], head, (o // 16)[:, None, None], places[o % 16][:, None]]
        q = torch.stack([both & 15, both >> 4], -1).flatten(-2)
        behind = dim * 8 + (o % 16)[:, None] * (dim // 8) + torch.arange(dim // 8, device=DEV)[None]
        params = tiles[p[:, None, None], head, (o // 16)[:, None, None], behind[:, None]].view(torch.float16)
        out.append(_values(q, params[..., :dim // 32], params[..., dim // 32:]).half())
    return tuple(out)


def _plain_decode4(s):
    c = s["case"]
    kv = c["heads_kv"]
    t = s["table"].long()
    k = _values(*_unpack(s["k_pool"][t], c["dim"], False)).transpose(1, 2).flatten(2, 3)  # [batch, head, position, dim]
    q = s["q"].float().unflatten(1, (kv, -1))
    x = (q @ k.transpose(2, 3)) * s["scale"]
    del k
    live = (torch.arange(x.shape[-1], device=DEV)[None] < s["lens"][:, None])[:, None, None]
    x = torch.where(live, x, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True))
    v = _values(*_unpack(s["v_pool"][t], c["dim"], True)).transpose(1, 2).flatten(2, 3)
    return ((p @ v) / p.sum(-1, keepdim=True)).flatten(1, 2).to(s["q"].dtype)


def _plain_rotate(s):
    c = s["case"]
    heads, kv, dim, turned = c["heads"], c["heads_kv"], c["dim"], c["turned"]
    x = s["qkv"].float()
    if c["bias"]:
        x = x + s["bias"]
    x = x.unflatten(1, (-1, dim))
    q, k, v = x.split([heads, kv, kv], 1)
    i = torch.arange(turned // 2, device=DEV, dtype=torch.float64)
    angle = s["pos"].double()[:, None, None] * torch.pow(torch.tensor(s["base"], dtype=torch.float64, device=DEV), -2.0 * i / turned)
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    done = []
    for n, y in enumerate((q, k)):
        if c["norm"]:
            y = y * torch.rsqrt((y * y).mean(-1, keepdim=True) + s["eps"]) * s["norm"][n]
        a, b, rest = y[..., :turned // 2], y[..., turned // 2:turned], y[..., turned:]
        done.append(torch.cat([a * cos - b * sin, a * sin + b * cos, rest], -1))
    s["q_out"].copy_(done[0])
    at, off = s["slots"] // c["page"], s["slots"] % c["page"]
    s["k_pool"][at, :, off] = done[1].half()
    s["v_pool"][at, :, off] = v.half()
    return s["q_out"], s["k_pool"], s["v_pool"]


def _plain_place(s):
    c = s["case"]
    page, width, pages, rows = c["page"], c["width"], s["pages"], s["rows"].long()
    cached = s["cached"][rows].long()
    after = cached + s["new"]
    old, need = (cached + page - 1) // page, (after + page - 1) // page
    first = (need - old).cumsum(0) - (need - old)  # of the pages that a sequence takes
    taken = (need - old).sum()
    # nothing of what refuses a batch happens here: a program that makes its own tables knows its sizes
    j = torch.arange(width, device=DEV)[None]
    new = s["free"].long()[(s["n_free"].long() - 1 - first[:, None] - (j - old[:, None])).clamp(0, pages - 1)]
    mine = torch.where(j < old[:, None], s["table"][rows].long(), torch.where(j < need[:, None], new, 0))
    inside = j < need[:, None]
    s["table"][rows] = torch.where(inside, mine, s["table"][rows].long()).int()
    s["batch_table"].copy_(torch.where(inside, mine, s["batch_table"].long()))
    s["lens_out"].copy_(after)
    s["cu_q"][1:] = s["new"].cumsum(0)
    s["cu_kv"][1:] = after.cumsum(0)

    def slots_of(n, cu, begin):
        i = torch.arange(n, device=DEV)
        seq = torch.searchsorted(cu[1:].long(), i, right=True).clamp_max(c["batch"] - 1)
        pos = begin[seq] + i - cu[seq]
        slot = mine[seq, (pos // page).clamp_max(width - 1)] * page + pos % page
        return torch.where(i < cu[-1], slot, -1), torch.where(i < cu[-1], pos, 0)

    slot, pos = slots_of(s["tokens"], s["cu_q"], cached)
    s["slots"].copy_(slot)
    s["positions"].copy_(pos)
    if c["context"]:
        s["context"].copy_(slots_of(s["n_context"], s["cu_kv"], torch.zeros_like(cached))[0])
    s["cached"][rows] = after.int()
    s["n_free"] -= taken.int()
    # and back: the pages behind the old lengths, the last of the last sequence first
    back = (j >= old[:, None]) & inside
    at = s["n_free"].long() + taken - 1 - (first[:, None] + j - old[:, None])
    free = torch.cat([s["free"], s["n_free"]])  # one more place, for what does not go back
    free.scatter_(0, torch.where(back, at, pages).flatten(), mine.int().flatten())
    s["free"].copy_(free[:pages])
    s["n_free"] += taken.int()
    s["cached"][rows] = cached.int()
    s["status"].zero_()
    return _place_outputs(s)


_run_plain = {"cache4": _plain_cache4, "decode4": _plain_decode4, "rotate": _plain_rotate, "place": _plain_place}


# ---- the definitions in 64 bits ----
def exact(case, seed):
    op = case["op"]
    if op == "place":
        return None  # whole numbers
    s = prepare(case, seed)
    return {"cache4": _exact_cache4, "decode4": _exact_decode4, "rotate": _exact_rotate}[op](s)


def _exact_blocks(x):
    """What a block of 32 stands for: 15 borders, each met by what is not below it."""
    b = x.double().reshape(*x.shape[:-1], -1, 32)
    lo, hi = b.min(-1, keepdim=True).values, b.max(-1, keepdim=True).values
    q = torch.zeros_like(b)
    for i in range(1, 16):
        q += (30.0 * (b - lo) >= (2 * i - 1) * (hi - lo)) & (hi > lo)
    d, m = _nearest((hi - lo) / 15.0), _nearest(lo)
    return (q * d + m).reshape(x.shape)


def _nearest(x):
    """The f16 number nearest to each, ties to the even one, found among the neighbours of a first guess."""
    guess = x.half()
    best, off = guess.double(), (guess.double() - x).abs()
    bits = guess.view(torch.int16)
    for step in (-1, 1):
        other = (bits + step).view(torch.float16).double()
        far = (other - x).abs()
        take = (far < off) | ((far == off) & ((bits & 1) == 1))
        best, off = torch.where(take & torch.isfinite(other), other, best), torch.where(take & torch.isfinite(other), far, off)
    return best


def _exact_pool(pool, case, of_v):
    """Every slot's row in 64 bits: [slot, head, dim], dim by dim from where its nibble, scale and minimum lie."""
    dim, page, kv = case["dim"], case["page"], case["heads_kv"]
    tiles = pool.reshape(-1, kv, page // 16, dim * 10)
    words = tiles[..., dim * 8:].contiguous().view(torch.float16).double().reshape(*tiles.shape[:3], 16, 2, dim // 32)
    x = torch.empty(*tiles.shape[:3], 16, dim, dtype=torch.float64, device=DEV)
    for row in range(16):
        for i in range(dim):
            block, inside = i // 32, i % 32
            if of_v:
                group = inside // 4
                if dim == 128 and row & 2:
                    group ^= 4
                byte, odd = group * (dim // 16) + block * 2 + inside % 4 // 2, inside % 2
            else:
                byte, odd = inside // 8 * (dim // 8) + block * 4 + inside % 8 // 2, inside % 2
            n = (tiles[..., row * (dim // 2) + byte] >> (4 * odd)) & 15
            x[..., row, i] = n.double() * words[..., row, 0, block] + words[..., row, 1, block]
    return x.permute(0, 2, 3, 1, 4).reshape(-1, kv, dim)


def _exact_cache4(s):
    case, out = s["case"], []
    for new, pool, of_v in ((s["k"], s["k_pool"], False), (s["v"], s["v_pool"], True)):
        rows = _exact_pool(pool, case, of_v)
        rows[s["new"]] = _exact_blocks(new)
        out.append(rows[s["slots"]])
    return tuple(out)


def _exact_decode4(s):
    case = s["case"]
    group = case["heads"] // case["heads_kv"]
    out = torch.zeros(case["batch"], case["heads"], case["dim"], dtype=torch.float64, device=DEV)
    k, v = _exact_pool(s["k_pool"], case, False), _exact_pool(s["v_pool"], case, True)
    for b, n in enumerate(_spread(case, case["lo"], case["hi"], case["batch"])):
        pos = torch.arange(n, device=DEV)
        slot = s["table"][b].long()[pos // case["page"]] * case["page"] + pos % case["page"]
        for h in range(case["heads_kv"]):
            mine = slice(h * group, (h + 1) * group)
            out[b, mine] = torch.softmax((s["q"][b, mine].double() @ k[slot, h].T) * s["scale"], -1) @ v[slot, h]
    return out


def _exact_rotate(s):
    c = s["case"]
    heads, kv, dim, turned = c["heads"], c["heads_kv"], c["dim"], c["turned"]
    x = s["qkv"].double()
    if c["bias"]:
        x = x + s["bias"].double()
    x = x.reshape(c["tokens"], -1, dim)
    if c["norm"]:
        w = torch.ones(heads + kv, dim, dtype=torch.float64, device=DEV)
        w[:heads], w[heads:] = s["norm"][0].double(), s["norm"][1].double()
        y = x[:, :heads + kv]
        x[:, :heads + kv] = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / dim + s["eps"]) * w
    half = turned // 2
    rate = torch.tensor([math.pow(s["base"], -2.0 * i / turned) for i in range(half)], dtype=torch.float64, device=DEV)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=DEV), s["pos"].double()[:, None] * rate)[:, None]
    z = torch.complex(x[:, :heads + kv, :half], x[:, :heads + kv, half:turned]) * turn
    x[:, :heads + kv, :turned] = torch.cat([z.real, z.imag], -1)
    at, off = s["slots"] // c["page"], s["slots"] % c["page"]
    pools = []
    for pool, rows in ((s["k_pool"], x[:, heads:heads + kv]), (s["v_pool"], x[:, heads + kv:])):
        pool = pool.double()
        pool[at, :, off] = rows
        pools.append(pool)
    return x[:, :heads], pools[0], pools[1]
