"""cfi_paged_place and cfi_paged_trim (include/cfi_serve.h) against lists in Python: everything is whole numbers and has to be equal."""
import random

import numpy as np
import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = "cuda"


def stream():
    return torch.cuda.current_stream().cuda_stream


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


class Lists:
    """The definition: a stack and a list of pages for each row."""

    def __init__(self, rows, max_pages, page, pages, seed=0):
        self.rows, self.max_pages, self.page, self.n_pages = rows, max_pages, page, pages
        self.free = list(range(pages))
        random.Random(seed).shuffle(self.free)
        self.own = [[] for _ in range(rows)]
        self.cached = [0] * rows

    def why(self, rows, new, max_new, max_context):
        if len(set(rows)) < len(rows) or any(r < 0 or r >= self.rows for r in rows) or any(n < 0 for n in new):
            return cfi.PLACE_BAD_ROW
        after = [self.cached[r] + n for r, n in zip(rows, new)]
        if any(a > self.max_pages * self.page for a in after):
            return cfi.PLACE_TOO_LONG
        if sum(new) > max_new or (max_context is not None and sum(after) > max_context):
            return cfi.PLACE_NO_ROOM
        if sum(-(-a // self.page) - len(self.own[r]) for a, r in zip(after, rows)) > len(self.free):
            return cfi.PLACE_NO_PAGES
        return cfi.PLACED

    def place(self, rows, new):
        slots, positions, context = [], [], []
        for r, n in zip(rows, new):
            for p in range(self.cached[r], self.cached[r] + n):
                if p % self.page == 0:
                    self.own[r].append(self.free.pop())
                slots.append(self.own[r][p // self.page] * self.page + p % self.page)
                positions.append(p)
            self.cached[r] += n
            context += [self.own[r][p // self.page] * self.page + p % self.page for p in range(self.cached[r])]
        return slots, positions, context

    def trim(self, rows, keep):
        for r, k in list(zip(rows, keep))[::-1]:
            self.cached[r] = min(self.cached[r], max(k, 0))
            while len(self.own[r]) > -(-self.cached[r] // self.page):
                self.free.append(self.own[r].pop())


class Device:
    """The same state on the device, and buffers for a batch."""

    def __init__(self, m):
        self.m = m
        self.table = torch.full((m.rows, m.max_pages), -77, dtype=torch.int32, device=DEV)
        self.cached = i32([0] * m.rows)
        self.free = i32(m.free)
        self.n_free = i32([len(m.free)])
        self.t = cfi.page_table(self.table.data_ptr(), self.cached.data_ptr(), self.free.data_ptr(), self.n_free.data_ptr(), m.rows,
                                m.max_pages, m.page, m.n_pages)

    def place(self, rows, new, max_new, max_context):
        n, m = len(rows), self.m
        full = lambda k, t=torch.int32: torch.full((k,), -99, dtype=t, device=DEV)  # noqa: E731
        b = dict(rows=i32(rows), new=i32(new), lens=full(n + 1), table=full((n + 1) * m.max_pages).view(n + 1, -1), cu_q=full(n + 2),
                 cu_kv=full(n + 2), slots=full(max_new + 1, torch.int64), positions=full(max_new + 1),
                 context=full((max_context or 0) + 1, torch.int64), status=full(2))
        d = cfi.page_batch(b["rows"].data_ptr(), b["new"].data_ptr(), n, b["lens"].data_ptr(), b["table"].data_ptr(), b["cu_q"].data_ptr(),
                           b["cu_kv"].data_ptr(), b["slots"].data_ptr(), b["positions"].data_ptr(), max_new, b["status"].data_ptr(),
                           context=b["context"].data_ptr() if max_context is not None else 0, max_context=max_context or 0)
        cfi.paged_place(self.t, d, stream=stream())
        torch.cuda.synchronize()
        return {k: v.cpu().numpy() for k, v in b.items()}

    def trim(self, rows, keep):
        r, k, status = i32(rows), i32(keep), i32([-99, -99])
        cfi.paged_trim(self.t, r.data_ptr(), k.data_ptr(), len(rows), status.data_ptr(), stream=stream())
        torch.cuda.synchronize()
        assert int(status[1]) == -99
        return int(status[0])

    def check(self):
        m = self.m
        assert self.cached.tolist() == m.cached and int(self.n_free) == len(m.free)
        assert self.free[:len(m.free)].tolist() == m.free
        table = self.table.cpu().numpy()
        for r in range(m.rows):
            assert table[r, :len(m.own[r])].tolist() == m.own[r]


def step(m, d, rows, new, max_new, max_context):
    """One call on both."""
    why = m.why(rows, new, max_new, max_context)
    before = [m.cached[r] for r in rows] if why != cfi.PLACE_BAD_ROW else None
    got = d.place(rows, new, max_new, max_context)
    n, k = len(rows), max_context or 0
    assert got["status"].tolist() == [why, -99]
    for name in ("lens", "cu_q", "cu_kv", "slots", "positions", "context"):
        assert got[name][-1] == -99  # nothing behind
    if why:
        assert not got["lens"][:n].any() and not got["cu_q"][:n + 1].any() and not got["cu_kv"][:n + 1].any()
        assert (got["slots"][:max_new] == -1).all() and (got["positions"][:max_new] == 0).all()
        assert (got["context"][:k] == -1).all() and (got["table"] == -99).all()
    else:
        slots, positions, context = m.place(rows, new)
        after = [b + a for b, a in zip(before, new)]
        assert got["lens"][:n].tolist() == after
        assert got["cu_q"][:n + 1].tolist() == np.cumsum([0] + list(new)).tolist()
        assert got["cu_kv"][:n + 1].tolist() == np.cumsum([0] + after).tolist()
        assert got["slots"][:max_new].tolist() == slots + [-1] * (max_new - len(slots))
        assert got["positions"][:max_new].tolist() == positions + [0] * (max_new - len(positions))
        if max_context is not None:
            assert got["context"][:k].tolist() == context + [-1] * (k - len(context))
        for s, r in enumerate(rows):
            assert got["table"][s, :len(m.own[r])].tolist() == m.own[r]
            assert (got["table"][s, len(m.own[r]):] == -99).all()
        assert (got["table"][n] == -99).all()
    d.check()
    return why


@pytest.mark.parametrize("rows,max_pages,page,pages,most", [(5, 8, 16, 30, 40), (40, 20, 32, 300, 300), (300, 6, 64, 900, 100), (3, 4, 256, 9, 700)])
def test_a_long_run(rows, max_pages, page, pages, most):
    """Batches placed and cut back in turn, many of which do not fit."""
    m = Lists(rows, max_pages, page, pages, 3)
    d = Device(m)
    r, seen = random.Random(rows), set()
    for _ in range(60):
        n = r.randrange(0, min(rows, 40) + 1)
        batch = r.sample(range(rows), n)
        new = [r.choice([0, 1, 1, r.randrange(most), page]) for _ in batch]
        after = sum(m.cached[x] + y for x, y in zip(batch, new))
        max_context = r.choice([None, after, after + 7, max(0, after - 1)])
        seen.add(step(m, d, batch, new, r.choice([sum(new), sum(new) + 13, max(0, sum(new) - 1)]), max_context))
        cut = r.sample(range(rows), r.randrange(0, rows + 1))
        keep = [r.choice([0, -4, m.cached[x], max(0, m.cached[x] - 1), r.randrange(m.cached[x] + 1), 1 << 30]) for x in cut]
        if r.random() < 0.6:
            assert d.trim(cut, keep) == cfi.PLACED
            m.trim(cut, keep)
            d.check()
    assert {cfi.PLACED, cfi.PLACE_NO_ROOM} <= seen


def test_trim_undoes_place():
    m = Lists(8, 30, 16, 100, 1)
    d = Device(m)
    rows = [5, 0, 7, 2]
    step(m, d, rows, [33, 16, 1, 0], 60, 60)
    free, before = list(m.free), [m.cached[r] for r in rows]
    step(m, d, rows, [15, 64, 100, 1], 180, None)
    assert d.trim(rows, before) == cfi.PLACED
    m.trim(rows, before)
    assert m.free == free
    d.check()


@pytest.mark.parametrize("rows,new", [([1, 2, 1], [1, 1, 1]), ([0, 8], [1, 1]), ([-1, 3], [1, 1]), ([4, 5], [3, -1]), ([6, 6], [0, 0]),
                                      ([2147483647], [1]), ([-2147483648], [1])])
def test_bad_batches_change_nothing(rows, new):
    m = Lists(8, 4, 16, 20)
    d = Device(m)
    step(m, d, [1, 2, 6], [20, 5, 1], 30, 30)
    assert step(m, d, rows, new, 10, 100) == cfi.PLACE_BAD_ROW
    if new[-1] >= 0:
        assert d.trim(rows, [0] * len(rows)) == cfi.PLACE_BAD_ROW
        d.check()


def test_codes_in_order():
    """Of several reasons the least."""
    m = Lists(4, 4, 16, 5)
    d = Device(m)
    assert step(m, d, [0, 1], [65, 100], 1000, 1000) == cfi.PLACE_TOO_LONG
    assert step(m, d, [0, 1], [64, 64], 100, 1000) == cfi.PLACE_NO_ROOM
    assert step(m, d, [0, 1], [64, 64], 128, 127) == cfi.PLACE_NO_ROOM
    assert step(m, d, [0, 1], [64, 64], 128, 128) == cfi.PLACE_NO_PAGES
    assert step(m, d, [0, 1], [64, 16], 80, 80) == cfi.PLACED
    assert step(m, d, [2], [1], 1, None) == cfi.PLACE_NO_PAGES
    assert step(m, d, [0, 0], [200, 1], 1, None) == cfi.PLACE_BAD_ROW
    assert step(m, d, [], [], 3, 5) == cfi.PLACED
    assert step(m, d, [3], [0], 0, 0) == cfi.PLACED
    assert step(m, d, [0], [2147483647], 5, None) == cfi.PLACE_TOO_LONG


def test_counts_that_pass_31_bits():
    """Sums of counts beyond an int are refused, not wrapped."""
    m = Lists(8, 1 << 27, 16, 4)  # rows of a table that is never reached
    d = Device(Lists(8, 4, 16, 4))
    d.t = cfi.page_table(d.table.data_ptr(), d.cached.data_ptr(), d.free.data_ptr(), d.n_free.data_ptr(), 8, 1 << 27, 16, 4)
    status = i32([-1])
    out = torch.zeros(64, dtype=torch.int64, device=DEV)
    for new in ([1 << 30] * 8, [2147483647, 1], [2147483632, 2147483632, 64]):
        n = len(new)
        rows, add = i32(list(range(n))), i32(new)
        b = cfi.page_batch(rows.data_ptr(), add.data_ptr(), n, out.data_ptr(), out.data_ptr() + 64, out.data_ptr() + 128, out.data_ptr() + 192,
                           out.data_ptr() + 256, out.data_ptr() + 320, 8, status.data_ptr())
        cfi.paged_place(d.t, b, stream=stream())
        torch.cuda.synchronize()
        assert int(status) == cfi.PLACE_TOO_LONG
        assert d.cached.tolist() == [0] * 8 and int(d.n_free) == 4
    assert m.rows == 8


def test_the_largest_batch():
    m = Lists(8200, 4, 16, 30000, 2)
    d = Device(m)
    r = random.Random(4)
    rows = r.sample(range(8200), 8192)
    new = [r.randrange(0, 40) for _ in rows]
    assert step(m, d, rows, new, sum(new) + 3, sum(new) + 5) == cfi.PLACED
    assert step(m, d, rows, [1] * 8192, 8192, None) == cfi.PLACED
    assert d.trim(rows, [0] * 8192) == cfi.PLACED
    m.trim(rows, [0] * 8192)
    d.check()
    assert len(m.free) == 30000


def test_a_stack_that_does_not_hold():
    """A height outside the stack is cut to it, and pages given back never pass it."""
    m = Lists(2, 4, 16, 6)
    d = Device(m)
    step(m, d, [0], [40], 40, None)
    d.n_free.fill_(5)  # two of row 0's three pages are claimed to be free as well
    assert d.trim([0], [0]) == cfi.PLACE_NO_PAGES
    assert int(d.n_free) == 5 and int(d.cached[0]) == 40
    d.n_free.fill_(-3)
    got = d.place([1], [1], 1, None)
    assert got["status"][0] == cfi.PLACE_NO_PAGES


def test_captured_steps():
    """A step of place and trim in a graph goes on by itself from replay to replay."""
    m = Lists(6, 50, 16, 200, 9)
    d = Device(m)
    rows, new, keep = i32([4, 1, 3]), i32([1, 1, 1]), i32([1 << 30] * 3)
    lens, table, cu_q, cu_kv = i32([0] * 3), i32([0] * 150), i32([0] * 4), i32([0] * 4)
    slots, positions, status = torch.zeros(5, dtype=torch.int64, device=DEV), i32([0] * 5), i32([0, 0])
    b = cfi.page_batch(rows.data_ptr(), new.data_ptr(), 3, lens.data_ptr(), table.data_ptr(), cu_q.data_ptr(), cu_kv.data_ptr(),
                       slots.data_ptr(), positions.data_ptr(), 5, status.data_ptr())
    step(m, d, [4, 1, 3], [10, 0, 100], 110, None)

    def both():
        s = stream()
        cfi.paged_place(d.t, b, stream=s)
        cfi.paged_trim(d.t, rows.data_ptr(), keep.data_ptr(), 3, status.data_ptr() + 4, stream=s)

    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()  # the stream's workspace
    m.place([4, 1, 3], [1, 1, 1])
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        both()
    for i in range(40):
        if i == 20:
            rows.copy_(i32([0, 4, 5]))
        if i == 30:
            keep.copy_(i32([3, 17, 1 << 30]))
        graph.replay()
        r = rows.tolist()
        want = m.place(r, [1, 1, 1])
        m.trim(r, keep.tolist())
        torch.cuda.synchronize()
        assert status.tolist() == [0, 0] and slots.tolist() == want[0] + [-1, -1] and positions.tolist() == want[1] + [0, 0]
        d.check()
