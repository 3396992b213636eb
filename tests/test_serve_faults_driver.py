"""The serving driver (serve.py) after calls that fail, without a GPU: its tensors on the CPU, page tables on the "device" kept in them as
include/cfi_serve.h says, the other calls recorded."""
import ctypes as C

import pytest

torch = pytest.importorskip("torch")
import cfi_b200 as cfi  # noqa: E402
import serve  # noqa: E402
from test_serve_rows_driver import rig, word  # noqa: E402,F401


def place(t, b):
    """cfi_paged_place on memory of the host."""
    n = b.n_seq
    rows, new = list(word(b.rows, n)), list(word(b.n_new, n))
    cached, n_free, free = word(t.cached, t.n_rows), word(t.n_free), word(t.free_pages, t.n_pages)
    table, page = word(t.table, t.n_rows * t.max_pages), t.page_size
    slots, positions = (C.c_int64 * b.max_new).from_address(b.slots), word(b.positions, b.max_new)
    slots[:], positions[:] = [-1] * b.max_new, [0] * b.max_new
    word(b.lens, n)[:] = [0] * n
    pages = lambda k: -(-k // page)  # noqa: E731
    if len(set(rows)) < n or any(not 0 <= r < t.n_rows for r in rows) or min(new) < 0:
        return cfi.PLACE_BAD_ROW
    after = [cached[r] + k for r, k in zip(rows, new)]
    if any(a > t.max_pages * page for a in after):
        return cfi.PLACE_TOO_LONG
    if sum(new) > b.max_new or (b.context and sum(after) > b.max_context):
        return cfi.PLACE_NO_ROOM
    if sum(pages(a) - pages(cached[r]) for r, a in zip(rows, after)) > n_free[0]:
        return cfi.PLACE_NO_PAGES
    x = 0
    for s, (r, a) in enumerate(zip(rows, after)):
        for p in range(cached[r], a):
            if p % page == 0:
                n_free[0] -= 1
                table[r * t.max_pages + p // page] = free[n_free[0]]
            slots[x], positions[x] = table[r * t.max_pages + p // page] * page + p % page, p
            x += 1
        cached[r] = a
        word(b.lens, n)[s] = a
    return cfi.PLACED


def trim(t, rows, keep, n):
    """cfi_paged_trim the same way."""
    rows, keep = list(word(rows, n)), list(word(keep, n))
    cached, n_free, free = word(t.cached, t.n_rows), word(t.n_free), word(t.free_pages, t.n_pages)
    table, pages = word(t.table, t.n_rows * t.max_pages), lambda k: -(-k // t.page_size)
    if len(set(rows)) < n or any(not 0 <= r < t.n_rows for r in rows):
        return cfi.PLACE_BAD_ROW
    for r, k in list(zip(rows, keep))[::-1]:
        k = min(cached[r], max(k, 0))
        for i in range(pages(cached[r]) - 1, pages(k) - 1, -1):
            free[n_free[0]] = table[r * t.max_pages + i]
            n_free[0] += 1
        cached[r] = k
    return cfi.PLACED


@pytest.fixture
def held(rig, monkeypatch):  # noqa: F811
    """rig with page tables that are kept; refuse: what the next calls on them answer instead of being done; fail: names of calls that
    raise once each; stored: slots and positions of each layer's rows; attended: lengths of each step's sequences."""
    r = rig
    r.refuse, r.fail, r.stored, r.attended = [], [], [], []

    def once(name):
        if name in r.fail:
            r.fail.remove(name)
            raise MemoryError(name)

    def placed(table, batch, stream=None):
        once("paged_place")
        word(batch.status)[0] = r.refuse.pop(0) if r.refuse else place(table, batch)

    def trimmed(table, rows, keep, n, status, stream=None):
        once("paged_trim")
        word(status)[0] = r.refuse.pop(0) if r.refuse else trim(table, rows, keep, n)

    def rotated(rows, cache=None, stream=None):
        once("norm_rope")
        n = rows.n_tokens
        r.stored.append((list((C.c_int64 * n).from_address(rows.slots)), list(word(rows.pos, n))))

    def attention(cache, q, out, table, lens, n, *a, stream=None, **k):
        once("paged_attention")
        r.attended.append(list(word(lens, n)))

    monkeypatch.setattr(cfi, "paged_place", placed)
    monkeypatch.setattr(cfi, "paged_trim", trimmed)
    monkeypatch.setattr(cfi, "norm_rope", rotated)
    monkeypatch.setattr(cfi, "paged_attention", attention)
    monkeypatch.setattr(cfi, "packed_attention", lambda *a, stream=None, **k: once("packed_attention"))
    return r


def free_pages(s):
    """Of the server's own count, and of its state."""
    if not s.on_device:
        return len(s.free)
    assert s.n_free == int(s.state.n_free)
    return s.n_free


def run(r, s, *steps):
    """What the calls store and attend to."""
    del r.stored[:], r.attended[:]
    for x in steps:
        x()
    return list(r.stored), list(r.attended)


@pytest.mark.parametrize("tables", ["host", "device"])
@pytest.mark.parametrize("fails", ["norm_rope", "paged_attention", "paged_place"])
def test_a_failed_step_again(held, tables, fails):
    """A step that raises in a layer, and again: the same slots and lengths as if it had not raised."""
    if fails == "paged_place" and tables == "host":
        return
    out = []
    for broken in (False, True):
        s = held.build(cfi.Q4_1, pages=12, tables=tables)
        a, b = serve.Sequence(list(range(16))), serve.Sequence([1, 2, 3])
        s.prefill([a, b])
        a.tokens.append(7), b.tokens.append(8)
        if broken:
            held.fail[:] = [fails]
            with pytest.raises(MemoryError):
                s.step([a, b])
            assert (a.cached, b.cached) == (16, 3)
        out.append(run(held, s, lambda: s.step([a, b])))
        assert (a.cached, b.cached) == (17, 4) and free_pages(s) == 12 - 3
        for x in (a, b):
            s.release(x)
        assert free_pages(s) == 12
    assert out[0] == out[1]


@pytest.mark.parametrize("tables", ["host", "device"])
@pytest.mark.parametrize("fails", ["norm_rope", "packed_attention", "paged_place"])
def test_a_failed_prompt_again(held, tables, fails):
    """The same of prompts, new ones and the rest of one, which may be cut shorter before the next try."""
    if fails == "paged_place" and tables == "host":
        return
    s = held.build(cfi.Q4_1, pages=12, tables=tables)
    a, b = serve.Sequence(list(range(40))), serve.Sequence([5] * 20)
    s.prefill([a], [18])
    held.fail[:] = [fails]
    with pytest.raises(MemoryError):
        s.prefill([a, b])
    assert (a.cached, b.cached) == (18, 0)
    stored, _ = run(held, s, lambda: s.prefill([a, b], [33, 20]))
    assert stored[0][1] == list(range(18, 33)) + list(range(20))
    assert len(set(stored[0][0])) == 35 and min(stored[0][0]) >= 0
    held.fail[:] = [fails]
    with pytest.raises(MemoryError):
        s.prefill([a])
    s.cut([a], [30])
    assert (a.cached, len(a.tokens)) == (30, 30) and free_pages(s) == 12 - 2 - 2
    s.release(a)
    assert free_pages(s) == 10
    s.release(b)
    assert free_pages(s) == 12


@pytest.mark.parametrize("tables", ["host", "device"])
def test_release_after_a_failed_prompt(held, tables):
    """All pages come back, and the row."""
    s = held.build(cfi.Q4_1, pages=8, tables=tables, **(dict(rows=1) if tables == "device" else {}))
    for _ in range(5):
        held.fail[:] = ["packed_attention"]
        a = serve.Sequence(list(range(40)))
        with pytest.raises(MemoryError):
            s.prefill([a])
        s.release(a)
        assert free_pages(s) == 8 and a.row is None
    whole = serve.Sequence([1] * 128)
    s.prefill([whole])
    assert free_pages(s) == 0


def test_a_failed_trim_again(held):
    """Pages that a call could not give back go with the next one."""
    s = held.build(cfi.Q4_1, pages=8, tables="device")
    a = serve.Sequence(list(range(40)))
    s.prefill([a])
    for call in (lambda: s.cut([a], [10]), lambda: s.release(a)):
        held.fail[:] = ["paged_trim"]
        with pytest.raises(MemoryError):
            call()
    assert a.cached == 40 and a.row is not None and len(a.tokens) == 40
    s.cut([a], [10])
    assert a.cached == 10 and free_pages(s) == 7
    held.fail[:] = ["norm_rope", "paged_trim"]
    a.tokens.append(1)
    for _ in range(2):  # the step, then the cutting back before the next one
        with pytest.raises(MemoryError):
            s.step([a])
    s.step([a])
    assert held.attended[-1] == [11] and a.cached == 11
    s.release(a)
    assert free_pages(s) == 8


@pytest.mark.parametrize("call", ["step", "prompt"])
def test_a_refused_place_is_told_once(held, call):
    """The sample after it raises; the sequences then have what they had at the last tokens, and everything can be done again."""
    s = held.build(cfi.Q4_1, pages=8, tables="device")
    a, b = serve.Sequence(list(range(16))), serve.Sequence([1] * 20)
    s.sample([a], s.prefill([a]))
    held.refuse[:] = [cfi.PLACE_NO_PAGES]
    logits = s.step([a]) if call == "step" else s.prefill([b], [18])
    if call == "prompt":
        s.prefill([b])  # placed, but at the wrong positions: void
        s.step([a])  # placed as it should be; nothing says so
    with pytest.raises(RuntimeError, match="refused"):
        s.sample([a], logits)
    assert (a.cached, b.cached, len(a.tokens)) == (16, 0, 17)
    stored, lengths = run(held, s, lambda: s.prefill([b]), lambda: s.step([a]))
    assert [x[1] for x in stored] == [list(range(20))] * 2 + [[16]] * 2 and lengths == [[17]] * 2
    slots = stored[0][0] + stored[2][0]
    assert len(set(slots)) == 21 and free_pages(s) == 8 - 2 - 2
    s.sample([a], logits)  # in order again
    assert len(a.tokens) == 18
    s.release(a), s.release(b)
    assert free_pages(s) == 8 and int(s.state.status) == 0


@pytest.mark.parametrize("released", [False, True])
def test_a_refused_trim_is_told_once(held, released):
    """Its pages go back then, and a row that was given back is empty for the next sequence."""
    s = held.build(cfi.Q4_1, pages=8, tables="device", rows=2)
    a, b = serve.Sequence(list(range(40))), serve.Sequence([1])
    logits = s.prefill([a, b])
    s.sample([b], logits)
    held.refuse[:] = [cfi.PLACE_NO_PAGES]
    s.release(a) if released else s.cut([a], [5])
    with pytest.raises(RuntimeError, match="refused"):
        s.sample([b], logits)
    assert a.cached == (0 if released else 5)
    if released:
        assert free_pages(s) == 7
        a = serve.Sequence([3] * 17)
        assert run(held, s, lambda: s.prefill([a]))[0][0][1] == list(range(17))
    else:
        a.tokens.append(2)
        assert run(held, s, lambda: s.step([a]))[1][0] == [6]
    s.sample([b], logits)
    s.release(a), s.release(b)
    assert free_pages(s) == 8


def test_a_sequence_named_twice(held):
    """Its row cannot be placed twice in one call of the page table: refused before a page or a row is taken."""
    s = held.build(cfi.Q4_1, pages=8, tables="device", rows=2)
    a, b = serve.Sequence(list(range(20))), serve.Sequence([1])
    with pytest.raises(ValueError, match="twice"):
        s.prefill([a, b, a])
    assert a.row is None and len(s.rows) == 2 and free_pages(s) == 8
    s.prefill([a, b])
    a.tokens.append(1)
    with pytest.raises(ValueError, match="twice"):
        s.step([a, a])
    assert a.cached == 20
    assert run(held, s, lambda: s.step([a]))[1][0] == [21]
    s.sample([a], torch.zeros(1, 64))


def test_norms_that_a_kernel_cannot_read(held):
    """Another type, length, layout or device, or not two of a layer: refused when the server is made, not read by address."""
    good = torch.ones(64)
    for bad in (torch.ones(64, dtype=torch.float16), torch.ones(32), torch.ones(128)[::2], torch.ones(64, device="meta"), torch.ones(65)[1:],
                [1.0] * 64):
        for pair in ((good, bad), (bad, good)):
            with pytest.raises(ValueError, match="norms"):
                held.build(norms=[(good, good), pair])
    for layer in ((good,), (good, good, good)):
        with pytest.raises(ValueError, match="norms"):
            held.build(norms=[layer, (good, good)])
    s = held.build(norms=[(good, good), torch.ones(2, 64)])
    s.prefill([serve.Sequence([1, 2])])
    assert len(held.stored) == 2
