"""Refusals of the Q4_1 cache, cfi_norm_rope, cfi_paged_place and cfi_paged_trim (include/cfi_serve.h): arguments outside the
documented ones give cudaErrorInvalidValue before anything is launched, so none of these needs a GPU."""
import ctypes as C

import pytest

import cfi_b200 as cfi

INVALID = 1
P = 1 << 20  # an aligned address; nothing reads it


def cache(**kw):
    a = dict(k=P, v=P, type=cfi.Q4_1, n_pages=4, page_size=16, n_kv_head=2, head_dim=64)
    a.update(kw)
    return cfi.PagedCache(a["k"], a["v"], a["type"], a["n_pages"], a["page_size"], a["n_kv_head"], a["head_dim"])


def test_q4_1_page_bytes():
    assert cfi.paged_page_bytes(cfi.Q4_1, 16, 2, 64) == 16 * 2 * 64 * 20 // 32
    assert cfi.paged_page_bytes(cfi.Q4_1, 256, 3, 128) == 256 * 3 * 128 * 20 // 32
    for bad in (dict(type=4), dict(type=2), dict(page_size=8), dict(page_size=48), dict(head_dim=96), dict(n_kv_head=0), dict(n_pages=0)):
        assert cfi.lib().cfi_paged_page_bytes(cache(**bad)) == 0


@pytest.mark.parametrize("bad", [dict(type=7), dict(page_size=8), dict(head_dim=256), dict(k=None), dict(k=P + 8), dict(v=P + 4)])
def test_bad_q4_1_caches_are_refused(bad):
    L, c = cfi.lib(), cache(**bad)
    assert L.cfi_paged_kv_store(c, P, P, 0, 1024, 1024, P, 1, None) == INVALID
    assert L.cfi_paged_kv_load(c, P, P, P, 1024, 1024, 1, None) == INVALID
    assert L.cfi_paged_attention(c, P, 0, 4096, P, 0, 4096, P, 4, P, 1, 4, 0.125, None) == INVALID


@pytest.mark.parametrize("n_seq,max_pages", [(1, 2**31 - 1), (65535, 32764), (65536, 4)])
def test_longer_lists_are_refused(n_seq, max_pages):
    a = [cache(n_kv_head=1), P, 0, 64, P, 0, 64, P, max_pages, P, n_seq, 1, 0.125, None]
    assert cfi.lib().cfi_paged_attention(*a) == INVALID


# ---- rows ----
def rows(**kw):
    a = dict(q=P, q_out=P, pos=P, n_tokens=3, n_head=4, head_dim=64, k=P, v=P, n_kv_head=2, slots=P, k_out=P, v_out=P)
    a.update(kw)
    return cfi.norm_rope_rows(**a)


def call(r, c=None):
    return cfi.lib().cfi_norm_rope(r, c, None)


BAD_ROWS = [dict(head_dim=32), dict(head_dim=96), dict(head_dim=256), dict(n_tokens=-1), dict(n_head=0), dict(n_head=65536),
            dict(n_kv_head=-1), dict(n_kv_head=0), dict(in_type=8), dict(q_out_type=2), dict(kv_out_type=3), dict(n_rot=-8), dict(n_rot=72),
            dict(n_rot=12), dict(eps=-1e-6), dict(eps=float("nan")), dict(eps=float("inf")), dict(freq_base=0.0), dict(freq_base=-2.0),
            dict(freq_base=float("nan")), dict(freq_base=float("inf")), dict(freq_scale=float("nan")), dict(freq_scale=float("inf")),
            dict(q=0), dict(q=P + 8), dict(q_out=0), dict(q_out=P + 4), dict(k=P + 8), dict(v=P + 8), dict(k_out=P + 8), dict(v_out=P + 8),
            dict(q_stride=252), dict(q_stride=248), dict(k_stride=120), dict(v_stride=132), dict(q_out_stride=128), dict(k_out_stride=120),
            dict(v_out_stride=129), dict(k=0), dict(v=0), dict(k_out=0), dict(v_out=0), dict(q_bias=P + 4), dict(k_bias=P + 8),
            dict(v_bias=P + 4), dict(q_norm=P + 8), dict(k_norm=P + 4), dict(freq_factors=P + 2), dict(pos=0), dict(pos=P + 2),
            dict(n_tokens=1 << 28, n_head=16)]


@pytest.mark.parametrize("bad", BAD_ROWS)
def test_norm_rope_refusals(bad):
    assert call(rows(**bad)) == INVALID
    with pytest.raises(RuntimeError):
        cfi.norm_rope(rows(**bad))


@pytest.mark.parametrize("bad,c", [(dict(), dict(head_dim=128)), (dict(), dict(n_kv_head=3)), (dict(slots=0), {}), (dict(slots=P + 4), {}),
                                   (dict(k=0, k_out=0), {}), (dict(v=0, v_out=0), {}), (dict(), dict(type=2)), (dict(), dict(page_size=20))])
def test_norm_rope_cache_refusals(bad, c):
    assert call(rows(**bad), cache(**c)) == INVALID


def test_no_tokens_launch_nothing():
    assert call(rows(n_tokens=0), cache()) == 0
    assert call(rows(n_tokens=0, k_out=0, v_out=0), cache()) == 0
    assert call(rows(n_tokens=0, k=0, v=0, k_out=0, v_out=0, n_kv_head=0)) == 0
    assert call(rows(n_tokens=0, n_rot=0, pos=0)) == 0
    assert cfi.lib().cfi_norm_rope(None, None, None) == INVALID


# ---- page tables ----
def table(**kw):
    a = dict(table=P, cached=P, free_pages=P, n_free=P, n_rows=4, max_pages=8, page_size=16, n_pages=32)
    a.update(kw)
    return cfi.PageTable(**a)


def batch(**kw):
    a = dict(rows=P, n_new=P, lens=P, batch_table=P, cu_q=P, cu_kv=P, positions=P, status=P, slots=P, context=P, n_seq=2, max_new=4,
             max_context=64)
    a.update(kw)
    return cfi.PagedPlace(**a)


BAD_TABLES = [dict(table=None), dict(table=P + 2), dict(cached=None), dict(cached=P + 1), dict(free_pages=None), dict(free_pages=P + 2),
              dict(n_free=None), dict(n_free=P + 2), dict(n_rows=0), dict(n_rows=65537), dict(max_pages=0), dict(page_size=8),
              dict(page_size=24), dict(page_size=512), dict(n_pages=0)]


@pytest.mark.parametrize("bad", BAD_TABLES)
def test_bad_tables_are_refused(bad):
    assert cfi.lib().cfi_paged_place(table(**bad), batch(), None) == INVALID
    assert cfi.lib().cfi_paged_trim(table(**bad), P, P, 1, P, None) == INVALID
    with pytest.raises(RuntimeError):
        cfi.paged_place(table(**bad), batch())
    with pytest.raises(RuntimeError):
        cfi.paged_trim(table(**bad), P, P, 1, P)


@pytest.mark.parametrize("bad", [dict(rows=None), dict(rows=P + 2), dict(n_new=None), dict(n_new=P + 1), dict(lens=None), dict(lens=P + 2),
                                 dict(batch_table=None), dict(batch_table=P + 2), dict(cu_q=None), dict(cu_q=P + 2), dict(cu_kv=None),
                                 dict(cu_kv=P + 2), dict(positions=None), dict(positions=P + 2), dict(status=None), dict(status=P + 2),
                                 dict(slots=None), dict(slots=P + 4), dict(context=P + 4), dict(n_seq=-1), dict(n_seq=8193),
                                 dict(max_new=-1), dict(max_context=-1)])
def test_place_refusals(bad):
    assert cfi.lib().cfi_paged_place(table(), batch(**bad), None) == INVALID
    assert cfi.lib().cfi_paged_place(None, batch(), None) == INVALID
    assert cfi.lib().cfi_paged_place(table(), None, None) == INVALID


@pytest.mark.parametrize("at,value", [(0, None), (1, None), (1, P + 2), (2, None), (2, P + 2), (3, -1), (3, 8193), (4, None), (4, P + 2)])
def test_trim_refusals(at, value):
    a = [table(), P, P, 1, P, None]
    a[at] = value
    assert cfi.lib().cfi_paged_trim(*a) == INVALID


def test_structs_are_the_headers():
    """Sizes as a C compiler lays them out (14 pointers, 6 long longs, 8 ints, 3 floats; 4 and 4; 10 and 3)."""
    assert C.sizeof(cfi.NormRope) == 14 * 8 + 6 * 8 + 8 * 4 + 3 * 4 + 4
    assert C.sizeof(cfi.PageTable) == 4 * 8 + 4 * 4
    assert C.sizeof(cfi.PagedPlace) == 10 * 8 + 3 * 4 + 4
