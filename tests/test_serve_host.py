"""Refusals of the serving operators (include/cfi_serve.h): arguments outside the documented ones give
cudaErrorInvalidValue before anything is launched, so none of these needs a GPU."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import cfi_b200 as cfi

INVALID = 1
P = 1 << 20  # an aligned address; nothing reads it


def cache(**kw):
    a = dict(k=P, v=P, type=cfi.T_F16, n_pages=4, page_size=16, n_kv_head=2, head_dim=64)
    a.update(kw)
    return cfi.PagedCache(a["k"], a["v"], a["type"], a["n_pages"], a["page_size"], a["n_kv_head"], a["head_dim"])


BAD_CACHES = [dict(type=0), dict(type=2), dict(n_pages=0), dict(page_size=8), dict(page_size=24), dict(page_size=512),
              dict(n_kv_head=0), dict(head_dim=32), dict(head_dim=96)]


def test_page_bytes():
    assert cfi.paged_page_bytes(cfi.T_F16, 16, 2, 64) == 16 * 2 * 64 * 2
    assert cfi.paged_page_bytes(cfi.Q8_0, 32, 3, 128) == 32 * 3 * 128 * 34 // 32
    for bad in BAD_CACHES:
        assert cfi.lib().cfi_paged_page_bytes(cache(**bad)) == 0
    assert cfi.lib().cfi_paged_page_bytes(None) == 0
    with pytest.raises(ValueError):
        cfi.paged_cache(cfi.T_F16, P, P, 4, 20, 2, 64)


@pytest.mark.parametrize("bad", BAD_CACHES + [dict(k=None), dict(v=P + 8)])
def test_bad_caches_are_refused(bad):
    L, c = cfi.lib(), cache(**bad)
    assert L.cfi_paged_kv_store(c, P, P, 0, 1024, 1024, P, 1, None) == INVALID
    assert L.cfi_paged_kv_load(c, P, P, P, 1024, 1024, 1, None) == INVALID
    assert L.cfi_paged_attention(c, P, 0, 4096, P, 0, 4096, P, 4, P, 1, 4, 0.125, None) == INVALID


@pytest.mark.parametrize("at,value", [(1, None), (1, P + 4), (2, None), (3, 8), (4, 120), (4, 129), (5, 64), (6, None), (6, P + 4),
                                      (7, -1), (7, 1 << 30)])
def test_store_refusals(at, value):
    a = [cache(), P, P, 0, 128, 128, P, 1, None]
    a[at] = value
    assert cfi.lib().cfi_paged_kv_store(*a) == INVALID


@pytest.mark.parametrize("at,value", [(1, None), (2, None), (3, P + 8), (4, 64), (5, 132), (6, -1)])
def test_load_refusals(at, value):
    a = [cache(), P, P, P, 128, 128, 1, None]
    a[at] = value
    assert cfi.lib().cfi_paged_kv_load(*a) == INVALID


@pytest.mark.parametrize("at,value", [(1, None), (1, P + 8), (2, 8), (3, 192), (3, 260), (4, None), (5, 14), (6, 128), (7, None),
                                      (8, 0), (9, None), (9, P + 2), (10, -1), (11, 0), (11, 3), (12, 0.0), (12, -1.0),
                                      (12, float("nan")), (12, float("inf"))])
def test_paged_attention_refusals(at, value):
    a = [cache(), P, 0, 256, P, 0, 256, P, 4, P, 1, 4, 0.125, None]
    a[at] = value
    assert cfi.lib().cfi_paged_attention(*a) == INVALID


@pytest.mark.parametrize("bad", [dict(q=None), dict(k=P + 8), dict(v=None), dict(out=P + 4), dict(cu_q=None), dict(cu_kv=P + 1),
                                 dict(q_stride=192), dict(k_stride=132), dict(v_stride=64), dict(out_stride=250), dict(n_seq=-1),
                                 dict(n_q=-1), dict(n_kv=-1), dict(n_head=3), dict(n_head=0), dict(n_kv_head=0), dict(head_dim=80),
                                 dict(out_type=8), dict(scale=0.0), dict(scale=-0.5), dict(scale=float("nan")), dict(scale=float("inf")),
                                 dict(n_head=258, n_kv_head=2, q_stride=1 << 15, out_stride=1 << 15)])
def test_packed_attention_refusals(bad):
    a = dict(q=P, k=P, v=P, out=P, cu_q=P, cu_kv=P, q_stride=256, k_stride=128, v_stride=128, out_stride=256, n_seq=1, n_q=5,
             n_kv=5, n_head=4, n_kv_head=2, head_dim=64, out_type=0, causal=1, scale=0.125)
    a.update(bad)
    assert cfi.lib().cfi_packed_attention(cfi.PackedAttention(**a), None) == INVALID
    assert cfi.lib().cfi_packed_attention(None, None) == INVALID


@pytest.mark.parametrize("at,value", [(0, None), (0, P + 2), (1, 99), (2, -1), (3, 0), (3, 400001), (4, P + 1), (8, None), (9, None),
                                      (10, P + 3)])
def test_sample_refusals(at, value):
    a = [P, 1 << 20, 1, 100, None, None, None, None, P, P, None, None]
    a[at] = value
    assert cfi.lib().cfi_sample(*a) == INVALID


def test_nothing_to_do_launches_nothing():
    L, c = cfi.lib(), cache()
    assert L.cfi_paged_kv_store(c, P, P, 0, 128, 128, P, 0, None) == 0
    assert L.cfi_paged_kv_load(c, P, P, P, 128, 128, 0, None) == 0
    assert L.cfi_paged_attention(c, P, 0, 256, P, 0, 256, P, 4, P, 0, 4, 0.125, None) == 0
    a = cfi.PackedAttention(P, P, P, P, P, P, 256, 128, 128, 256, 1, 0, 5, 4, 2, 64, 0, 1, 0.125)
    assert L.cfi_packed_attention(a, None) == 0
    assert L.cfi_sample(P, 100, 0, 100, None, None, None, None, P, P, None, None) == 0


def test_wrappers_raise():
    with pytest.raises(RuntimeError):
        cfi.paged_kv_store(cache(), P, P, P, 1, src_type=5)
    with pytest.raises(RuntimeError):
        cfi.sample(P, P, P, 1, 0)


# ---- the cut of cfi_paged_attention's list into runs (csrc/paged_cut.h), as the kernel computes it ----
@pytest.fixture(scope="module")
def cut(tmp_path_factory):
    d = tmp_path_factory.mktemp("cut")
    csrc = os.path.join(os.path.dirname(cfi.__file__), "csrc")
    (d / "cut.cpp").write_text('''#include "paged_cut.h"
extern "C" int quota(int total, int ctas, int least) { return paged_quota(total, ctas, least); }
extern "C" int runs(int total, int q) { return paged_runs(total, q); }
extern "C" int run_end(int begin, int q, int total) { return paged_run_end(begin, q, total); }
''')
    # -fwrapv: sums that pass an int wrap, as they do on the device
    subprocess.run(["g++", "-O1", "-fwrapv", "-shared", "-fPIC", "-I", csrc, str(d / "cut.cpp"), "-o", str(d / "cut.so")], check=True)
    return C.CDLL(str(d / "cut.so"))


@pytest.mark.parametrize("total", [1, 8, 9, 10, 2663, 2664, 2665, 100003, 2**30 + 7, 2**31 - 4000000, 2**31 - 444, 2**31 - 2, 2**31 - 1])
@pytest.mark.parametrize("ctas", [1, 2, 148, 296, 444])
def test_runs_cover_the_list(cut, total, ctas):
    """Every unit is in one run, up to the most that the host accepts."""
    q = cut.quota(total, ctas, 9)
    assert q >= 9 and q * ctas >= total and (q == 9 or (q - 1) * ctas < total)
    n = cut.runs(total, q)
    assert 1 <= n <= ctas
    ends = [cut.run_end(b * q, q, total) for b in range(n)]
    assert ends == [min((b + 1) * q, total) for b in range(n)] and ends[-1] == total and ends[-1] > (n - 1) * q


@pytest.mark.parametrize("n_seq,max_pages", [(1, 2**31 - 1), (1, 2**31 - 5), (65535, 32764), (65536, 4)])
def test_longer_lists_are_refused(n_seq, max_pages):
    a = [cache(n_kv_head=1), P, 0, 64, P, 0, 64, P, max_pages, P, n_seq, 1, 0.125, None]
    assert cfi.lib().cfi_paged_attention(*a) == INVALID


# ---- the quotient by a temperature (csrc/quotient.h) ----
@pytest.mark.parametrize("low,high", [(-3, 3), (-59, 59), (0, 1)])
def test_quotient_is_the_divisions(tmp_path, low, high):
    """Bit for bit, for temperatures and logits over the powers of two where the kernel takes it: |l| above 2^-60, T between 2^-60
    and 2^60, |l / T| below 2^13 for the largest logit."""
    csrc = os.path.join(os.path.dirname(cfi.__file__), "csrc")
    (tmp_path / "q.cpp").write_text('''#include "quotient.h"
extern "C" void many(const float *l, const float *t, float *by, float *div, int n) {
    for (int i = 0; i < n; i++) by[i] = quotient_by(l[i], t[i], 1.0f / t[i]), div[i] = l[i] / t[i];
}
''')
    subprocess.run(["g++", "-O2", "-ffp-contract=off", "-shared", "-fPIC", "-I", csrc, str(tmp_path / "q.cpp"), "-o", str(tmp_path / "q.so")],
                   check=True)
    rng, n = np.random.default_rng(low + 100), 1 << 20
    t = (rng.uniform(1, 2, n) * 2.0 ** rng.integers(low, high, n)).astype(np.float32)
    t[:4096] = np.nextafter(np.float32(2) ** rng.integers(low + 1, high + 1, 4096).astype(np.float32), np.float32(0))  # all ones
    l = (rng.normal(size=n) * 2.0 ** np.minimum(rng.integers(-59, 20, n), 12 + np.floor(np.log2(t)))).astype(np.float32)
    l[np.abs(l) <= 2.0 ** -60] = 1.0
    by, div = np.empty_like(l), np.empty_like(l)
    f = C.POINTER(C.c_float)
    C.CDLL(str(tmp_path / "q.so")).many(*(x.ctypes.data_as(f) for x in (l, t, by, div)), n)
    np.testing.assert_array_equal(by.view(np.uint32), div.view(np.uint32))
