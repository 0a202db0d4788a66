"""Arguments that the paged-cache operators and sampling refuse, on the host, before any device call."""
import ctypes

import pytest

import pitorch_amd as pa
from tests._paged import byref

ARG = 1
P = 1 << 20        # an aligned address that nothing dereferences


def cache(**kw):
    d = dict(k=P, v=P, type=pa.F32, n_pages=8, page_size=16, n_kv_heads=2, head_dim=64, page_stride=16 * 128,
             pos_stride=128, head_stride=64)
    d.update(kw)
    return pa.Pages(*d.values())


BAD_CACHE = [dict(k=None), dict(v=None), dict(k=P + 8), dict(type=2), dict(n_pages=0), dict(page_size=0),
             dict(n_pages=1 << 16, page_size=1 << 15), dict(n_kv_heads=0), dict(head_dim=0), dict(head_dim=66),
             dict(head_dim=132, page_stride=1 << 20, pos_stride=264, head_stride=132), dict(page_stride=60),
             dict(pos_stride=130), dict(head_stride=32)]


def store(c, q=P, ldq=256, q_out=P, ldo=256, heads=4, k=P, v=P, ldkv=128, pos=P, slot=P, rows=3, rope=P, rope_len=9):
    return pa.load_ptmi().ptmi_paged_store_dev(byref(c) if c else None, q, ldq, q_out, ldo, heads, k, v, ldkv, pos, slot, rows,
                                               rope, rope_len, None)


def attend(c, table=P, width=4, start=P, kv=P, n=2, new=1, q=P, ldq=256, out=2 * P, ldo=256, rows=2, heads=4, scale=0.125,
           work=P, work_bytes=1 << 40):
    return pa.load_ptmi().ptmi_paged_attention_dev(byref(c) if c else None, table, width, start, kv, n, new, q, ldq, out, ldo, rows,
                                                   heads, scale, work, work_bytes, None)


def plan(past=P, fresh=P, n=2, pool=P, count=P, n_pages=8, page=16, table=P, width=4, kv=P, left=P, start=P, pos=P, slot=P,
         max_rows=8, status=P):
    return pa.load_ptmi().ptmi_paged_plan_dev(past, fresh, n, pool, count, n_pages, page, table, width, kv, left, start, pos, slot,
                                              max_rows, status, None)


def sample(x=P, ld=100, rows=1, vocab=100, token=P):
    return pa.load_ptmi().ptmi_sample_dev(x, ld, rows, vocab, None, None, None, None, None, token, None)


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_caches(bad):
    assert store(cache(**bad)) == ARG
    assert attend(cache(**bad)) == ARG
    assert pa.load_ptmi().ptmi_paged_attention_work(byref(cache(**bad)), 4, 1) == 0
    assert pa.load_ptmi().ptmi_last_error()


def test_null_cache():
    assert store(None) == ARG and attend(None) == ARG
    assert pa.load_ptmi().ptmi_paged_attention_work(None, 4, 1) == 0


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(heads=0), dict(k=None), dict(v=None), dict(slot=None), dict(pos=None),
                                 dict(q_out=None), dict(rope_len=0), dict(ldq=252), dict(ldq=258), dict(ldo=128),
                                 dict(ldkv=124), dict(q=P + 4), dict(rope=P + 8), dict(k=P + 4), dict(ldo=260)], ids=str)
def test_store_refuses(bad):
    assert store(cache(), **bad) == ARG


@pytest.mark.parametrize("bad", [dict(n=-1), dict(width=0), dict(rows=-1), dict(new=-1), dict(heads=0), dict(heads=3),
                                 dict(scale=float("nan")), dict(scale=float("inf")), dict(scale=3e38), dict(table=None), dict(start=None),
                                 dict(kv=None), dict(q=None), dict(out=None), dict(work=None), dict(q=P + 4), dict(out=P),
                                 dict(ldq=252), dict(ldo=257), dict(work=P + 8), dict(work_bytes=0),
                                 dict(width=1 << 27)], ids=str)
def test_attention_refuses(bad):
    assert attend(cache(), **bad) == ARG


@pytest.mark.parametrize("bad", [dict(n=-1), dict(n=8193), dict(max_rows=-1), dict(n_pages=0), dict(page=0), dict(width=0),
                                 dict(n_pages=1 << 16, page=1 << 15), dict(pool=None), dict(count=None), dict(left=None),
                                 dict(start=None), dict(status=None), dict(past=None), dict(fresh=None), dict(table=None),
                                 dict(kv=None), dict(pos=None), dict(slot=None)], ids=str)
def test_plan_refuses(bad):
    assert plan(**bad) == ARG


@pytest.mark.parametrize("bad", [dict(rows=-1), dict(vocab=0), dict(vocab=(1 << 18) + 1, ld=1 << 19), dict(ld=99),
                                 dict(x=None), dict(token=None), dict(x=P + 2)], ids=str)
def test_sample_refuses(bad):
    assert sample(**bad) == ARG


def test_nothing_to_do_is_no_error():
    assert store(cache(), rows=0) == 0
    assert attend(cache(), rows=0) == 0 and attend(cache(), n=0) == 0
    assert sample(rows=0) == 0


def test_work_is_for_any_lengths():
    """The workspace depends on the cache's shape and the rows of a request, and holds for fewer."""
    L = pa.load_ptmi()
    w = [L.ptmi_paged_attention_work(byref(cache()), 4, n) for n in (1, 8, 64, 4096, 0)]
    assert all(w) and max(w) == w[-1]
    assert ctypes.sizeof(pa.Pages) == 64
