"""What the paged-cache entry points refuse, on the host, before any GPU call: null pointers, shapes without a kernel,
counts that would leave their buffers, misaligned pages."""
import ctypes

import pytest

ARG, SHAPE, RANGE = -1, -2, -6
P = 1 << 20                                     # a stand-in address: refused calls touch no memory


def cache(X, **kw):
    c = dict(k=P, v=P, ks=P, vs=P, kv_group=32, nkv=8, hd=128, n_pages=10, page=16, page_stride=0, table=P, table_stride=4,
             lens=P, row_start=P, n_seq=2)
    c.update(kw)
    return X.PagedKV(**c)


def prep(X, kv, **kw):
    a = dict(qkv=P, stride=10240, qn=P, kn=P, cos=P, sin=P, rot=32, n_pos=100, pos=P, pos_stride=5, n_axes=3,
             axes=(ctypes.c_uint8 * 128)(*([0, 1, 2, 0] * 32)), qh=P, nq=32, gate=1, eps=1e-6, nrows=5)
    a.update(kw)
    return X.lib().q27x_paged_prep_rows(a["qkv"], a["stride"], a["qn"], a["kn"], a["cos"], a["sin"], a["rot"], a["n_pos"], a["pos"],
                                        a["pos_stride"], a["n_axes"], a["axes"], ctypes.byref(kv) if kv else None, a["qh"], a["nq"],
                                        a["gate"], a["eps"], a["nrows"], None)


def attn(X, kv, **kw):
    a = dict(qh=P, qkv=P, stride=10240, nq=32, gate=1, max_len=60, max_rows=1, nrows=2, work=P, out=P, xq=None, xs=None, w=None, ws=0)
    a.update(kw)
    return X.lib().q27x_paged_attn_rows(a["qh"], a["qkv"], a["stride"], ctypes.byref(kv) if kv else None, a["nq"], a["gate"],
                                        a["max_len"], a["max_rows"], a["nrows"], a["work"], a["out"], a["xq"], a["xs"], a["w"],
                                        a["ws"], None)


def evict(X, kv, **kw):
    a = dict(w=P, ws=60, n_acc=P, nrows=2, decay=1.0, acc=P, ord=P, stride=60, state=P, high=50, budget=40, recent=10, max_len=60,
             work=P, new=P)
    a.update(kw)
    return X.lib().q27x_paged_evict(ctypes.byref(kv) if kv else None, a["w"], a["ws"], a["n_acc"], a["nrows"], a["decay"], a["acc"],
                                    a["ord"], a["stride"], a["state"], a["high"], a["budget"], a["recent"], a["max_len"], a["work"],
                                    a["new"], None)


CACHES = [(dict(k=None), ARG), (dict(v=None), ARG), (dict(ks=None), ARG), (dict(vs=None), ARG), (dict(table=None), ARG),
          (dict(lens=None), ARG), (dict(k=P + 8), ARG), (dict(v=P + 2), ARG), (dict(hd=64), SHAPE), (dict(hd=192), SHAPE),
          (dict(nkv=0), SHAPE), (dict(kv_group=8), SHAPE), (dict(kv_group=128), SHAPE), (dict(kv_group=-1), SHAPE),
          (dict(page=0), ARG), (dict(page=24), ARG), (dict(page_stride=8), ARG), (dict(page_stride=-16), ARG), (dict(n_pages=0), ARG),
          (dict(table_stride=0), ARG), (dict(n_seq=0), ARG), (dict(n_pages=1 << 28), RANGE), (dict(table_stride=1 << 28), RANGE),
          (dict(n_seq=65536), RANGE)]


@pytest.mark.parametrize("kw,rc", CACHES)
@pytest.mark.parametrize("call", [prep, attn, evict])
def test_caches_refused(X, call, kw, rc):
    assert call(X, cache(X, **kw)) == rc
    assert X.lib().q27x_last_error().decode().startswith("q27x_paged_")


@pytest.mark.parametrize("call", [prep, attn, evict])
def test_null_cache(X, call):
    assert call(X, None) == ARG


@pytest.mark.parametrize("kw,rc", [(dict(qkv=None), ARG), (dict(qn=None), ARG), (dict(kn=None), ARG), (dict(cos=None), ARG),
                                   (dict(sin=None), ARG), (dict(pos=None), ARG), (dict(qh=None), ARG), (dict(axes=None), ARG),
                                   (dict(rot=0), SHAPE), (dict(rot=31), SHAPE), (dict(rot=130), SHAPE), (dict(nq=12), SHAPE),
                                   (dict(nq=0), SHAPE), (dict(n_pos=0), ARG), (dict(n_axes=0), ARG), (dict(n_axes=5), ARG),
                                   (dict(n_axes=2), ARG), (dict(nrows=0), ARG), (dict(pos_stride=4), ARG), (dict(stride=-1), ARG)])
def test_prep_refused(X, kw, rc):
    assert prep(X, cache(X), **kw) == rc


@pytest.mark.parametrize("kw,rc", [(dict(qh=None), ARG), (dict(qkv=None), ARG), (dict(work=None), ARG), (dict(out=None), ARG),
                                   (dict(xq=P), ARG), (dict(work=P + 4), ARG), (dict(nq=20), SHAPE), (dict(nq=0), SHAPE),
                                   (dict(max_len=0), SHAPE), (dict(nrows=0), SHAPE), (dict(max_rows=0), SHAPE),
                                   (dict(max_rows=9), SHAPE), (dict(w=P, ws=59), ARG), (dict(stride=-1), ARG)])
def test_attn_refused(X, kw, rc):
    assert attn(X, cache(X), **kw) == rc


def test_attn_refuses_more_rows_than_a_grid(X):
    assert attn(X, cache(X, n_seq=60000), max_rows=2) == RANGE


@pytest.mark.parametrize("kw", [dict(acc=None), dict(ord=None), dict(state=None), dict(work=None), dict(new=None), dict(work=P + 8),
                                dict(max_len=0), dict(stride=59), dict(ws=59), dict(nrows=0), dict(recent=-1), dict(budget=0, recent=0),
                                dict(recent=41), dict(high=39), dict(decay=1.5), dict(decay=-0.1), dict(decay=float("nan"))])
def test_evict_refused(X, kw):
    assert evict(X, cache(X), **kw) == ARG


def test_work_bytes(X):
    """The workspace grows with what a call splits, covers the weights if they are wanted, and is 0 for refused counts."""
    f = X.lib().q27x_paged_attn_work_bytes
    assert 0 < f(32, 128, 256, 1, 0) < f(32, 128, 257, 1, 0) < f(32, 128, 257, 2, 0) < f(32, 128, 257, 2, 1)
    assert f(32, 128, 257, 2, 1) - f(32, 128, 257, 2, 0) >= 2 * 32 * 257 * 4
    assert f(32, 64, 257, 2, 0) == f(0, 128, 257, 2, 0) == f(32, 128, 0, 2, 0) == f(32, 128, 257, 0, 0) == 0
    e = X.lib().q27x_paged_evict_work_bytes
    assert 0 < e(1, 100) < e(2, 100) and e(0, 100) == e(1, 0) == 0
    # sizes that pass 32 bits
    assert f(32, 128, 131072, 512, 1) > 1 << 33


def test_lengths_that_indexes_cannot_run_over(X):
    """The kernels' indexes go a tile past max_len: lengths within that of 2^31 are refused, the last ones before it not."""
    big = 2 ** 31 - 65536
    assert evict(X, cache(X), max_len=big, stride=big, ws=big) == ARG
    e, f = X.lib().q27x_paged_evict_work_bytes, X.lib().q27x_paged_attn_work_bytes
    assert e(1, big) == 0 and e(1, big - 1) > 1 << 33
    assert f(32, 128, 2 ** 31 - 256, 1, 0) == 0 and f(32, 128, 2 ** 31 - 257, 1, 0) > 1 << 36
    assert attn(X, cache(X), max_len=2 ** 31 - 256) == SHAPE
