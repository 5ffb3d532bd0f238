"""What the NVFP4 projections refuse, on the host, before any GPU call."""
import ctypes

import pytest

ARG, SHAPE = -1, -2
P = 1 << 20                                     # a stand-in address: refused calls touch no memory


def matrix(X, **kw):
    a = dict(w=P, s=P, alpha=1.0, rows=64, K=256)
    a.update(kw)
    return X.NVFP4(a["w"], a["s"], a["alpha"], a["rows"], a["K"])


def proj(X, w, **kw):
    a = dict(xq=P, xstride=256, xs=P, y=P, ystride=64, res=None, rstride=64, nr=3)
    a.update(kw)
    return X.lib().q27x_proj_nvfp4_rows(ctypes.byref(w) if w else None, a["xq"], a["xstride"], a["xs"], a["y"], a["ystride"], 0, a["res"], 0,
                                        a["rstride"], 1.0, a["nr"], None)


def swiglu(X, w, up=None, **kw):
    a = dict(xq=P, xstride=256, xs=P, oq=P, os=P, in_scale=1.0, nr=3)
    a.update(kw)
    up = matrix(X) if up is None else up
    return X.lib().q27x_swiglu_nvfp4_rows(ctypes.byref(w) if w else None, ctypes.byref(up), a["xq"], a["xstride"], a["xs"], a["oq"], a["os"],
                                          a["in_scale"], a["nr"], None)


@pytest.mark.parametrize("kw,rc", [(dict(w=None), ARG), (dict(s=None), ARG), (dict(rows=0), SHAPE), (dict(rows=-5), SHAPE),
                                   (dict(rows=2 ** 31 - 1), SHAPE), (dict(rows=2 ** 31 - (1 << 19)), SHAPE), (dict(K=0), SHAPE), (dict(K=8), SHAPE), (dict(K=250), SHAPE),
                                   (dict(K=57360), SHAPE), (dict(K=2 ** 31 - 16), SHAPE)])
@pytest.mark.parametrize("call", [proj, swiglu])
def test_matrices_refused(X, call, kw, rc):
    assert call(X, matrix(X, **kw), xstride=2 ** 31 - 16) == rc
    assert "nvfp4_rows" in X.lib().q27x_last_error().decode()


@pytest.mark.parametrize("kw,rc", [(dict(xq=None), ARG), (dict(xs=None), ARG), (dict(nr=0), SHAPE), (dict(nr=9), SHAPE), (dict(nr=-1), SHAPE),
                                   (dict(xstride=240), ARG), (dict(xstride=264), ARG)])
@pytest.mark.parametrize("call", [proj, swiglu])
def test_rows_refused(X, call, kw, rc):
    assert call(X, matrix(X), **kw) == rc


@pytest.mark.parametrize("call", [proj, swiglu])
def test_rows_past_2_31_bytes_refused(X, call):
    assert call(X, matrix(X), xstride=1 << 30, nr=3) == -6
    assert call(X, matrix(X), xstride=(1 << 31) - 16, nr=2) == -6


@pytest.mark.parametrize("call", [proj, swiglu])
def test_null_matrix(X, call):
    assert call(X, None) == ARG


@pytest.mark.parametrize("kw", [dict(y=None), dict(ystride=63), dict(res=P, rstride=63)])
def test_proj_refused(X, kw):
    assert proj(X, matrix(X), **kw) == ARG


@pytest.mark.parametrize("kw", [dict(oq=None), dict(os=None), dict(in_scale=0.0), dict(in_scale=-1.0), dict(in_scale=float("nan"))])
def test_swiglu_refused(X, kw):
    assert swiglu(X, matrix(X), **kw) == ARG


@pytest.mark.parametrize("gate,up", [(dict(rows=48), {}), (dict(K=128), {}), ({}, dict(rows=32)), (dict(rows=72), dict(rows=72))])
def test_swiglu_refuses_matrices_that_differ(X, gate, up):
    assert swiglu(X, matrix(X, **gate), matrix(X, **up)) == SHAPE
    assert swiglu(X, matrix(X), matrix(X, w=None)) == ARG
