"""The NVFP4 projections on the GPU against their float64 forms.

Tolerances, elementwise (u = 2^-24):
- proj: a slab's dot is exact; the product of its scales and the product with the dot round once each, and a sum of n terms in
  any order is off by at most n u of the sum of their sizes: with the wave's sums, alpha and the residual (n + 16) u (sum |alpha
  dot ws xs| + |rs res|), n = K/16. A bf16 result adds half a step, 2^-8 of itself.
- swiglu: v = silu(g) u / in_scale with g, u off by dg, du as above: (1.1 (|u| + du) dg + |silu(g)| du) / in_scale (silu' is
  at most 1.1), and fewer than 64 roundings of its own, 64 u |v|. A scale is off by the largest of those over 127 and 2 u of
  itself; code x scale is off by half a scale, and by v's own error and 2^-16 of the scale.
"""
import ctypes

import numpy as np
import pytest
import torch

from ref64 import bf16_rne, bf2f, silu

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
MAG = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float64)


def e4m3(b):
    """E4M3 bytes as their values."""
    return torch.from_numpy(np.ascontiguousarray(b)).view(torch.float8_e4m3fn).double().numpy()


class Matrix:
    """[rows][K] random codes and scales; `odd`: bytes before each array on the device."""

    def __init__(self, X, rng, rows, K, alpha=0.37, odd=0, scales=None):
        self.rows, self.K, self.alpha = rows, K, float(np.float32(alpha))
        self.w = rng.integers(0, 256, (rows, K // 2)).astype(np.uint8)
        self.s = rng.integers(0x20, 0x70, (rows, K // 16)).astype(np.uint8) if scales is None else scales
        pad = lambda a: np.concatenate([np.zeros(odd, np.uint8), a.reshape(-1)])
        self.bufs = [X.DevBuf(array=pad(self.w)), X.DevBuf(array=pad(self.s))]
        self.handle = X.NVFP4(self.bufs[0].ptr + odd, self.bufs[1].ptr + odd, self.alpha, rows, K)

    def codes(self):
        nib = np.stack([self.w & 15, self.w >> 4], -1).reshape(self.rows, self.K // 16, 16)
        return np.where(nib & 8, -1.0, 1.0) * MAG[nib & 7]

    def product(self, xq, xs):
        """y and the sum of the terms' sizes, [nr][rows]."""
        nr = len(xq)
        y, size = np.zeros((2, nr, self.rows))
        c, s = self.codes(), e4m3(self.s)
        for n in range(nr):
            with np.errstate(invalid="ignore"):
                terms = (c * xq[n].reshape(1, -1, 16)).sum(-1) * s * xs[n].astype(np.float64)[None] * self.alpha
            y[n], size[n] = terms.sum(-1), np.abs(terms).sum(-1)
        return y, size


def rows_of(rng, nr, K, stride=None):
    """Codes [nr][stride] (what lies behind K is never read as one) and scales [nr][stride/16]."""
    stride = K if stride is None else stride
    xq = rng.integers(-128, 128, (nr, stride)).astype(np.int8)
    xs = (rng.uniform(0.2, 2.0, (nr, stride // 16)) / 127).astype(np.float32)
    xq[:, K:], xs[:, K // 16:] = 99, np.nan
    return xq, xs


def project(X, m, xq, xs, bf16=False, res=None, rs=0.0, odd=0, pad=0, stream=None):
    """y [nr][rows] of the call, checked to leave what lies beside its rows."""
    nr, rows = len(xq), m.rows
    shift = np.zeros(odd, np.uint8)
    dq = X.DevBuf(array=np.concatenate([shift, xq.reshape(-1).view(np.uint8)]))
    ds = X.DevBuf(array=xs)
    dt = np.uint16 if bf16 else np.float32
    y = np.full((nr, rows + pad), 0x1234, np.uint16) if bf16 else np.full((nr, rows + pad), 7.25, np.float32)
    dy = X.DevBuf(array=y)
    dr = None if res is None else X.DevBuf(array=res)
    X.call("q27x_proj_nvfp4_rows", ctypes.byref(m.handle), dq.ptr + odd, xq.shape[1], ds.ptr, dy.ptr, rows + pad, int(bf16),
           dr.ptr if dr else None, int(res is not None and res.dtype == np.uint16), 0 if res is None else res.shape[1], rs, nr, stream)
    X.call("q27x_device_sync")
    got = dy.download(dt, y.shape)
    assert np.array_equal(got[:, rows:], y[:, rows:]), "columns behind the rows were written"
    return got[:, :rows]


def check(got, m, xq, xs, res=None, rs=0.0):
    y, size = m.product(xq[:, :m.K], xs[:, :m.K // 16])
    if res is not None:
        r = (bf2f(res) if res.dtype == np.uint16 else res).astype(np.float64)[:, :m.rows] * float(np.float32(rs))
        y, size = y + r, size + np.abs(r)
    tol = (m.K // 16 + 16) * U * size
    bf16 = got.dtype == np.uint16
    err = np.abs((bf2f(got) if bf16 else got).astype(np.float64) - y)
    bad = err > tol + (2.0 ** -8 * (np.abs(y) + tol) if bf16 else 0)
    assert not bad.any(), (np.argwhere(bad)[:5], err[bad][:5], tol[bad][:5], y[bad][:5])


SHAPES = [(1, 16), (16, 32), (17, 48), (33, 112), (15, 128), (64, 144), (100, 272), (1024, 768), (257, 1040), (48, 5120), (40, 5136),
          (31, 17408), (16, 20480), (2, 40976), (4099, 2064)]


@pytest.mark.parametrize("rows,K", SHAPES)
def test_proj(gpu, rows, K):
    """Sizes around the tiles: one row to ragged thousands, K from one slab to many, 1 to 8 activation rows."""
    rng = np.random.default_rng(rows * 31 + K)
    m = Matrix(gpu, rng, rows, K)
    for nr in (1, 2, 3, 4, 5, 7, 8) if rows * K < 1 << 19 else (1, 3, 6):
        xq, xs = rows_of(rng, nr, K)
        check(project(gpu, m, xq, xs), m, xq, xs)


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("res", [None, "bf16", "f32"])
@pytest.mark.parametrize("nr", [1, 3, 8])
def test_proj_outputs_and_residuals(gpu, bf16, res, nr):
    rng = np.random.default_rng(nr + 10 * bf16)
    m = Matrix(gpu, rng, 203, 656, alpha=-0.01)
    xq, xs = rows_of(rng, nr, 656, 704)
    r = None
    if res:
        r = rng.standard_normal((nr, 210)).astype(np.float32) * 3
        r = bf16_rne(r) if res == "bf16" else r
    check(project(gpu, m, xq, xs, bf16, r, 0.75, pad=5), m, xq, xs, r, 0.75)


@pytest.mark.parametrize("odd", [1, 2, 3, 6, 13])
def test_proj_any_alignment(gpu, odd):
    """Codes, scales and activation codes at any byte."""
    rng = np.random.default_rng(odd)
    for rows, K in ((37, 304), (64, 2048)):
        m = Matrix(gpu, rng, rows, K, odd=odd)
        xq, xs = rows_of(rng, 5, K, K + 16)
        check(project(gpu, m, xq, xs, odd=odd), m, xq, xs)


def test_proj_every_code_and_scale(gpu):
    """Every pair of a weight code and an activation code, every finite scale byte, negative and subnormal ones included."""
    X, rng = gpu, np.random.default_rng(2)
    K = 16 * 256
    m = Matrix(X, rng, 16, K, alpha=1.0)
    m.w[:] = (np.arange(16) * 17).astype(np.uint8)[:, None]         # row r: code r everywhere
    s = np.arange(256).astype(np.uint8)
    s[(s & 127) == 127] = 0x38                                      # (not a number: below)
    m.s[:] = s[None]
    m.bufs[0].upload(m.w)
    m.bufs[1].upload(m.s)
    xq = np.zeros((1, K), np.int8)
    xq[0] = np.resize(np.arange(-128, 128), K)
    xs = np.ones((1, K // 16), np.float32)
    check(project(X, m, xq, xs), m, xq, xs)
    for i in range(0, 256, 5):                                      # a slab alone: one rounding of its scales' product
        one = np.zeros_like(xq)
        one[0, 16 * i:16 * i + 16] = rng.integers(-128, 128, 16)
        y, size = m.product(one, xs)
        assert (np.abs(project(X, m, one, xs) - y) <= 2 * U * np.abs(y)).all()


def test_proj_not_finite_stays_with_its_rows(gpu):
    """A scale that is not a number reaches its weight row alone, an infinite activation scale its activation row."""
    X, rng = gpu, np.random.default_rng(3)
    rows, K, nr = 40, 1040, 6
    m = Matrix(X, rng, rows, K)
    xq, xs = rows_of(rng, nr, K)
    clean = project(X, m, xq, xs)
    bad, xb = m.s.copy(), xs.copy()
    bad[7, 3], bad[39, 64], bad[20, 10] = 0x7F, 0xFF, 0x7F
    xb[4, 64] = np.inf
    m.bufs[1].upload(bad)
    got = project(X, m, xq, xb)
    for n in range(nr):
        for r in range(rows):
            if r in (7, 20, 39):
                assert np.isnan(got[n, r])
            elif n == 4:
                assert not np.isfinite(got[n, r])
            else:
                assert got[n, r] == clean[n, r]


def test_proj_zero_scales_and_rows(gpu):
    X, rng = gpu, np.random.default_rng(4)
    m = Matrix(X, rng, 30, 400, scales=np.zeros((30, 25), np.uint8))
    xq, xs = rows_of(rng, 2, 400)
    assert (project(X, m, xq, xs) == 0).all()
    m = Matrix(X, rng, 30, 400)
    xs[1] = 0
    assert (project(X, m, xq, xs)[1] == 0).all()


@pytest.mark.parametrize("K", [400, 5120, 17408])
def test_proj_rows_do_not_depend_on_each_other(gpu, K):
    """A row's bits are the same alone, first, last and among eight."""
    X, rng = gpu, np.random.default_rng(5)
    m = Matrix(X, rng, 100, K)
    xq, xs = rows_of(rng, 8, K)
    all8 = project(X, m, xq, xs).view(np.uint32)
    for lo, hi in ((0, 1), (7, 8), (0, 4), (3, 8), (2, 4)):
        assert np.array_equal(project(X, m, xq[lo:hi], xs[lo:hi]).view(np.uint32), all8[lo:hi])


def test_proj_past_32_bits(gpu):
    """Codes beyond 2^32 bytes: the last rows of a matrix of 4.3 GB, against a matrix of those rows."""
    X, rng = gpu, np.random.default_rng(6)
    K, tail = 16384, 24
    rows = (1 << 32) // (K // 2) + tail
    t = Matrix(X, rng, tail, K)
    w, s = X.DevBuf(rows * (K // 2)), X.DevBuf(rows * (K // 16))
    L = X.lib()
    for big, part, per in ((w, t.bufs[0], K // 2), (s, t.bufs[1], K // 16)):
        X.call("q27x_memset", big.ptr, 0, rows * per, None)
        X.call("q27x_memcpy_d2d", big.ptr + (rows - tail) * per, part.ptr, tail * per, None)
    X.call("q27x_device_sync")
    xq, xs = rows_of(rng, 2, K)
    dq, ds, dy = X.DevBuf(array=xq), X.DevBuf(array=xs), X.DevBuf(2 * rows * 4)
    h = X.NVFP4(w.ptr, s.ptr, t.alpha, rows, K)
    X.check(L.q27x_proj_nvfp4_rows(ctypes.byref(h), dq.ptr, K, ds.ptr, dy.ptr, rows, 0, None, 0, 0, 0.0, 2, None))
    X.call("q27x_device_sync")
    y = dy.download(np.float32, (2, rows))
    assert (y[:, :-tail] == 0).all()
    assert np.array_equal(y[:, -tail:], project(X, t, xq, xs))


# ---------------------------------------------------------------- gate | up
def swiglu(X, gate, up, xq, xs, in_scale, stream=None):
    nr, rows = len(xq), gate.rows
    dq, ds = X.DevBuf(array=xq), X.DevBuf(array=xs)
    oq, os_ = X.DevBuf(array=np.full((nr + 1, rows), 55, np.int8)), X.DevBuf(array=np.full((nr + 1, rows // 16), 7.25, np.float32))
    X.call("q27x_swiglu_nvfp4_rows", ctypes.byref(gate.handle), ctypes.byref(up.handle), dq.ptr, xq.shape[1], ds.ptr, oq.ptr, os_.ptr,
           in_scale, nr, stream)
    X.call("q27x_device_sync")
    q, s = oq.download(np.int8, (nr + 1, rows)), os_.download(np.float32, (nr + 1, rows // 16))
    assert (q[nr] == 55).all() and (s[nr] == 7.25).all(), "behind the last row was written"
    return q[:nr], s[:nr]


def check_swiglu(q, s, gate, up, xq, xs, in_scale):
    K, isc = gate.K, float(np.float32(in_scale))
    (g, sg), (u, su) = (m.product(xq[:, :K], xs[:, :K // 16]) for m in (gate, up))
    dg, du = ((K // 16 + 16) * U * z for z in (sg, su))
    v = silu(g) * u / isc
    dv = (1.1 * (np.abs(u) + du) * dg + np.abs(silu(g)) * du) / isc + 64 * U * np.abs(v)
    nr = len(xq)
    v, dv = v.reshape(nr, -1, 16), dv.reshape(nr, -1, 16)
    s = s.astype(np.float64)
    top = np.abs(v).max(-1) / 127
    assert (np.abs(s - top) <= dv.max(-1) / 127 + 2 * U * top).all()
    off = np.abs(q.reshape(v.shape) * s[..., None] - v)
    assert (off <= (0.5 + 2.0 ** -16) * s[..., None] + dv + dv.max(-1, keepdims=True)).all()


@pytest.mark.parametrize("rows,K", [(16, 16), (32, 144), (48, 1040), (2048, 1024), (272, 5120), (64, 17408)])
@pytest.mark.parametrize("nr", [1, 2, 4, 5, 8])
def test_swiglu(gpu, rows, K, nr):
    rng = np.random.default_rng(rows + K + nr)
    # outputs of a few units: gates on both sides of what the sigmoid turns
    gate, up = (Matrix(gpu, rng, rows, K, alpha=a / np.sqrt(K)) for a in (0.05, -0.03))
    xq, xs = rows_of(rng, nr, K, K + 48)
    q, s = swiglu(gpu, gate, up, xq, xs, 0.6)
    check_swiglu(q, s, gate, up, xq, xs, 0.6)


@pytest.mark.parametrize("K", [17408, 20480, 57344, 57328])
def test_activations_that_do_not_fit_together(gpu, K):
    """Rows too long for LDS at once, up to the longest: brought in turns, alone and eight together, a ragged end."""
    rng = np.random.default_rng(K)
    gate, up = (Matrix(gpu, rng, 48, K, alpha=a / np.sqrt(K)) for a in (0.05, 0.03))
    for nr in (1, 4, 7, 8):
        xq, xs = rows_of(rng, nr, K)
        check(project(gpu, gate, xq, xs), gate, xq, xs)
        q, s = swiglu(gpu, gate, up, xq, xs, 0.6)
        check_swiglu(q, s, gate, up, xq, xs, 0.6)


@pytest.mark.parametrize("rows,K", [(16 * 1100, 336), (16 * 2300 + 5, 160)])
def test_proj_more_tiles_than_blocks(gpu, rows, K):
    """Blocks that go through several tiles, the last round not full; a step that K does not fill in each."""
    rng = np.random.default_rng(rows)
    m = Matrix(gpu, rng, rows, K)
    for nr in (1, 4, 8):
        xq, xs = rows_of(rng, nr, K)
        check(project(gpu, m, xq, xs), m, xq, xs)


def test_swiglu_large_gates_and_zero_groups(gpu):
    """Gates far outside what e^-g holds in fp32, and a group whose outputs are all zero."""
    X, rng = gpu, np.random.default_rng(8)
    gate, up = Matrix(X, rng, 48, 256, alpha=1.0), Matrix(X, rng, 48, 256, alpha=0.1)
    xq, xs = rows_of(rng, 3, 256)
    xs *= 10
    up.s[16:32] = 0
    up.bufs[1].upload(up.s)
    g, _ = gate.product(xq, xs)
    assert g.min() < -200 and g.max() > 200
    q, s = swiglu(X, gate, up, xq, xs, 1.0)
    check_swiglu(q, s, gate, up, xq, xs, 1.0)
    assert (q[:, 16:32] == 0).all() and (s[:, 1] == 0).all()


def test_swiglu_like_its_three_calls(gpu):
    """The same numbers as gate, up and the quantizer one after another (a code may differ where a sum's order turns it)."""
    X, rng = gpu, np.random.default_rng(9)
    rows, K, nr = 176, 1040, 6
    gate, up = (Matrix(X, rng, rows, K, alpha=a / np.sqrt(K)) for a in (0.05, 0.03))
    xq, xs = rows_of(rng, nr, K)
    q, s = swiglu(X, gate, up, xq, xs, 0.6)
    dg, du = X.DevBuf(array=project(X, gate, xq, xs)), X.DevBuf(array=project(X, up, xq, xs))
    oq, os_ = X.DevBuf(nr * rows), X.DevBuf(nr * rows // 4)
    X.call("q27x_swiglu_quant_rows", dg.ptr, du.ptr, rows, oq.ptr, os_.ptr, rows, 0.6, nr, None)
    X.call("q27x_device_sync")
    q2, s2 = oq.download(np.int8, (nr, rows)), os_.download(np.float32, (nr, rows // 16))
    check_swiglu(q2, s2, gate, up, xq, xs, 0.6)
    assert np.abs(q.astype(int) - q2).max() <= 1 and (np.abs(s - s2) <= 2.0 ** -12 * s2).all()
