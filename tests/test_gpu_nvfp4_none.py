"""Values that are not numbers through the NVFP4 projections: a weight scale, an activation scale or a residual that is none makes the outputs
that it has a part in none, in fp32 and bf16 and behind SwiGLU's quantizer, and no other."""
import numpy as np
import pytest

from ref64 import bf2f
from test_gpu_nvfp4 import Matrix, project, rows_of, swiglu

pytestmark = pytest.mark.gpu

# NaN as operations leave it, and with every bit of its fraction set, of either sign
NANS = np.array([0x7FC00000, 0x7FFFFFFF, 0xFFFFFFFF, 0xFFC00000, 0x7F800001], np.uint32).view(np.float32)


def values(y):
    return bf2f(y) if y.dtype == np.uint16 else y


def matrix(X, rng, rows, K, bad=(), alpha=0.02):
    m = Matrix(X, rng, rows, K, alpha=alpha)
    s = m.s.copy()
    for r, slab, byte in bad:
        s[r, slab] = byte
    m.bufs[1].upload(s)
    return m


# tiles of 16 and of 32 weight rows, activations held and in turns
SHAPES = [(40, 1040, 1), (40, 1040, 6), (5136, 1040, 7), (48, 20480, 8), (5120, 17424, 5)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,K,nr", SHAPES)
def test_proj_scales(gpu, rows, K, nr, bf16):
    bad = [(7, 3, 0x7F), (rows - 1, K // 16 - 1, 0xFF), (20, 10, 0x7F)]
    clean, m = (matrix(gpu, np.random.default_rng(rows), rows, K, b) for b in ((), bad))
    xq, xs = rows_of(np.random.default_rng(1), nr, K)
    want, got = project(gpu, clean, xq, xs, bf16), project(gpu, m, xq, xs, bf16)
    at = np.zeros(rows, bool)
    at[[r for r, _, _ in bad]] = True
    assert np.isnan(values(got)[:, at]).all()
    assert np.array_equal(got[:, ~at], want[:, ~at])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("rows,K,nr", SHAPES)
@pytest.mark.parametrize("nan", range(len(NANS)))
def test_proj_activation_scales_and_residuals(gpu, rows, K, nr, bf16, nan):
    m = matrix(gpu, np.random.default_rng(rows), rows, K)
    rng = np.random.default_rng(nan)
    xq, xs = rows_of(rng, nr, K)
    want = project(gpu, m, xq, xs, bf16)
    x2 = xs.copy()
    x2.view(np.uint32)[nr - 1, K // 16 - 1] = NANS.view(np.uint32)[nan]
    got = project(gpu, m, xq, x2, bf16)
    assert np.isnan(values(got)[nr - 1]).all() and np.array_equal(got[:nr - 1], want[:nr - 1])
    for res in (np.zeros((nr, rows), np.float32), np.zeros((nr, rows), np.uint16)):
        res[0, rows // 2:] = NANS[nan] if res.dtype == np.float32 else NANS.view(np.uint32)[nan] >> 16 | 1
        got = project(gpu, m, xq, xs, bf16, res, 1.0)
        assert np.isnan(values(got)[0, rows // 2:]).all()
        got[0, rows // 2:] = want[0, rows // 2:]
        assert np.array_equal(got, want)


@pytest.mark.parametrize("rows,K,nr", [(48, 1040, 1), (48, 1040, 4), (48, 1040, 6), (2576, 1040, 8), (48, 20480, 8), (2592, 12304, 5)])
@pytest.mark.parametrize("which", [0, 1])
def test_swiglu_scales(gpu, rows, K, nr, which):
    """A scale of gate or of up: the scale of its group of 16 outputs is none, and what is projected from them; other groups keep their bits."""
    bad = [(5, 3, 0x7F), (rows - 1, K // 16 - 1, 0xFF)]
    make = lambda b: [matrix(gpu, np.random.default_rng(i), rows, K, b if i == which else (), a / np.sqrt(K)) for i, a in enumerate((0.05, -0.03))]
    (gate, up), (gate2, up2) = make(()), make(bad)
    xq, xs = rows_of(np.random.default_rng(9), nr, K)
    q, s = swiglu(gpu, gate, up, xq, xs, 0.6)
    q2, s2 = swiglu(gpu, gate2, up2, xq, xs, 0.6)
    at = np.zeros(rows // 16, bool)
    at[[r // 16 for r, _, _ in bad]] = True
    assert np.isfinite(s).all() and np.isnan(s2[:, at]).all()
    assert np.array_equal(s2[:, ~at], s[:, ~at])
    groups = lambda c, which: c.reshape(nr, -1, 16)[:, which]
    assert np.array_equal(groups(q2, ~at), groups(q, ~at)) and (groups(q2, at) == 0).all()
    down = matrix(gpu, np.random.default_rng(3), 32, rows)
    assert np.isnan(project(gpu, down, q2, s2)).all()


@pytest.mark.parametrize("rows,K,nr", [(48, 1040, 3), (2576, 1040, 8), (2592, 12304, 5)])
def test_swiglu_activation_scales(gpu, rows, K, nr):
    """An activation scale that is none, and one that is infinite: no group of its row is finite, other rows keep their bits."""
    gate, up = (matrix(gpu, np.random.default_rng(i), rows, K, (), a / np.sqrt(K)) for i, a in enumerate((0.05, -0.03)))
    xq, xs = rows_of(np.random.default_rng(9), nr, K)
    q, s = swiglu(gpu, gate, up, xq, xs, 0.6)
    for v in (np.nan, np.inf):
        x2 = xs.copy()
        x2[1, K // 16 - 1] = v
        q2, s2 = swiglu(gpu, gate, up, xq, x2, 0.6)
        assert np.isnan(s2[1]).all() if np.isnan(v) else not np.isfinite(s2[1]).any()
        rest = [n for n in range(nr) if n != 1]
        assert np.array_equal(q2[rest], q[rest]) and np.array_equal(s2[rest], s[rest])
