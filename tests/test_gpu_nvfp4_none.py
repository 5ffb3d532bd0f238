"""Values that are not numbers through gate and up on NVFP4 weights: a weight scale or an activation scale that is none makes the scale of the 16
outputs that it has a part in none, and what is projected from them, and no other."""
import numpy as np
import pytest

from test_gpu_nvfp4 import Matrix, project, rows_of, swiglu

pytestmark = pytest.mark.gpu


def matrix(X, rng, rows, K, bad=(), alpha=0.02):
    m = Matrix(X, rng, rows, K, alpha=alpha)
    s = m.s.copy()
    for r, slab, byte in bad:
        s[r, slab] = byte
    m.bufs[1].upload(s)
    return m


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
