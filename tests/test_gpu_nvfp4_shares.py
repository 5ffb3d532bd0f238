"""The NVFP4 projections where a compute unit has three tiles of weight rows, which are one block's: parts against the float64 form, every
output's bits against those of calls of one row, whose blocks have a tile each, nothing written beside the rows, a residual in place."""
import ctypes

import numpy as np
import pytest

from ref64 import bf16_rne
from test_gpu_nvfp4 import Matrix, check, project, rows_of

pytestmark = pytest.mark.gpu


def part(m, lo, hi):
    """Rows lo .. hi - 1 of a matrix, on the host alone."""
    p = Matrix.__new__(Matrix)
    p.rows, p.K, p.alpha, p.w, p.s = hi - lo, m.K, m.alpha, m.w[lo:hi], m.s[lo:hi]
    return p


# the fewest and most rows of three tiles, a last block that is not full, K of one slab, a ragged end, waves that go through K in
# turns, activations that leave no room for three tiles' sums
@pytest.mark.parametrize("rows,K", [(8193, 16), (12288, 272), (8970, 784), (9001, 5136), (12287, 2064), (8195, 8208), (10240, 14352), (9217, 17424)])
def test_three_tiles_a_unit(gpu, rows, K):
    rng = np.random.default_rng(rows + K)
    m = Matrix(gpu, rng, rows, K, alpha=-0.02)
    xq, xs = rows_of(rng, 8, K, K + 16)
    alone = np.array([project(gpu, m, xq[n:n + 1], xs[n:n + 1])[0] for n in range(8)])
    for lo, hi in ((0, 60), (4000, 4060), (rows - 60, rows)):
        check(alone[:, lo:hi], part(m, lo, hi), xq, xs)
    for nr in (3, 4, 5, 6, 7, 8):
        got = project(gpu, m, xq[:nr], xs[:nr], pad=3)
        assert np.array_equal(got.view(np.uint32), alone[:nr].view(np.uint32)), nr


@pytest.mark.parametrize("nr", [3, 6, 8])
def test_residual_in_place(gpu, nr):
    X, rng = gpu, np.random.default_rng(nr)
    rows, K = 9001, 1040
    m = Matrix(X, rng, rows, K, alpha=0.01, odd=5)
    xq, xs = rows_of(rng, nr, K)
    res = bf16_rne(rng.standard_normal((nr, rows + 2)).astype(np.float32))
    apart = project(X, m, xq, xs, True, res, 1.0)
    check(apart[:, -200:], part(m, rows - 200, rows), xq, xs, res[:, rows - 200:rows], 1.0)
    y, dq, ds = X.DevBuf(array=res), X.DevBuf(array=xq), X.DevBuf(array=xs)
    X.call("q27x_proj_nvfp4_rows", ctypes.byref(m.handle), dq.ptr, K, ds.ptr, y.ptr, rows + 2, 1, y.ptr, 1, rows + 2, 1.0, nr, None)
    X.call("q27x_device_sync")
    got = y.download(np.uint16, res.shape)
    assert np.array_equal(got[:, :rows], apart) and np.array_equal(got[:, rows:], res[:, rows:])
