"""The NVFP4 projections where tiles of 32 weight rows serve 5 to 8 activation rows: against their float64 forms, and a row's bits against
those of calls with fewer rows, which other tiles serve."""
import numpy as np
import pytest

from test_gpu_nvfp4 import Matrix, check, check_swiglu, project, rows_of, swiglu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,K", [(5121, 16), (5120, 1040), (9001, 2064), (16384 + 7, 272), (16 * 2300 + 5, 656), (5130, 9216), (5120, 10256)])
def test_proj(gpu, rows, K):
    """Few tiles and many, ragged ends of both sides; rows that fill LDS, and some that do not fit it."""
    rng = np.random.default_rng(rows + K)
    m = Matrix(gpu, rng, rows, K)
    for nr in (5, 6, 7, 8):
        xq, xs = rows_of(rng, nr, K, K + 32)
        got = project(gpu, m, xq, xs, pad=3)
        check(got[:, -2000:], _last(m, 2000), xq, xs)
        check(got[:, :2000], _last(m, 2000, 0), xq, xs)
        for lo, hi in ((0, 1), (nr - 1, nr), (1, 5)):               # (every output against the other form's)
            assert np.array_equal(project(gpu, m, xq[lo:hi], xs[lo:hi]).view(np.uint32), got[lo:hi].view(np.uint32))


def _last(m, n, at=None):
    """Rows of a matrix on the host alone."""
    at = m.rows - n if at is None else at
    part = Matrix.__new__(Matrix)
    part.rows, part.K, part.alpha, part.w, part.s = n, m.K, m.alpha, m.w[at:at + n], m.s[at:at + n]
    return part


@pytest.mark.parametrize("rows,K", [(2560, 16), (2576, 1040), (8192, 272), (8208, 2064), (8208, 5120)])
@pytest.mark.parametrize("nr", [5, 7, 8])
def test_swiglu(gpu, rows, K, nr):
    rng = np.random.default_rng(rows + K + nr)
    gate, up = (Matrix(gpu, rng, rows, K, alpha=a / np.sqrt(K)) for a in (0.05, -0.03))
    xq, xs = rows_of(rng, nr, K, K + 48)
    q, s = swiglu(gpu, gate, up, xq, xs, 0.6)
    for at in (0, rows - 512):
        check_swiglu(q[:, at:at + 512], s[:, at // 16:at // 16 + 32], _last(gate, 512, at), _last(up, 512, at), xq, xs, 0.6)
    for lo, hi in ((0, 4), (4, nr)):
        q2, s2 = swiglu(gpu, gate, up, xq[lo:hi], xs[lo:hi], 0.6)
        assert np.array_equal(q2, q[lo:hi]) and np.array_equal(s2, s[lo:hi])


def test_every_code(gpu):
    """Every weight code by every activation code, each activation row with codes of its own; the products of a slab alone exact."""
    X, rng = gpu, np.random.default_rng(2)
    rows, K = 5120, 16 * 16
    m = Matrix(X, rng, rows, K, alpha=1.0, scales=np.full((rows, K // 16), 0x38, np.uint8))
    m.w[:] = ((np.arange(rows) % 16) * 17).astype(np.uint8)[:, None]
    m.bufs[0].upload(m.w)
    for i in range(16):                                             # codes 16 i - 128 .. of one slab, by rows of one code
        xq = np.zeros((8, K), np.int8)
        for n in range(8):
            slab = (i + 5 * n) % 16
            xq[n, 16 * slab:16 * slab + 16] = np.arange(16 * i - 128, 16 * i - 112)
            xq[n, 16 * slab + n] = 0
        y, _ = m.product(xq, np.ones((8, K // 16), np.float32))
        assert np.array_equal(project(X, m, xq, np.ones((8, K // 16), np.float32)).astype(np.float64), y)


@pytest.mark.parametrize("odd", [1, 6])
def test_any_alignment_outputs_and_residuals(gpu, odd):
    from ref64 import bf16_rne
    rng = np.random.default_rng(odd)
    m = Matrix(gpu, rng, 5131, 304, odd=odd, alpha=0.01)
    xq, xs = rows_of(rng, 7, 304, 320)
    res = bf16_rne(rng.standard_normal((7, 5140)).astype(np.float32) * 3)
    check(project(gpu, m, xq, xs, True, res, 0.75, odd=odd, pad=5), m, xq, xs, res, 0.75)


def test_not_finite_stays_with_its_rows(gpu):
    X, rng = gpu, np.random.default_rng(3)
    rows, K, nr = 5136, 1040, 7
    m = Matrix(X, rng, rows, K)
    xq, xs = rows_of(rng, nr, K)
    clean = project(X, m, xq, xs)
    bad, xb = m.s.copy(), xs.copy()
    at = [7, 39, 2000, rows - 1]
    bad[7, 3], bad[39, 64], bad[2000, 10], bad[rows - 1, 64] = 0x7F, 0xFF, 0x7F, 0x7F
    xb[4, 64] = np.inf
    m.bufs[1].upload(bad)
    got = project(X, m, xq, xb)
    assert np.isnan(got[:, at]).all() and not np.isfinite(got[4]).any()
    rest = np.setdiff1d(np.arange(rows), at)
    keep = [n for n in range(nr) if n != 4]
    assert np.array_equal(got[np.ix_(keep, rest)], clean[np.ix_(keep, rest)])


@pytest.mark.parametrize("rows,K", [(4097, 272), (4113, 1040), (5120, 784), (8193, 144), (9001, 1296), (12295, 16)])
def test_tiles_of_fewer_rows(gpu, rows, K):
    """More tiles than compute units, in even shares: all outputs of 1 to 4 rows, with residual, nothing beside them."""
    rng = np.random.default_rng(rows * K)
    m = Matrix(gpu, rng, rows, K, alpha=-0.03)
    for nr in (1, 2, 3, 4):
        xq, xs = rows_of(rng, nr, K, K + 16)
        res = rng.standard_normal((nr, rows + 2)).astype(np.float32)
        check(project(gpu, m, xq, xs, res=res, rs=0.5, pad=7), m, xq, xs, res, 0.5)


@pytest.mark.parametrize("rows,K,nrs", [(5120, 17408, (5, 6, 8)), (5137, 12304, (7, 8)), (8195, 17424, (5, 8)), (5121, 57344, (5, 8))])
def test_activations_in_turns(gpu, rows, K, nrs):
    """Rows that LDS does not hold at once, even shares of weight rows: the ends against float64, every output against fewer rows' bits."""
    rng = np.random.default_rng(rows + K)
    m = Matrix(gpu, rng, rows, K, alpha=-0.02)
    xq, xs = rows_of(rng, 8, K, K + 16)
    alone = [project(gpu, m, xq[n:n + 1], xs[n:n + 1])[0] for n in range(8)]
    part = [(0, 100), (rows - 100, rows), (2550, 2650)]
    for nr in nrs:
        got = project(gpu, m, xq[:nr], xs[:nr], pad=1)
        assert np.array_equal(got.view(np.uint32), np.array(alone[:nr]).view(np.uint32))
    for lo, hi in part:
        check(got[:, lo:hi], _last(m, hi - lo, lo), xq[:nr], xs[:nr])


@pytest.mark.parametrize("nr", [5, 8])
def test_swiglu_in_turns(gpu, nr):
    rng = np.random.default_rng(nr)
    rows, K = 2592, 12304
    gate, up = (Matrix(gpu, rng, rows, K, alpha=a / np.sqrt(K)) for a in (0.05, -0.03))
    xq, xs = rows_of(rng, nr, K)
    q, s = swiglu(gpu, gate, up, xq, xs, 0.6)
    check_swiglu(q[:, -96:], s[:, -6:], _last(gate, 96), _last(up, 96), xq, xs, 0.6)
    for n in range(nr):
        q1, s1 = swiglu(gpu, gate, up, xq[n:n + 1], xs[n:n + 1], 0.6)
        assert np.array_equal(q1[0], q[n]) and np.array_equal(s1[0], s[n])
