"""q27x_sample_rows on the GPU against the definition in float64.

A token is equal unless a random number or a cut falls next to a border. The kernel's weights are multiples of 2^-44 of the largest,
each off by half of that and 2^-46 of itself, so a running sum is off by (n/2 + S/4) 2^-44 (S: the sum of n weights), and what it is
compared with, a share of such a sum, by no more: together (n + S/2) 2^-44. Every row is checked against the definition at the numbers
given and at numbers that far to both sides (u and top_p by 1.5 n 2^-44 / S, min_p by 2^-43): tokens on a border may fall to either
side, all others are pinned. prob is off by those and half a step of fp32.
"""
import numpy as np
import pytest

from ref64 import bf16_rne, bf2f

pytestmark = pytest.mark.gpu


def reference(x, t, k, p, m, u):
    """(token, probability, sum of the weights) of one row by the definition."""
    x = np.asarray(x, np.float64)
    ids = np.flatnonzero(np.isfinite(x))
    if not len(ids):
        return 0, 0.0, 1.0
    ids = ids[np.lexsort((ids, -x[ids]))]
    if not t > 0:
        return int(ids[0]), 1.0, 1.0
    w = np.exp((x[ids] - x[ids[0]]) / t)
    total = w.sum()
    if k >= 1:
        w = w[:k]
    if p < 1:
        sums = np.cumsum(w)
        w = w[:max(1, int(np.searchsorted(sums, max(p, 0) * sums[-1], side="left")) + 1)]
    if m > 0:
        w = w[:max(1, int((w >= m).sum()))]
    sums = np.cumsum(w)
    i = min(int(np.searchsorted(sums, max(u, 0) * sums[-1], side="right")), len(w) - 1)
    return int(ids[i]), w[i] / sums[-1], total


def answers(x, t, k, p, m, u):
    """{token: probability} at the numbers given and at the ends of what rounding may make of them."""
    i, pr, total = reference(x, t, k, p, m, u)
    d = 1.5 * len(x) * 2.0 ** -44 / total
    got = {i: [pr]}
    for pp in (p - d, p, p + d) if 0 < p < 1 else (p,):
        for mm in (m - 2.0 ** -43, m, m + 2.0 ** -43) if 0 < m < 1 else (m,):
            for uu in (u - d, u, u + d):
                i, pr, _ = reference(x, t, k, pp, mm, uu)
                got.setdefault(i, []).append(pr)
    return got


def sample(X, x, t=None, k=None, p=None, m=None, u=None, ld=None, prob=True, stream=None, fill=0x5A):
    """idx, prob of the call on rows x (fp32 or bf16 bits); a workspace full of something."""
    nr, n = x.shape
    ld = n if ld is None else ld
    buf = np.full((nr, ld), 0x7149 if x.dtype == np.uint16 else 3e38, x.dtype)
    buf[:, :n] = x
    dev = lambda a, dt: None if a is None else X.DevBuf(array=np.ascontiguousarray(a, dt))
    d = [dev(buf, x.dtype), dev(t, np.float32), dev(k, np.int32), dev(p, np.float32), dev(m, np.float32), dev(u, np.float32)]
    work = X.DevBuf(array=np.full(X.lib().q27x_sample_work_bytes(n, nr), fill, np.uint8))
    idx, pr = X.DevBuf(array=np.full(nr + 1, -7, np.int32)), X.DevBuf(array=np.full(nr + 1, -7.0, np.float32))
    q = [b.ptr if b else None for b in d]
    X.call("q27x_sample_rows", q[0], int(x.dtype == np.uint16), n, ld, nr, *q[1:], work.ptr, idx.ptr, pr.ptr if prob else None, stream)
    X.call("q27x_device_sync")
    i, f = idx.download(np.int32, (nr + 1,)), pr.download(np.float32, (nr + 1,))
    assert i[nr] == -7 and f[nr] == -7 and (prob or (f == -7).all()), "behind the rows was written"
    return i[:nr], f[:nr]


def check(X, x, t, k, p, m, u, **kw):
    nr, n = x.shape
    v = bf2f(x) if x.dtype == np.uint16 else x
    full = lambda a, d, dt: np.full(nr, d, dt) if a is None else np.broadcast_to(np.asarray(a, dt), (nr,)).copy()
    t_, k_, p_, m_, u = full(t, 1, np.float32), full(k, 0, np.int32), full(p, 1, np.float32), full(m, 0, np.float32), full(u, 0, np.float32)
    idx, prob = sample(X, x, None if t is None else t_, None if k is None else k_, None if p is None else p_, None if m is None else m_, u, **kw)
    pinned = 0
    for r in range(nr):
        want = answers(v[r], float(t_[r]), int(k_[r]), float(p_[r]), float(m_[r]), float(u[r]))
        pinned += len(want) == 1
        assert idx[r] in want, (r, idx[r], want, prob[r])
        assert min(abs(prob[r] - pr) - pr * (2.0 ** -24 + 2.0 ** -43) for pr in want[idx[r]]) <= 1.5 * n * 2.0 ** -44, (r, prob[r], want)
    assert 2 * pinned >= nr, (pinned, nr)         # (or nothing was tested)
    return idx, prob


def logits(rng, nr, n, std=2.0, peaks=40):
    x = rng.standard_normal((nr, n)) * std
    for r in range(nr):
        at = rng.integers(0, n, min(peaks, n))
        x[r, at] += rng.exponential(2.5, len(at)) + 2
    return x.astype(np.float32)


SIZES = [1, 2, 3, 63, 64, 65, 1000, 4095, 4096, 4097, 20000, 62080]
HOW = {"plain": (1.0, 0, 1.0, 0.0), "hot": (3.0, 0, 1.0, 0.0), "cold": (0.05, 0, 1.0, 0.0), "k": (0.8, 40, 1.0, 0.0), "k1": (1.0, 1, 1.0, 0.0),
       "k many": (1.1, 3000, 1.0, 0.0), "p": (0.9, 0, 0.9, 0.0), "p low": (1.0, 0, 0.05, 0.0), "p high": (1.2, 0, 0.9999, 0.0),
       "m": (1.0, 0, 1.0, 0.05), "m tiny": (1.5, 0, 1.0, 1e-9), "all": (0.7, 50, 0.95, 0.02), "all wide": (1.3, 2500, 0.999, 1e-5)}


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("how", HOW)
def test_settings_and_sizes(gpu, how, bf16):
    rng = np.random.default_rng(len(how) + bf16)
    t, k, p, m = HOW[how]
    for n in SIZES:
        x = logits(rng, 7, n)
        x = bf16_rne(x) if bf16 else x
        check(gpu, x, t, k, p, m, rng.random(7).astype(np.float32), ld=n + n % 5)


def test_whole_vocabulary(gpu):
    rng = np.random.default_rng(1)
    x = logits(rng, 3, 248320, peaks=200)
    for how in ("plain", "all", "p high"):
        check(gpu, x, *HOW[how], rng.random(3).astype(np.float32))
        check(gpu, bf16_rne(x), *HOW[how], rng.random(3).astype(np.float32))
    x = logits(rng, 1, 1 << 19, std=0.5, peaks=0)
    check(gpu, x, *HOW["plain"], [0.7])


def test_rows_of_a_batch_with_their_own_settings(gpu):
    """150 rows of every kind, greedy ones among them; each the same alone and without prob."""
    X, rng = gpu, np.random.default_rng(2)
    nr, n = 150, 5003
    x = logits(rng, nr, n)
    t = rng.choice([0.0, -1.0, 0.3, 0.9, 2.0], nr).astype(np.float32)
    k = rng.choice([0, -3, 1, 5, 50, 5002, 5003, 2 ** 31 - 1], nr).astype(np.int32)
    p = rng.choice([1.0, 1.5, 0.5, 0.97, 0.0, -1.0], nr).astype(np.float32)
    m = rng.choice([0.0, -1.0, 0.01, 0.3, 1.0, 2.0], nr).astype(np.float32)
    u = rng.random(nr).astype(np.float32)
    idx, prob = check(X, x, t, k, p, m, u)
    for r in range(0, nr, 17):
        i, f = sample(X, x[r:r + 1], t[r:r + 1], k[r:r + 1], p[r:r + 1], m[r:r + 1], u[r:r + 1], fill=0xFF)
        assert i[0] == idx[r] and f[0] == prob[r]
    i, _ = sample(X, x, t, k, p, m, u, prob=False)
    assert np.array_equal(i, idx)


def test_no_settings_and_unlikely_numbers(gpu):
    """NULL for every setting; numbers at and outside the ends; settings that are not numbers cut nothing."""
    X, rng = gpu, np.random.default_rng(3)
    x = logits(rng, 6, 700)
    order = np.argsort(-x, axis=1, kind="stable")
    u = np.array([0.0, -0.5, np.nan, 1.0, 7.0, 0.5], np.float32)
    idx, _ = sample(X, x, u=u)
    assert idx[:3].tolist() == order[:3, 0].tolist()
    assert idx[3:5].tolist() == order[3:5, -1].tolist()             # (all within 2^-44 of the largest)
    assert idx[5] == reference(x[5], 1, 0, 1, 0, 0.5)[0]
    nan = np.full(6, np.nan, np.float32)
    assert np.array_equal(sample(X, x, p=nan, m=nan, u=u)[0], idx)
    assert np.array_equal(sample(X, x, t=nan, u=u)[0], order[:, 0])


def test_greedy_like_argmax(gpu):
    """Temperature 0 takes what q27x_argmax_rows takes: ties, both zeros, values that are not finite."""
    X, rng = gpu, np.random.default_rng(4)
    x = rng.integers(-3, 3, (8, 9001)).astype(np.float32)
    x[1, 5] = np.inf
    x[2, ::2] = np.nan
    x[3] = -np.inf
    x[4] = -0.0
    x[4, 77] = 0.0
    x[5, :] = -1e30
    idx, prob = sample(X, x, t=np.zeros(8), k=np.full(8, 7), p=np.full(8, 0.3), m=np.full(8, 0.5), u=np.full(8, 0.99))
    d, di, dv = X.DevBuf(array=x), X.DevBuf(32), X.DevBuf(32)
    X.call("q27x_argmax_rows", d.ptr, 9001, 9001, 8, di.ptr, dv.ptr, None)
    X.call("q27x_device_sync")
    assert np.array_equal(idx, di.download(np.int32, (8,)))
    assert prob.tolist() == [1.0, 1.0, 1.0, 0.0, 1.0, 1.0, 1.0, 1.0]


def test_logits_that_are_not_finite_are_left_out(gpu):
    rng = np.random.default_rng(5)
    x = logits(rng, 8, 6000)
    x[rng.random(x.shape) < 0.3] = -np.inf
    x[rng.random(x.shape) < 0.1] = np.nan
    x[rng.random(x.shape) < 0.01] = np.inf
    x[6] = -np.inf
    x[6, 4321] = -5.0
    x[7] = -np.finfo(np.float32).max                                # (a mask of the type's lowest value)
    x[7, [10, 5990]] = [1.0, 1.5]
    for how in ("plain", "all", "p", "m"):
        check(gpu, x, *HOW[how], rng.random(8).astype(np.float32))
    assert sample(gpu, np.full((1, 4100), np.nan, np.float32), u=[0.3])[0][0] == 0


@pytest.mark.parametrize("n", [5, 3000, 9000, 62080])
@pytest.mark.parametrize("bf16", [False, True])
def test_equal_logits(gpu, n, bf16):
    """All equal: the token at floor(u x kept), whatever cuts; every weight is 1, so borders are exact."""
    X, rng = gpu, np.random.default_rng(n)
    x = np.full((8, n), 1.25, np.float32)
    x = bf16_rne(x) if bf16 else x
    u = np.array([0.0, 0.25, 0.5, 0.75, 0.999, 0.125, 0.6, 0.3], np.float32)
    k = np.array([0, 0, 3, n, n // 2, 0, n - 1, 0], np.int32)
    p = np.array([1, 0.5, 1, 1, 0.5, 0.25, 1, 0.75], np.float32)
    m = np.array([0, 0, 0, 1.0, 0, 1.0, 0.5, 0], np.float32)
    idx, prob = sample(X, x, k=k, p=p, m=m, u=u)
    for r in range(8):
        kept = min(int(k[r]), n) if k[r] > 0 else n
        kept = max(1, int(np.ceil(float(p[r]) * kept)))
        assert idx[r] == int(np.floor(float(u[r]) * kept)), r
        assert prob[r] == np.float32(1 / kept)


def test_few_values_many_ties(gpu):
    """Logits on a grid of 8 values: cuts and draws inside ties take the lowest indexes first."""
    rng = np.random.default_rng(7)
    for n in (300, 5000, 62080):
        x = rng.integers(0, 8, (12, n)).astype(np.float32)
        check(gpu, x, np.float32(1.7), np.array([0, 1, 7, n // 3, n // 2, n - 1] * 2), np.float32(0.83), np.float32(0.0), rng.random(12))
        check(gpu, x, np.float32(0.9), 0, np.float32(0.31), np.float32(0.01), rng.random(12))


def test_exact_borders(gpu):
    """Weights that are powers of two: cuts and numbers exactly on a border. Running sums 1, 1.5, 1.75, 2, 2.125 ... : a cut that a
    sum reaches ends there; a number that a running sum only reaches goes on to the next token."""
    X = gpu
    ln2 = np.log(2)
    t = np.float32(1 / ln2)                                          # w = 2^(l - l0) to 2^-24 of the exponent: whole exponents
    x = np.array([[0, -40, -1, -2, -2, -40, 0]], np.float32)         # order 0 6 2 3 4 (1 5): w 1 1 .5 .25 .25 2^-40 2^-40
    for k, u, want in ((2, 0.5, 6), (2, 0.49, 0), (4, 0.0, 0), (1, 0.9, 0), (5, 0.999, 4)):
        assert sample(X, x, t=[t], k=[k], u=[u])[0][0] == want, (k, u)
    assert sample(X, x, t=[t], k=[2], p=[0.5], u=[0.99])[0][0] == 0   # two of weight 1: the first reaches half
    assert sample(X, x, t=[t], k=[2], p=[0.51], u=[0.99])[0][0] == 6
    assert sample(X, x, t=[t], m=[1.0], u=[0.99])[0][0] == 6


@pytest.mark.parametrize("t", [1e-30, 1e-6, 1e6, 1e30, np.inf])
def test_temperatures_far_out(gpu, t):
    """Very cold: the largest (equal ones share); very hot: all alike."""
    X, rng = gpu, np.random.default_rng(8)
    x = logits(rng, 4, 5000)
    x[0, [7, 4000]] = 90.0
    u = np.array([0.7, 0.2, 0.5, 0.9], np.float32)
    idx, _ = sample(X, x, t=np.full(4, t), u=u)
    if t < 1:
        assert idx.tolist() == [4000] + np.argmax(x[1:], axis=1).tolist()
    elif t >= 1e30:
        order = np.argsort(-x, axis=1, kind="stable")
        assert idx.tolist() == [order[r, int(np.floor(float(u[r]) * 5000))] for r in range(4)]
    else:
        check(X, x, np.float32(t), 0, 1.0, 0.0, u)


def test_frequencies(gpu):
    """An even grid of numbers draws each token as often as its probability says, to one number of the grid."""
    X, rng = gpu, np.random.default_rng(9)
    x = np.repeat(logits(rng, 1, 50), 4096, 0)
    u = ((np.arange(4096) + 0.5) / 4096).astype(np.float32)
    idx, prob = sample(X, x, t=np.full(4096, 0.8), u=u)
    w = np.exp((x[0].astype(np.float64) - x[0].max()) / np.float64(np.float32(0.8)))
    w /= w.sum()
    got = np.bincount(idx, minlength=50) / 4096
    assert (np.abs(got - w) <= 1 / 4096).all()
    assert (np.abs(prob - w[idx]) <= 2.0 ** -23 * w[idx]).all()
