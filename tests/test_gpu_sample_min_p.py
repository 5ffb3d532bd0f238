"""q27x_sample_rows with min_p at and above 1 where logits tie for the largest: at 1 every one of them is kept, above it none reaches it and the
first alone is. Weights of ties are exactly 1, so every token is pinned. Rows of one block and of slices; few ties, counted among each
other, and many, searched for."""
import numpy as np
import pytest

from ref64 import bf16_rne
from test_gpu_sample import check, logits, sample

pytestmark = pytest.mark.gpu
ABOVE = [np.nextafter(np.float32(1), np.float32(2)), np.float32(1.5), np.float32(1e30), np.float32(np.inf)]
U = np.array([0.0, 0.3, 0.5, 0.75, 0.999], np.float32)


def rows_with_ties(rng, n, ties, bf16):
    x = np.repeat(logits(rng, 1, n), len(U), 0)
    at = np.sort(rng.choice(n, min(ties, n), replace=False))
    x[:, at] = 40.0
    return (bf16_rne(x) if bf16 else x), at


@pytest.mark.parametrize("n", [1, 2, 300, 4096, 9000, 62080, 140000])
@pytest.mark.parametrize("ties", [1, 2, 100, 1000])
@pytest.mark.parametrize("bf16", [False, True])
def test_ties_of_the_largest(gpu, n, ties, bf16):
    x, at = rows_with_ties(np.random.default_rng(n + ties), n, ties, bf16)
    full = lambda v: np.full(len(U), v, np.float32)
    for m in ABOVE:
        idx, prob = sample(gpu, x, m=full(m), u=U)
        assert (idx == at[0]).all() and (prob == 1).all(), (m, idx, at[:3])
    idx, prob = sample(gpu, x, m=full(1), u=U)
    assert idx.tolist() == [at[int(np.floor(float(u) * len(at)))] for u in U] and (prob == np.float32(1 / len(at))).all()


@pytest.mark.parametrize("n", [300, 5000, 62080])
def test_beside_other_cuts(gpu, n):
    """Above 1 with top-k and top-p that keep more, with a temperature that makes all tokens tie, and on greedy rows."""
    X, rng = gpu, np.random.default_rng(n)
    x, at = rows_with_ties(rng, n, 400, False)
    first = int(at[0])
    full = lambda v, dt=np.float32: np.full(len(U), v, dt)
    for m in ABOVE:
        for k, p in ((0, 0.9), (7, 1.0), (290, 0.5), (1, 0.1)):
            idx, prob = sample(X, x, k=full(k, np.int32), p=full(p), m=full(m), u=U)
            assert (idx == first).all() and (prob == 1).all(), (m, k, p)
        for t in (np.inf, 0.0, 1e-20):
            idx, prob = sample(X, x, t=full(t), m=full(m), u=U)
            assert (idx == first).all() and (prob == 1).all(), (m, t)
    y = logits(rng, 4, n)
    check(X, y, np.float32(0.8), 0, 1.0, np.array([1.0, 1.5, 0.5, 2.0]), rng.random(4))
