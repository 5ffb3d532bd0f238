"""q27x_sample_rows where a row's slices change their size, and logits at any element of memory."""
import numpy as np
import pytest

from ref64 import bf16_rne, bf2f
from test_gpu_sample import HOW, answers, check, logits, sample

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [65536, 65537, 100003, 131072, 131073, 262144, 262145])
@pytest.mark.parametrize("bf16", [False, True])
def test_slices(gpu, n, bf16):
    """At most 16 slices of 4096, 8192, 16384 or 32768 tokens: the last and first sizes of each."""
    rng = np.random.default_rng(n + bf16)
    x = logits(rng, 2, n, peaks=100)
    x[0, n - 1] = x[0].max() + 1                                    # (the last token leads)
    x = bf16_rne(x) if bf16 else x
    for how in ("plain", "all wide", "p high"):
        check(gpu, x, *HOW[how], rng.random(2).astype(np.float32))


@pytest.mark.parametrize("n", [1001, 62080])
@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("odd", [1, 2, 3])
def test_any_element(gpu, n, bf16, odd):
    """Logits that begin at any element, settings at any."""
    X, rng = gpu, np.random.default_rng(odd)
    x = logits(rng, 3, n)
    x = bf16_rne(x) if bf16 else x
    v = bf2f(x) if bf16 else x
    u = rng.random(3).astype(np.float32)
    pad = lambda a: X.DevBuf(array=np.concatenate([np.zeros(odd, a.dtype), a.reshape(-1)]))
    d = [pad(x), pad(np.full(3, 0.9, np.float32)), pad(np.full(3, 60, np.int32)), pad(np.full(3, 0.95, np.float32)), pad(np.full(3, 0.01, np.float32)),
         pad(u)]
    work = X.DevBuf(X.lib().q27x_sample_work_bytes(n, 3))
    idx, prob = X.DevBuf(4 * (3 + odd)), X.DevBuf(4 * (3 + odd))
    q = [b.ptr + odd * (2 if bf16 and b is d[0] else 4) for b in d]
    X.call("q27x_sample_rows", q[0], int(bf16), n, n, 3, *q[1:], work.ptr, idx.ptr + 4 * odd, prob.ptr + 4 * odd, None)
    X.call("q27x_device_sync")
    got = idx.download(np.int32, (3 + odd,))[odd:]
    f = np.float32
    for r in range(3):
        assert got[r] in answers(v[r], float(f(0.9)), 60, float(f(0.95)), float(f(0.01)), float(u[r]))


@pytest.mark.parametrize("n", [4097, 20000, 62080])
def test_few_and_many_blocks(gpu, n):
    """Rows on both sides of one block for each compute unit have the same tokens and probabilities."""
    X, rng = gpu, np.random.default_rng(n)
    x = np.repeat(logits(rng, 5, n), 30, 0)
    u = np.tile(rng.random(30).astype(np.float32), 5)
    for how in ("all", "p high"):
        t, k, p, m = HOW[how]
        full = lambda v, dt: np.full(150, v, dt)
        many = sample(X, x, full(t, np.float32), full(k, np.int32), full(p, np.float32), full(m, np.float32), u)
        few = [sample(X, x[i:i + 5], full(t, np.float32)[:5], full(k, np.int32)[:5], full(p, np.float32)[:5], full(m, np.float32)[:5], u[i:i + 5])
               for i in range(0, 150, 5)]
        for j in range(2):
            assert np.array_equal(np.concatenate([f[j] for f in few]), many[j])
