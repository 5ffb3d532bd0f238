"""What q27x_sample_rows refuses, on the host, before any GPU call, and its workspace."""
import pytest

ARG, SHAPE = -1, -2
P = 1 << 20                                     # a stand-in address: refused calls touch no memory


def sample(X, **kw):
    a = dict(logits=P, bf16=0, n=1000, ld=1000, nr=3, t=P, k=P, p=P, m=P, u=P, work=P, idx=P, prob=P)
    a.update(kw)
    return X.lib().q27x_sample_rows(*(a[c] for c in ("logits", "bf16", "n", "ld", "nr", "t", "k", "p", "m", "u", "work", "idx", "prob")), None)


@pytest.mark.parametrize("kw,rc", [(dict(logits=None), ARG), (dict(u=None), ARG), (dict(work=None), ARG), (dict(idx=None), ARG),
                                   (dict(work=P + 8), ARG), (dict(n=0), SHAPE), (dict(n=-1), SHAPE), (dict(n=(1 << 19) + 1), SHAPE),
                                   (dict(nr=0), SHAPE), (dict(nr=65536), SHAPE), (dict(ld=999), ARG), (dict(ld=-1), ARG)])
def test_refused(X, kw, rc):
    assert sample(X, **kw) == rc
    assert X.lib().q27x_last_error().decode().startswith("q27x_sample_rows")


def test_work_bytes(X):
    f = X.lib().q27x_sample_work_bytes
    assert 0 < f(1, 1) <= f(1000, 1) < f(62080, 1) < f(62080, 2) and f(1 << 19, 1) > 1 << 20
    assert f(0, 1) == f(1, 0) == f((1 << 19) + 1, 1) == f(1, 65536) == 0
    assert f(1 << 19, 65535) > 1 << 36           # a size that passes 32 bits
