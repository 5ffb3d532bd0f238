"""The paged-cache operators on the GPU against their float64 forms (paged_ref.py).

Tolerances, elementwise, from the roundings on the way (u = 2^-24, a bf16 result is off by at most 2^-8 of itself):
- prepared rows: a head's norm and a turn are fewer than 64 fp32 roundings of values no larger than |a| + |b|, the pair's
  normed values: 2^-18 (|a| + |b|); bf16 adds 2^-8 of the result; a code is off by half a scale and those.
- attention: a score is hd + 8 fp32 roundings of terms of |q k| / sqrt(hd), so a weight is off by d = 2 (hd + 8) u max
  sum |q k| / sqrt(hd) relative at most, and its normalised form by 2 d; the sums add (keys + 64) u. Weights and values
  enter with 11 bits each (2^-11 relative; below 2^-14 an absolute 2^-25 of the largest scale), sum p |v| bounds what
  they multiply.
- eviction: sums in the documented order of fp32 operations and moved bytes are equal.
"""
import ctypes

import numpy as np
import pytest

from paged_ref import Cache, attention, bf, evict, rmsnorm, rotate, tables
from ref64 import bf2f, sigmoid

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
GEOMS = {"4x1x128": (4, 1, 128), "6x1x256": (6, 1, 256), "32x8x128": (32, 8, 128), "24x4x256": (24, 4, 256), "3x3x128": (3, 3, 128),
         "40x2x128": (40, 2, 128)}


# ---------------------------------------------------------------- prep
def run_prep(X, cache, rng, geom, rot, n_axes, axes, gate, n_pos=64, tail=0, odd=0, row_start=True, pos=None):
    nq, nkv, hd = geom
    n = int(cache.row_start[-1]) + tail
    qw = (2 if gate else 1) * hd
    width = nq * qw + 2 * nkv * hd
    x = np.zeros((n, width + odd), np.uint16)
    x[:, :width] = bf(rng.standard_normal((n, width)) * 2)
    qn, kn = bf(rng.standard_normal(hd) * 0.2), bf(rng.standard_normal(hd) * 0.2)
    pos = rng.integers(0, n_pos, (n_axes, n)).astype(np.int32) if pos is None else pos
    cos, sin = tables(n_pos, rot)
    kv = cache.push(X, row_start)
    dev = [X.DevBuf(array=a) for a in (x, qn, kn, cos, sin, pos)]
    qh = X.DevBuf(array=np.full((n, nq * hd), 0x1234, np.uint16))
    ax = (ctypes.c_uint8 * (rot // 2))(*axes) if axes is not None else None
    X.call("q27x_paged_prep_rows", dev[0].ptr, width + odd, dev[1].ptr, dev[2].ptr, dev[3].ptr, dev[4].ptr, rot, n_pos, dev[5].ptr, n,
           n_axes, ax, ctypes.byref(kv), qh.ptr, nq, int(gate), 1e-6, n, None)
    X.call("q27x_device_sync")
    f = bf2f(x).astype(np.float64)
    q = f[:, :nq * qw].reshape(n, nq, qw)[..., :hd]
    k = f[:, nq * qw:nq * qw + nkv * hd].reshape(n, nkv, hd)
    v = f[:, nq * qw + nkv * hd:width].reshape(n, nkv, hd)
    yq, yk = rmsnorm(q, bf2f(qn).astype(np.float64), 1e-6), rmsnorm(k, bf2f(kn).astype(np.float64), 1e-6)
    p = np.clip(pos, 0, n_pos - 1)
    ax = [0] * (rot // 2) if axes is None else list(axes)
    return qh.download(np.uint16, (n, nq * hd)).reshape(n, nq, hd), cache.pull(), (yq, yk, v, rotate(yq, p, ax, rot), rotate(yk, p, ax, rot))


def pair_size(y, rot):
    """|a| + |b| of a dim's pair, |y| behind the rotary dims."""
    m = np.abs(y)
    half = rot // 2
    s = m[..., :half] + m[..., half:rot]
    return np.concatenate([s, s, m[..., rot:]], -1)


def check_prep(cache, got_q, got, ref, rot, skip=()):
    yq, yk, v, rq, rk = ref
    n = int(cache.row_start[-1])
    tol = 2.0 ** -8 * np.abs(rq) + 2.0 ** -18 * pair_size(yq, rot)
    assert (np.abs(bf2f(got_q[:n]) - rq[:n]) <= tol[:n]).all()
    assert (got_q[n:] == 0x1234).all(), "rows behind the last sequence were written"
    written = np.zeros(len(cache.k), bool)
    for b, cnt in enumerate(cache.counts):
        for i in range(cnt):
            r, slot = cache.row_start[b] + i, cache.slot(b, int(cache.lens[b]) - cnt + i)
            if slot < 0:
                continue
            written[slot] = True
            for name, want, size in (("k", rk[r], pair_size(yk[r], rot)), ("v", v[r], np.abs(v[r]))):
                want, size = want.reshape(-1), size.reshape(-1)
                if not cache.group:
                    assert (np.abs(bf2f(got[name][slot]) - want) <= 2.0 ** -8 * np.abs(want) + 2.0 ** -18 * size).all()
                    continue
                s = got[name + "s"][slot].astype(np.float64)
                top = np.abs(want.reshape(-1, cache.group)).max(1) / 127
                big = size.reshape(-1, cache.group).max(1)
                assert (np.abs(s - top) <= 2.0 ** -18 * big / 127 + 2.0 ** -22 * top).all()
                off = np.abs(got[name][slot].reshape(-1, cache.group) * s[:, None] - want.reshape(-1, cache.group))
                assert (off <= (0.5 + 2.0 ** -14) * s[:, None] + 2.0 ** -17 * big[:, None]).all()
    for name, a in got.items():
        keep = np.ascontiguousarray(a[~written])
        assert np.array_equal(keep, np.ascontiguousarray(getattr(cache, name)[~written])), f"{name}: other positions were written"


@pytest.mark.parametrize("group", [0, 16, 32, 64])
@pytest.mark.parametrize("geom,rot", [("4x1x128", 32), ("6x1x256", 64), ("32x8x128", 128), ("24x4x256", 66), ("3x3x128", 2), ("6x1x256", 256)])
def test_prep_rows(gpu, group, geom, rot):
    """Ragged batches with a sequence that has no row, three axes in turn, a gate beside the queries."""
    rng = np.random.default_rng(rot + group)
    nq, nkv, hd = GEOMS[geom]
    cache = Cache(rng, [5, 1, 40, 17, 16], [5, 1, 3, 0, 7], nkv, hd, group, page=8, fill=False)
    axes = [i % 3 for i in range(rot // 2)]
    q, got, ref = run_prep(gpu, cache, rng, GEOMS[geom], rot, 3, axes, True)
    check_prep(cache, q, got, ref, rot)


@pytest.mark.parametrize("group", [0, 32])
def test_prep_sections_tail_and_odd_rows(gpu, group):
    """Axes in sections, four of them; no gate; an odd row stride; rows behind the last sequence; positions outside the
    tables taken as the nearest end."""
    rng = np.random.default_rng(3)
    cache = Cache(rng, [9, 30], [2, 11], 2, 128, group, page=4, fill=False)
    axes = [0] * 7 + [1] * 3 + [3] * 4 + [2] * 2
    pos = rng.integers(-5, 80, (4, 16)).astype(np.int32)
    q, got, ref = run_prep(gpu, cache, rng, (6, 2, 128), 32, 4, axes, False, tail=3, odd=5, pos=pos)
    check_prep(cache, q, got, ref, 32)


def test_prep_one_row_per_sequence_and_many_sequences(gpu):
    """No row_start: row b is sequence b's; more sequences than a wave looks through at once, with row_start too."""
    rng = np.random.default_rng(4)
    for row_start in (False, True):
        cache = Cache(rng, rng.integers(1, 20, 150), [1] * 150, 1, 128, 32, page=16, fill=False)
        q, got, ref = run_prep(gpu, cache, rng, (4, 1, 128), 32, 1, None, True, tail=2, row_start=row_start)
        check_prep(cache, q, got, ref, 32)


def test_prep_pages_that_are_not_there(gpu):
    """A page outside the pool, a negative one, a position behind the table or before 0: nothing is written."""
    rng = np.random.default_rng(5)
    cache = Cache(rng, [10, 12, 20, 1], [4, 4, 4, 3], 2, 128, 32, page=4, fill=False, cap=16)
    cache.table[0, 2] = cache.n_pages
    cache.table[1, 2] = -7
    q, got, ref = run_prep(gpu, cache, rng, (4, 2, 128), 32, 1, None, True)
    check_prep(cache, q, got, ref, 32)


@pytest.mark.parametrize("group", [0, 32])
def test_prep_pages_of_keys_and_values_in_turn(gpu, group):
    """A pool whose pages hold keys, then values: page_stride is twice the page."""
    rng = np.random.default_rng(6)
    cache = Cache(rng, [21, 9], [6, 9], 2, 128, group, page=8, page_stride=16, fill=False)
    q, got, ref = run_prep(gpu, cache, rng, (4, 2, 128), 32, 1, None, True)
    check_prep(cache, q, got, ref, 32)


def test_prep_like_the_contiguous_entry(gpu):
    """One axis over pages that count up is q27x_attn_prep_rows: the same scales and values to fp32 rounding, codes off by one
    at ties at most."""
    X, rng = gpu, np.random.default_rng(7)
    nq, nkv, hd, n, pos0 = 8, 2, 128, 8, 21
    cache = Cache(rng, [pos0 + n], [n], nkv, hd, 32, page=16, spare=0, fill=False)
    cache.table[0] = np.arange(cache.n_pages)
    pos = (pos0 + np.arange(n, dtype=np.int32))[None]
    st = rng.bit_generator.state
    q, got, _ = run_prep(X, cache, rng, (nq, nkv, hd), 32, 1, None, True, pos=pos)
    rng.bit_generator.state = st
    width = nq * 2 * hd + 2 * nkv * hd
    x = bf(rng.standard_normal((n, width)) * 2)
    qn, kn = bf(rng.standard_normal(hd) * 0.2), bf(rng.standard_normal(hd) * 0.2)
    cos, sin = tables(64, 32)
    other = Cache(rng, [pos0 + n], [n], nkv, hd, 32, page=16, spare=0, fill=False)
    other.push(X)
    dev = [X.DevBuf(array=a) for a in (x, qn, kn, cos, sin)]
    qh = X.DevBuf(n * nq * hd * 2)
    X.call("q27x_attn_prep_rows", dev[0].ptr, width, dev[1].ptr, dev[2].ptr, dev[3].ptr, dev[4].ptr, 32, other.d["k"].ptr,
           other.d["ks"].ptr, other.d["v"].ptr, other.d["vs"].ptr, 32, qh.ptr, nq, nkv, hd, 1, 1e-6, pos0, n, None)
    X.call("q27x_device_sync")
    want = other.pull()
    assert np.array_equal(got["v"], want["v"]) and np.array_equal(got["vs"], want["vs"])
    # (each side is within 64 fp32 roundings of the exact value)
    assert np.abs(got["ks"] / want["ks"] - 1).max() <= 2.0 ** -17
    assert np.abs(got["k"].astype(int) - want["k"]).max() <= 1 and (got["k"] != want["k"]).mean() < 0.01
    a, b = bf2f(q.reshape(n, -1)), bf2f(qh.download(np.uint16, (n, nq * hd)))
    assert (np.abs(a - b) <= 2.0 ** -7 * np.abs(b) + 2.0 ** -15).all()


# ---------------------------------------------------------------- attention
def run_attn(X, cache, q, gate, nq, weights=True, codes=True, max_len=None, max_rows=None, tail=0, odd=0, row_start=True, stream=None):
    """q [row][head][dim] bf16, gate the same or None -> out, codes, scales, weights as they lie."""
    n, hd = int(cache.row_start[-1]) + tail, cache.hd
    max_len = max(int(max(cache.lens)), 1) if max_len is None else max_len
    max_rows = max(1, int(max(cache.counts))) if max_rows is None else max_rows
    kv = cache.push(X, row_start)
    dq = X.DevBuf(array=q)
    width = nq * 2 * hd + 2 * cache.nkv * hd + odd
    g = np.zeros((n, width), np.uint16)
    if gate is not None:
        g[:, :nq * 2 * hd].reshape(n, nq, 2, hd)[:, :, 1] = gate
    dg = X.DevBuf(array=g)
    out = X.DevBuf(array=np.full((n, nq * hd), 0x1234, np.uint16))
    xq, xs = X.DevBuf(array=np.full(n * nq * hd, 55, np.int8)), X.DevBuf(array=np.full(n * nq * hd // 16, 5, np.float32))
    w = X.DevBuf(array=np.full((n, max_len + 2), -3, np.float32))
    nb = X.lib().q27x_paged_attn_work_bytes(nq, hd, max_len, n, int(weights))
    work = X.DevBuf(array=np.full(nb, 0xFF, np.uint8))             # (not a number wherever it is read as floats)
    X.call("q27x_paged_attn_rows", dq.ptr, dg.ptr if gate is not None else None, width, ctypes.byref(kv), nq, int(gate is not None),
           max_len, max_rows, n, work.ptr, out.ptr, xq.ptr if codes else None, xs.ptr if codes else None, w.ptr if weights else None,
           max_len + 2, stream)
    X.call("q27x_device_sync")
    return (out.download(np.uint16, (n, nq, hd)), xq.download(np.int8, (n, nq * hd)), xs.download(np.float32, (n, nq * hd // 16)),
            w.download(np.float32, (n, max_len + 2)))


def queries(rng, n, nq, hd, std=1.5):
    return bf(rng.standard_normal((n, nq, hd)) * std), bf(rng.standard_normal((n, nq, hd)))


def check_attn(cache, got, q, gate, nq, max_len=None, weights=True, rows=None):
    out, xq, xs, w = got
    n, hd, L = int(cache.row_start[-1]), cache.hd, int(max(max(cache.lens), 1))
    ref, mag, rw, big = attention(cache, bf2f(q).astype(np.float64), nq, max_len)
    sg = sigmoid(bf2f(gate).astype(np.float64)) if gate is not None else np.ones(q.shape)
    d = 2 * (hd + 8) * U * big
    rel = (2 * 2.0 ** -11 + 2 * d + (L + 64) * U + 2.0 ** -20)[:, None, None]
    small = 2.0 ** -24 * L * (np.abs(cache.vs).max() * 127 if cache.group else 6.0)
    tol = 2.0 ** -8 * np.abs(ref[:n] * sg[:n]) + sg[:n] * (rel * mag + small)[:n]
    pick = np.arange(n) if rows is None else np.asarray(rows)
    off = np.abs(bf2f(out[:n]) - ref[:n] * sg[:n])
    assert (off <= tol)[pick].all(), f"worst {np.nanmax((off / tol)[pick]):.3g} of the tolerance"
    # (a rounding error is random: the whole result is far nearer than its bound, near bf16's own 2^-9.3)
    err = np.linalg.norm((bf2f(out[:n]) - ref[:n] * sg[:n])[pick]) / max(np.linalg.norm((ref[:n] * sg[:n])[pick]), 1e-30)
    assert err <= 2.0 ** -8, err
    assert (out[n:] == 0x1234).all() and (xq[n:] == 55).all() and (w[n:] == -3).all()
    # codes of the bf16 output, exactly
    y = bf2f(out[pick]).reshape(len(pick), -1, 16)
    s = (np.abs(y).max(-1) * np.float32(1 / 127)).astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(s > 0, np.float32(1) / s, np.float32(0)).astype(np.float32)
    assert np.array_equal(xs[pick], s) and np.array_equal(xq[pick].reshape(y.shape), np.clip(np.rint(y * inv[..., None]), -127, 127))
    if weights:
        for b, cnt in enumerate(cache.counts):
            for i in range(cnt):
                r, m = cache.row_start[b] + i, int(cache.lens[b])
                if rows is not None and r not in rows:
                    continue
                assert (np.abs(w[r, :m] - rw[r, :m]) <= rw[r, :m] * (2 * d[r] + (m + nq + 64) * U + 2.0 ** -20) + nq * 2.0 ** -120).all()
                assert (w[r, m:] == -3).all(), "weights behind the sequence's length were written"


LENS = [1, 2, 63, 64, 65, 255, 256, 257, 600]


@pytest.mark.parametrize("group", [0, 16, 32, 64])
@pytest.mark.parametrize("geom", list(GEOMS))
def test_attention_one_row(gpu, group, geom):
    """One new token of sequences whose lengths sit at the borders of tiles, chunks and splits."""
    rng = np.random.default_rng(group)
    nq, nkv, hd = GEOMS[geom]
    cache = Cache(rng, LENS, [1] * len(LENS), nkv, hd, group, page=16)
    q, gate = queries(rng, len(LENS), nq, hd)
    check_attn(cache, run_attn(gpu, cache, q, gate, nq), q, gate, nq)


@pytest.mark.parametrize("group", [0, 16, 32, 64])
@pytest.mark.parametrize("geom", list(GEOMS))
def test_attention_rows(gpu, group, geom):
    """1 to 8 rows of a sequence, more rows than keys (the first see nothing), a sequence without rows, one without keys,
    rows behind the last sequence."""
    rng = np.random.default_rng(50 + group)
    nq, nkv, hd = GEOMS[geom]
    counts = [3, 8, 0, 5, 1, 2, 4]
    cache = Cache(rng, [70, 300, 40, 3, 0, 513, 64], counts, nkv, hd, group, page=32)
    q, gate = queries(rng, sum(counts) + 2, nq, hd)
    check_attn(cache, run_attn(gpu, cache, q, gate, nq, tail=2, odd=3), q, gate, nq)


@pytest.mark.parametrize("page", [1, 2, 8, 64, 1024])
def test_attention_pages(gpu, page):
    """Pages smaller than a tile, and larger than a split; no gate, no weights, no codes."""
    rng = np.random.default_rng(page)
    cache = Cache(rng, [37, 300], [1, 2], 2, 128, 32, page=page, page_stride=2 * page)
    q, _ = queries(rng, 3, 8, 128)
    out, xq, xs, w = run_attn(gpu, cache, q, None, 8, weights=False, codes=False)
    assert (w == -3).all() and (xq == 55).all()
    got = out, *[a for a in run_attn(gpu, cache, q, None, 8)[1:]]
    check_attn(cache, got, q, None, 8)


def test_attention_long(gpu):
    """Many splits: a long sequence beside short ones."""
    rng = np.random.default_rng(8)
    cache = Cache(rng, [20011, 5, 4100], [2, 1, 3], 1, 128, 32, page=64)
    q, gate = queries(rng, 6, 4, 128)
    check_attn(cache, run_attn(gpu, cache, q, gate, 4), q, gate, 4)


def test_attention_peaked_scores(gpu):
    """Queries that make one key take all: weights down to underflow."""
    rng = np.random.default_rng(9)
    cache = Cache(rng, [400, 90], [1, 2], 2, 128, 32)
    q, gate = queries(rng, 3, 8, 128, std=40.0)
    check_attn(cache, run_attn(gpu, cache, q, gate, 8), q, gate, 8)


@pytest.mark.parametrize("group", [0, 32])
def test_attention_keys_that_are_not_there(gpu, group):
    """Pages outside the pool are passed over; max_len and the table's end cut a sequence; a row with nothing left gets
    zeros; what lies behind the length, NaN and infinities, does not enter."""
    rng = np.random.default_rng(10)
    cache = Cache(rng, [300, 200, 20, 90], [1, 2, 1, 1], 2, 128, group, page=16, cap=256)
    cache.table[0, 3], cache.table[0, 9] = -1, cache.n_pages + 5
    cache.table[2, :2] = -1
    used = np.unique(np.concatenate([cache.rows(b, int(n)) for b, n in enumerate(cache.lens)]))
    rest = np.setdiff1d(np.arange(len(cache.k)), used)
    if group:
        cache.ks[rest], cache.vs[rest] = np.nan, np.inf
    else:
        cache.k[rest], cache.v[rest] = 0x7FC0, 0xFF80
    q, gate = queries(rng, 5, 4, 128)
    got = run_attn(gpu, cache, q, gate, 4, max_len=300, max_rows=2)
    check_attn(cache, got, q, gate, 4)
    assert (got[0][3] == 0).all() and (got[3][3, :20] == 0).all()
    # cut by max_len: the last rows' own keys lie behind it
    got = run_attn(gpu, cache, q, gate, 4, max_len=100, max_rows=2)
    ref, _, _, _ = attention(cache, bf2f(q).astype(np.float64), 4, 100)
    sg = sigmoid(bf2f(gate).astype(np.float64))
    assert np.linalg.norm(bf2f(got[0]) - ref * sg) <= 2.0 ** -8 * np.linalg.norm(ref * sg)


@pytest.mark.parametrize("max_len,times", [(200, 1), (24576, 1), (2048, 65)])
def test_attention_weights_behind_the_table(gpu, max_len, times):
    """The table ends inside a split, chunks before the sequence's length: the keys behind it have no weight, in both forms of
    the split kernel."""
    rng = np.random.default_rng(24)
    cache = Cache(rng, [200, 80, 60, 199] * times, [3, 1, 2, 3] * times, 2, 128, 32, page=16, cap=80)
    q, gate = queries(rng, 9 * times, 16, 128)
    got = run_attn(gpu, cache, q, gate, 16, max_len=max_len)
    check_attn(cache, got, q, gate, 16)
    assert (got[3][:3, 80:200] == 0).all()


@pytest.mark.parametrize("more", [0, 260])
@pytest.mark.parametrize("group", [0, 32])
@pytest.mark.parametrize("hd", [128, 256])
def test_attention_not_finite_stays_with_its_rows(gpu, group, hd, more):
    """A key that is not finite reaches the rows that see it and no other: the new rows before it are as they were. Alone, and
    among as many sequences as have a wave walk each split."""
    rng = np.random.default_rng(11)
    for bad in (np.nan, np.inf):
        cache = Cache(rng, [130, 70] + [3] * more, [5, 2] + [1] * more, 1, hd, group)
        q, gate = queries(rng, 7 + more, 4, hd)
        clean = run_attn(gpu, cache, q, gate, 4, max_len=2048)
        for b, key in ((0, 128), (1, 69)):             # row 3 of 5, row 1 of 2
            s = cache.slot(b, key)
            if group:
                cache.vs[s], cache.ks[s] = bad, bad
            else:
                cache.v[s], cache.k[s] = bf(np.full(hd, bad)), bf(np.full(hd, bad))
        got = run_attn(gpu, cache, q, gate, 4, max_len=2048)
        for r in (0, 1, 2, 5):
            a, b = bf2f(got[0][r]), bf2f(clean[0][r])
            assert (np.abs(a - b) <= 2.0 ** -7 * np.abs(b) + 2.0 ** -12).all()
            assert np.isfinite(got[3][r]).all()
        for r in (3, 4, 6):
            assert not np.isfinite(bf2f(got[0][r])).any()


@pytest.mark.parametrize("rows", [1, 4])
def test_attention_scores_of_minus_infinity(gpu, rows):
    """Keys whose score is -inf have no weight; a row that has no other gets zeros, in a chunk, a split and the whole."""
    rng = np.random.default_rng(35)
    lens = [300, 70, 600]
    cache = Cache(rng, lens, [rows] * 3, 1, 128, 0, page=16)
    q, gate = queries(rng, 3 * rows, 4, 128)
    q[..., 0] = bf(np.float32(1.0))
    low = [np.arange(300), np.arange(0, 70, 2), np.arange(0, 512)]
    for b, keys in enumerate(low):
        cache.k[cache.rows(b, lens[b])[keys], 0] = 0xFF80
    out, _, _, w = run_attn(gpu, cache, q, gate, 4)
    assert (bf2f(out[:rows]) == 0).all() and (w[:rows, :300] == 0).all()
    for b in (1, 2):
        slots = cache.rows(b, lens[b])
        K, V = cache.values(0, slots)[:, 0], cache.values(1, slots)[:, 0]
        for i in range(rows):
            r = b * rows + i
            see = np.setdiff1d(np.arange(lens[b] - rows + i + 1), low[b])
            total = np.zeros(lens[b])
            for h in range(4):
                x = K[see] @ bf2f(q[r, h]).astype(np.float64) / np.sqrt(128)
                p = np.exp(x - x.max())
                p /= p.sum()
                total[see] += p
                sg = sigmoid(bf2f(gate[r, h]).astype(np.float64))
                want, mag = p @ V[see] * sg, p @ np.abs(V[see]) * sg
                # (128 + 8 fp32 roundings of a score of at most 60 in all, twice; 2^-16 for the weights' two terms)
                rel = 4 * 136 * U * 60 + 2.0 ** -16
                assert (np.abs(bf2f(out[r, h]) - want) <= 2.0 ** -8 * np.abs(want) + rel * mag).all()
            assert (w[r, low[b]] == 0).all()
            assert (np.abs(w[r, :lens[b]] - total) <= (4 * 136 * U * 60 + 2.0 ** -16) * total).all()


def test_attention_value_scales_of_any_size(gpu):
    """Value scales far from 1, different by group: every group keeps its own precision."""
    rng = np.random.default_rng(12)
    cache = Cache(rng, [200], [1], 1, 256, 64)
    for i, f in enumerate((1e-30, 1.0, 1e25, 0.0)):
        cache.vs[:, i] *= np.float32(f)
    q, gate = queries(rng, 1, 4, 256)
    out = bf2f(run_attn(gpu, cache, q, gate, 4)[0])
    ref, mag, _, _ = attention(cache, bf2f(q).astype(np.float64), 4)
    sg = sigmoid(bf2f(gate).astype(np.float64))
    for i in range(3):
        part = slice(64 * i, 64 * i + 64)
        assert np.linalg.norm((out / 1 - ref * sg)[..., part].astype(np.float64)) <= 2.0 ** -8 * np.linalg.norm((mag * sg)[..., part])
    assert (out[..., 192:] == 0).all()


@pytest.mark.parametrize("group", [0, 32])
def test_attention_bits_do_not_depend_on_the_batch(gpu, group):
    """A row alone, the row among others, and the verify rows against single steps: the same bits."""
    rng = np.random.default_rng(13)
    nq, nkv, hd = 12, 2, 128
    cache = Cache(rng, [700, 90, 333], [3, 8, 1], nkv, hd, group)
    q, gate = queries(rng, 12, nq, hd)
    out, xq, xs, w = run_attn(gpu, cache, q, gate, nq)
    lens, counts, table, start = cache.lens, cache.counts, cache.table, cache.row_start
    for b in range(3):
        for i in range(counts[b]):
            r = start[b] + i
            cache.lens, cache.counts = np.array([lens[b] - counts[b] + i + 1], np.int32), np.array([1], np.int32)
            cache.row_start, cache.table = np.array([0, 1], np.int32), table[b:b + 1].copy()
            one = run_attn(gpu, cache, q[r:r + 1], gate[r:r + 1], nq)
            assert np.array_equal(one[0][0], out[r]), (b, i)
            assert np.array_equal(one[3][0, :cache.lens[0]], w[r, :cache.lens[0]]), (b, i)


# (lengths, rows, the row of each whose own key is the large one): inside a chunk, across one's end, at one's first key, the
# first key of a split, the last row, eight rows
LARGE = [([130, 66, 65, 257, 40, 300], [3, 3, 2, 2, 3, 8], [1, 2, 1, 1, 2, 4]),
         ([70, 129, 513, 20, 261, 8], [3, 2, 3, 5, 8, 8], [2, 1, 1, 3, 7, 2])]


@pytest.mark.parametrize("factor", [2.0 ** 10, 2.0 ** 16, 2.0 ** 24, 2.0 ** 32, np.inf, np.nan])
@pytest.mark.parametrize("more", [0, 260])
@pytest.mark.parametrize("geom,group", [("4x1x128", 16), ("4x1x128", 32), ("4x1x128", 64), ("4x1x128", 0), ("6x1x256", 16),
                                        ("6x1x256", 32), ("6x1x256", 64), ("6x1x256", 0)])
def test_attention_values_of_later_keys(gpu, geom, group, more, factor):
    """One of a call's rows has a value far above the others', or one that is not finite: every row has the bits of its single
    step, and the rows that do not see it stay within the bound that their own keys' values give. Alone, and among as many
    sequences as have a wave walk each split."""
    nq, nkv, hd = GEOMS[geom]
    for seed, (lens, counts, which) in enumerate(LARGE):
        rng = np.random.default_rng(300 + seed)
        few, n = len(lens), sum(counts)
        cache = Cache(rng, lens + [3] * more, counts + [1] * more, nkv, hd, group, page=16)
        part = slice(0, None if seed else 1)                        # (of the scales: one group, or all)
        for b in range(few):
            s = cache.slot(b, lens[b] - counts[b] + which[b])
            if group:
                cache.vs[s, part] *= np.float32(factor)
            else:
                with np.errstate(invalid="ignore"):
                    cache.v[s, ::1 if seed else 32] = bf(bf2f(cache.v[s, ::1 if seed else 32]) * np.float32(factor))
        q, gate = queries(rng, n + more, nq, hd)
        out, xq, xs, w = run_attn(gpu, cache, q, gate, nq, max_len=2048)
        table, start = cache.table, cache.row_start
        for b in range(few):
            for i in range(counts[b]):
                r, m = start[b] + i, lens[b] - counts[b] + i + 1
                cache.lens, cache.counts = np.array([m], np.int32), np.array([1], np.int32)
                cache.row_start, cache.table = np.array([0, 1], np.int32), table[b:b + 1].copy()
                one = run_attn(gpu, cache, q[r:r + 1], gate[r:r + 1], nq)
                alike = (one[0][0] == out[r]) | (np.isnan(bf2f(one[0][0])) & np.isnan(bf2f(out[r])))
                assert alike.all(), (b, i, int((~alike).sum()))
                assert np.array_equal(one[3][0, :m], w[r, :m]), (b, i)
                if i >= which[b] or m <= 0:
                    continue
                assert np.array_equal(one[1][0], xq[r]) and np.array_equal(one[2][0], xs[r])
                ref, mag, _, big = attention(cache, bf2f(q[r:r + 1]).astype(np.float64), nq)
                sg = sigmoid(bf2f(gate[r:r + 1]).astype(np.float64))
                d = 2 * (hd + 8) * U * big[0]
                rel = 2 * 2.0 ** -11 + 2 * d + (m + 64) * U + 2.0 ** -20
                own = cache.rows(b=0, n=m)                          # (below 2^-14: 2^-25 of the largest value that the row sees)
                small = 2.0 ** -24 * m * (np.abs(cache.vs[own]).max() * 127 if group else 0.0)
                tol = 2.0 ** -8 * np.abs(ref * sg) + sg * (rel * mag + small)
                assert (np.abs(bf2f(out[r:r + 1]) - ref * sg) <= tol).all(), (b, i)


@pytest.mark.parametrize("std", [1.5, 12.0])
@pytest.mark.parametrize("size", [2.0 ** -110, 2.0 ** -70, 2.0 ** 90])
@pytest.mark.parametrize("factor", [2.0 ** 7, 2.0 ** 11, 2.0 ** 13, 2.0 ** 14])
def test_attention_values_of_later_keys_near_the_limits(gpu, factor, size, std):
    """Ratios of scales around what one factor holds, with scales near the ends of what fp32 does, and weights down to none
    beside an earlier chunk's: the rows have the bits of their single steps."""
    rng = np.random.default_rng(310)
    nq, nkv, hd = 6, 1, 256
    lens, counts, which = LARGE[0]
    cache = Cache(rng, lens, counts, nkv, hd, 32, page=16)
    cache.vs *= np.float32(size)
    for b in range(len(lens)):
        cache.vs[cache.slot(b, lens[b] - counts[b] + which[b])] *= np.float32(factor)
    q, gate = queries(rng, sum(counts), nq, hd, std=std)
    out = run_attn(gpu, cache, q, gate, nq, max_len=2048)[0]
    table, start = cache.table, cache.row_start
    for b in range(len(lens)):
        for i in range(counts[b]):
            cache.lens, cache.counts = np.array([lens[b] - counts[b] + i + 1], np.int32), np.array([1], np.int32)
            cache.row_start, cache.table = np.array([0, 1], np.int32), table[b:b + 1].copy()
            r = start[b] + i
            assert np.array_equal(run_attn(gpu, cache, q[r:r + 1], gate[r:r + 1], nq)[0][0], out[r]), (b, i)


@pytest.mark.parametrize("geom,group", [("4x1x128", 32), ("6x1x256", 32), ("4x1x128", 0), ("6x1x256", 16)])
@pytest.mark.parametrize("rows", [1, 5])
def test_attention_bits_of_a_large_batch(gpu, geom, group, rows):
    """A batch of enough keys and rows for the other forms of the kernels: the bits of each sequence alone."""
    rng = np.random.default_rng(16)
    nq, nkv, hd = GEOMS[geom]
    n = 100
    lens = rng.integers(rows, 700, n)
    lens[:4] = [rows, 256, 257, 1500]
    cache = Cache(rng, lens, [rows] * n, nkv, hd, group, page=32)
    q, gate = queries(rng, n * rows, nq, hd)
    # max_len far above the lengths counts as much work: whole splits for a wave, a block per head in the join
    out, xq, xs, w = run_attn(gpu, cache, q, gate, nq, max_len=256 * (1800 * 8 // n + 1))
    table, start = cache.table, cache.row_start
    for b in (0, 1, 2, 3, 50, 99):
        cache.lens, cache.counts = lens[b:b + 1].astype(np.int32), np.array([rows], np.int32)
        cache.row_start, cache.table = np.array([0, rows], np.int32), table[b:b + 1].copy()
        r = slice(start[b], start[b] + rows)
        one = run_attn(gpu, cache, q[r], gate[r], nq)
        assert np.array_equal(one[0], out[r]) and np.array_equal(one[1], xq[r]) and np.array_equal(one[2], xs[r]), b
        assert np.array_equal(one[3][:, :lens[b]], w[r, :lens[b]]), b
        check_attn(cache, one, q[r], gate[r], nq)


@pytest.mark.parametrize("group", [0, 16, 32, 64])
@pytest.mark.parametrize("geom", list(GEOMS))
def test_attention_with_room_for_many_keys(gpu, group, geom):
    """The borders of tiles, chunks and splits under a max_len that stands for much work: waves that walk whole splits."""
    rng = np.random.default_rng(70 + group)
    nq, nkv, hd = GEOMS[geom]
    counts = [1] * len(LENS) if nq // nkv < 20 else [1, 2, 1, 3, 1, 1, 2, 1, 1]
    cache = Cache(rng, LENS, counts, nkv, hd, group, page=16)
    q, gate = queries(rng, sum(counts), nq, hd)
    got = run_attn(gpu, cache, q, gate, nq, max_len=256 * (1800 * 8 // (len(LENS) * nkv) + 1))
    check_attn(cache, got, q, gate, nq)


@pytest.mark.parametrize("group", [0, 16, 32, 64])
@pytest.mark.parametrize("geom", list(GEOMS))
def test_attention_many_sequences(gpu, group, geom):
    """More sequences than are counted ahead: a wave walks each split."""
    rng = np.random.default_rng(80 + group)
    nq, nkv, hd = GEOMS[geom]
    n = 260
    lens = rng.integers(0, 300, n)
    lens[:len(LENS)] = LENS
    counts = rng.integers(0, 3, n) if nq // nkv < 20 else np.ones(n, np.int64)
    cache = Cache(rng, lens, counts, nkv, hd, group, page=32)
    q, gate = queries(rng, int(sum(counts)), nq, hd)
    check_attn(cache, run_attn(gpu, cache, q, gate, nq, max_len=2048), q, gate, nq)


@pytest.mark.parametrize("geom,group,rows,n,max_len", [("32x8x128", 32, 1, 130, None), ("32x8x128", 0, 1, 130, None),
                                                       ("32x8x128", 16, 5, 130, None), ("24x4x256", 0, 1, 130, None),
                                                       ("24x4x256", 32, 3, 130, None), ("24x4x256", 16, 1, 130, None),
                                                       ("32x8x128", 32, 1, 70, 1024), ("32x8x128", 0, 2, 90, 1024),
                                                       ("24x4x256", 64, 1, 150, 1024)])
def test_attention_rounds_and_their_rest(gpu, geom, group, rows, n, max_len):
    """A few units more than the waves take at once, the rest by whole blocks, or by blocks and some waves: within the tolerances,
    and the bits of a sequence alone, the first, some in between and the last."""
    rng = np.random.default_rng(90 + group + rows)
    nq, nkv, hd = GEOMS[geom]
    lens = rng.integers(257, 320, n)
    cache = Cache(rng, lens, [rows] * n, nkv, hd, group, page=32)
    q, gate = queries(rng, n * rows, nq, hd)
    got = run_attn(gpu, cache, q, gate, nq, max_len=max_len)
    check_attn(cache, got, q, gate, nq)
    table, start = cache.table, cache.row_start
    for b in (0, 3, 7, n // 2, n - 3, n - 2, n - 1):
        cache.lens, cache.counts = lens[b:b + 1].astype(np.int32), np.array([rows], np.int32)
        cache.row_start, cache.table = np.array([0, rows], np.int32), table[b:b + 1].copy()
        r = slice(start[b], start[b] + rows)
        one = run_attn(gpu, cache, q[r], gate[r], nq)
        assert np.array_equal(one[0], got[0][r]) and np.array_equal(one[1], got[1][r]) and np.array_equal(one[2], got[2][r]), b
        assert np.array_equal(one[3][:, :lens[b]], got[3][r, :lens[b]]), b


def test_attention_many_heads(gpu):
    """More query heads than the weights' kernel takes at a time, and five column tiles of a kv head."""
    rng = np.random.default_rng(25)
    cache = Cache(rng, [300, 70], [2, 1], 2, 128, 32)
    q, gate = queries(rng, 3, 160, 128)
    check_attn(cache, run_attn(gpu, cache, q, gate, 160), q, gate, 160)


def test_attention_shared_pages(gpu):
    """Sequences that begin on the same pages, and one whose pages repeat: what each reads alone."""
    rng = np.random.default_rng(26)
    cache = Cache(rng, [150, 131, 90], [1, 2, 1], 2, 128, 32, page=16)
    cache.table[1, :8] = cache.table[0, :8]
    cache.table[2, :6] = cache.table[2, 0]
    q, gate = queries(rng, 4, 8, 128)
    check_attn(cache, run_attn(gpu, cache, q, gate, 8), q, gate, 8)


@pytest.mark.parametrize("hd", [128, 256])
def test_arguments_of_their_types_alignment(gpu, hd):
    """Only the pages and the scratch memory are aligned to more than their type: everything else two bytes, or a float, on."""
    X, rng = gpu, np.random.default_rng(27)
    nq, nkv = 8, 2
    cache = Cache(rng, [70, 9], [1, 2], nkv, hd, 32)
    cache.push(X)
    q, gate = queries(rng, 3, nq, hd)
    want = run_attn(X, cache, q, gate, nq)
    held = []

    def shifted(a):
        n = a.dtype.itemsize
        b = X.DevBuf(array=np.concatenate([np.zeros(1, a.dtype), a.reshape(-1), np.zeros(1, a.dtype)]))
        held.append(b)
        return b.ptr + n

    kv = cache.push(X)
    kv.ks, kv.vs = shifted(cache.ks), shifted(cache.vs)
    width = nq * 2 * hd + 2 * nkv * hd + 1
    g = np.zeros((3, width), np.uint16)
    g[:, :nq * 2 * hd].reshape(3, nq, 2, hd)[:, :, 1] = gate
    out = X.DevBuf(array=np.zeros(3 * nq * hd + 1, np.uint16))
    xq, xs = X.DevBuf(array=np.zeros(3 * nq * hd + 1, np.int8)), X.DevBuf(array=np.zeros(3 * nq * hd // 16 + 1, np.float32))
    w = X.DevBuf(array=np.zeros(3 * 71 + 1, np.float32))
    work = X.DevBuf(X.lib().q27x_paged_attn_work_bytes(nq, hd, 70, 3, 1))
    X.call("q27x_paged_attn_rows", shifted(q), shifted(g), width, ctypes.byref(kv), nq, 1, 70, 2, 3, work.ptr, out.ptr + 2, xq.ptr + 1,
           xs.ptr + 4, w.ptr + 4, 71, None)
    X.call("q27x_device_sync")
    assert np.array_equal(out.download(np.uint16, (3 * nq * hd + 1,))[1:], want[0].reshape(-1))
    assert np.array_equal(xq.download(np.int8, (3 * nq * hd + 1,))[1:], want[1].reshape(-1))
    assert np.array_equal(xs.download(np.float32, (3 * nq * hd // 16 + 1,))[1:], want[2].reshape(-1))
    got = w.download(np.float32, (3 * 71 + 1,))[1:].reshape(3, 71)
    for r, n in enumerate((70, 9, 9)):
        assert np.array_equal(got[r, :n], want[3][r, :n])


def test_attention_like_the_contiguous_entry(gpu):
    """q27x_attn_rows over the same cache, its pages counting up: both within their roundings of the float64 form."""
    X, rng = gpu, np.random.default_rng(14)
    nq, nkv, hd, n, pos0 = 32, 8, 128, 3, 500
    cache = Cache(rng, [pos0 + n], [n], nkv, hd, 32, page=8, spare=0)
    cache.table[0] = np.arange(cache.n_pages)
    q, gate = queries(rng, n, nq, hd)
    out = run_attn(X, cache, q, gate, nq)[0]
    width = nq * 2 * hd + 2 * nkv * hd
    g = np.zeros((n, width), np.uint16)
    g[:, :nq * 2 * hd].reshape(n, nq, 2, hd)[:, :, 1] = gate
    dq, dg, o2 = X.DevBuf(array=q), X.DevBuf(array=g), X.DevBuf(n * nq * hd * 2)
    work = X.DevBuf(X.lib().q27x_attn_work_bytes(nq, hd, pos0 + n, n))
    X.call("q27x_attn_rows", dq.ptr, dg.ptr, width, cache.d["k"].ptr, cache.d["ks"].ptr, cache.d["v"].ptr, cache.d["vs"].ptr, 32, nq,
           nkv, hd, 1, pos0, n, work.ptr, o2.ptr, None, None, None)
    X.call("q27x_device_sync")
    a, b = bf2f(out), bf2f(o2.download(np.uint16, (n, nq, hd)))
    _, mag, _, _ = attention(cache, bf2f(q).astype(np.float64), nq)
    assert (np.abs(a - b) <= 2 * 2.0 ** -8 * np.abs(b) + 2.0 ** -9 * mag).all()


def test_attention_positions_past_32_bits(gpu):
    """Pages whose bytes lie past 4 GiB of the pool."""
    X, rng = gpu, np.random.default_rng(15)
    nq, nkv, hd, page = 8, 8, 256, 16
    cache = Cache(rng, [100], [1], nkv, hd, 32, page=page, spare=0)
    n_pages = (9 << 29) // (nkv * hd * page)                       # 4.5 GiB of codes
    far = {}
    cache.push(X)
    for name, width, size in (("k", nkv * hd, 1), ("v", nkv * hd, 1), ("ks", nkv * hd // 32, 4), ("vs", nkv * hd // 32, 4)):
        far[name] = X.DevBuf(n_pages * page * width * size)
        src = getattr(cache, name)
        for j, p in enumerate(cache.table[0]):
            rows = np.ascontiguousarray(src[p * page:(p + 1) * page])
            X.call("q27x_memcpy_h2d", far[name].ptr + (n_pages - 1 - j) * page * width * size, rows.ctypes.data, rows.nbytes, None)
    table = (n_pages - 1 - np.arange(cache.table.shape[1], dtype=np.int32))[None]
    dt = X.DevBuf(array=np.ascontiguousarray(table))
    kv = X.PagedKV(k=far["k"].ptr, v=far["v"].ptr, ks=far["ks"].ptr, vs=far["vs"].ptr, kv_group=32, nkv=nkv, hd=hd, n_pages=n_pages,
                   page=page, page_stride=0, table=dt.ptr, table_stride=table.shape[1], lens=cache.d["lens"].ptr, row_start=None, n_seq=1)
    q, _ = queries(rng, 1, nq, hd)
    dq, out = X.DevBuf(array=q), X.DevBuf(nq * hd * 2)
    work = X.DevBuf(X.lib().q27x_paged_attn_work_bytes(nq, hd, 100, 1, 0))
    X.call("q27x_paged_attn_rows", dq.ptr, None, 0, ctypes.byref(kv), nq, 0, 100, 1, 1, work.ptr, out.ptr, None, None, None, 0, None)
    X.call("q27x_device_sync")
    ref, mag, _, _ = attention(cache, bf2f(q).astype(np.float64), nq)
    assert (np.abs(bf2f(out.download(np.uint16, (1, nq, hd))) - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -9 * mag).all()
    for b in far.values():
        b.free()


# ---------------------------------------------------------------- eviction
class Evictor:
    """Device state of one layer's eviction and its host twin."""

    def __init__(self, X, cache, stride, rng=None):
        self.X, self.cache, self.stride = X, cache, stride
        n = len(cache.lens)
        self.acc = np.full((n, stride), 9e9, np.float32)
        self.ord = np.full((n, stride), -5, np.int32)
        self.state = np.zeros((n, 2), np.int32)
        self.dev = [X.DevBuf(array=a) for a in (self.acc, self.ord, self.state)]
        self.new = X.DevBuf(array=np.full(n, -9, np.int32))

    def call(self, w, w_stride, n_acc, nrows, decay, high, budget, recent, max_len, new=None):
        X, n = self.X, len(self.cache.lens)
        work = X.DevBuf(array=np.full(X.lib().q27x_paged_evict_work_bytes(n, max_len), 0xA5, np.uint8))
        X.call("q27x_paged_evict", ctypes.byref(self.cache.kv), w, w_stride, n_acc, nrows, decay, self.dev[0].ptr, self.dev[1].ptr,
               self.stride, self.dev[2].ptr, high, budget, recent, max_len, work.ptr, new or self.new.ptr, None)
        X.call("q27x_device_sync")

    def expect(self, lens, rows, decay, high, budget, recent):
        """The host twin: rows[b] the accepted weight rows. Moves the host cache's rows; returns the new lengths."""
        got = []
        for b, n in enumerate(lens):
            m, moves = evict(self.acc[b], self.ord[b], self.state[b], int(n), rows[b], decay, high, budget, recent)
            for src, dst in moves:
                s, d = self.cache.slot(b, src), self.cache.slot(b, dst)
                if s >= 0 and d >= 0:
                    for name in ("k", "v", "ks", "vs"):
                        a = getattr(self.cache, name)
                        if a is not None:
                            a[d] = a[s]
            got.append(m)
        return got

    def compare(self, want, new=None):
        n = len(want)
        assert np.array_equal((new or self.new).download(np.int32, (n,)), want)
        a, o, s = (d.download(x.dtype, x.shape) for d, x in zip(self.dev, (self.acc, self.ord, self.state)))
        assert np.array_equal(s, self.state)
        assert np.array_equal(a.view(np.uint32), self.acc.view(np.uint32)), "sums differ"
        assert np.array_equal(o, self.ord)
        for name, x in self.cache.pull().items():
            assert np.array_equal(x.view(np.uint8), getattr(self.cache, name).view(np.uint8)), name


@pytest.mark.parametrize("group", [0, 16, 32, 64])
@pytest.mark.parametrize("hd", [128, 256])
@pytest.mark.parametrize("recent,decay", [(0, 1.0), (7, 0.9), (40, 0.5)])
def test_evict(gpu, group, hd, recent, decay):
    """Ragged lengths around the limits, several rows of which some are accepted, equal sums, several calls in a row."""
    X, rng = gpu, np.random.default_rng(group + recent)
    counts = [1, 3, 2, 0, 8, 1, 1]
    lens = [41, 400, 64, 70, 1500, 0, 40]
    cache = Cache(rng, lens, counts, 1, hd, group, page=8)
    cache.push(X)
    ev = Evictor(X, cache, 1510)
    n = sum(counts)
    for call in range(3):
        w = (rng.integers(0, 12, (n, 1503)) / 8).astype(np.float32) if call < 2 else rng.random((n, 1503)).astype(np.float32)
        n_acc = np.array([rng.integers(0, c + 1) for c in counts], np.int32)
        n_acc[1] = 99                                              # (more than there are: all)
        now = [min(x, 40 + 3 * b) if call else x for b, x in enumerate(lens)]    # later calls: a few keys more than the budget
        cache.lens = np.asarray(now, np.int32)
        cache.d["lens"].upload(cache.lens)
        dw, da = X.DevBuf(array=w), X.DevBuf(array=n_acc)
        ev.call(dw.ptr, 1503, da.ptr, n, decay, 40, 40, recent, 1503)
        rows = [w[cache.row_start[b]:cache.row_start[b] + min(counts[b], n_acc[b])] for b in range(len(lens))]
        ev.compare(ev.expect(now, rows, decay, 40, 40, recent))


def test_evict_more_than_a_block(gpu):
    """A long sequence beside short ones, cut to a third, with a limit above the budget."""
    X, rng = gpu, np.random.default_rng(21)
    cache = Cache(rng, [9001, 3, 4096, 3500], [1, 1, 1, 1], 1, 128, 32, page=64)
    cache.push(X)
    ev = Evictor(X, cache, 9001)
    w = np.round(rng.random((4, 9001)) ** 6 * 4096).astype(np.float32) / 1024
    dw = X.DevBuf(array=w)
    ev.call(dw.ptr, 9001, None, 4, 1.0, 3999, 3001, 500, 9001)
    ev.compare(ev.expect([9001, 3, 4096, 3500], [w[b:b + 1] for b in range(4)], 1.0, 3999, 3001, 500))


@pytest.mark.parametrize("len_", [1024, 1025, 32768, 40001])
def test_evict_lengths_of_the_kernels(gpu, len_):
    """The ends of what a block holds in registers, and past it; sums that are all equal, and spread over many exponents; a
    budget of one key less, whose move needs no launch of its own, and of few."""
    X, rng = gpu, np.random.default_rng(len_)
    for budget, spread in ((len_ - 1, 0), (len_ - 1, 1), (len_ - 8, 0), (len_ - 8, 2), (len_ - 9, 0), (len_ - 20, 1), (17, 2)):
        cache = Cache(rng, [len_, 20], [1, 1], 1, 128, 64, page=16)
        cache.push(X)
        ev = Evictor(X, cache, len_)
        w = np.ones((2, len_), np.float32) if spread == 0 else rng.random((2, len_)).astype(np.float32) ** (1 if spread == 1 else 40)
        dw = X.DevBuf(array=w)
        ev.call(dw.ptr, len_, None, 2, 1.0, budget, budget, 5, len_)
        ev.compare(ev.expect([len_, 20], [w[:1], w[1:]], 1.0, budget, budget, 5))


@pytest.mark.parametrize("max_len", [32769, 90000])
def test_evict_long_sequences(gpu, max_len):
    """Lengths past what a block holds beside short ones, ends of its tiles, many equal sums, two accepted rows of three, one
    sequence between budget and limit; then calls that bring a few keys."""
    X, rng = gpu, np.random.default_rng(max_len)
    lens, counts = [max_len, 24577, 16384, 0, 16385, max_len - 1], [1, 3, 1, 1, 2, 0]
    cache = Cache(rng, lens, counts, 1, 128, 64, page=64)
    cache.push(X)
    ev = Evictor(X, cache, max_len + 3)
    n, n_acc = sum(counts), np.array([1, 2, 1, 1, 0, 1], np.int32)
    da = X.DevBuf(array=n_acc)
    for call, (high, budget, recent) in enumerate([(20000, 12301, 1000), (12301, 12301, 1000), (16384, 9000, 0)]):
        w = (rng.integers(0, 40, (n, max_len)) ** 3 / 8).astype(np.float32)
        now = [min(x, 12301 + 5 * b) if call else x for b, x in enumerate(lens)]
        cache.lens = np.asarray(now, np.int32)
        cache.d["lens"].upload(cache.lens)
        dw = X.DevBuf(array=w)
        ev.call(dw.ptr, max_len, da.ptr, n, 0.75, high, budget, recent, max_len)
        rows = [w[cache.row_start[b]:cache.row_start[b] + min(counts[b], n_acc[b])] for b in range(len(lens))]
        ev.compare(ev.expect(now, rows, 0.75, high, budget, recent))


def test_evict_sums_that_are_not_numbers(gpu):
    """NaN goes first, infinity stays, -0 and 0 are equal, negative sums are ordered; no weights at all leaves the sums."""
    X, rng = gpu, np.random.default_rng(22)
    cache = Cache(rng, [200], [1], 1, 128, 32)
    cache.push(X)
    ev = Evictor(X, cache, 256)
    w = rng.choice(np.array([np.nan, np.inf, -np.inf, 0.0, -0.0, 1.0, -1.0, 1e-40, -1e-40, 3e38], np.float32), (1, 200))
    dw = X.DevBuf(array=w)
    ev.call(dw.ptr, 200, None, 1, 1.0, 200, 200, 0, 200)
    with np.errstate(invalid="ignore"):
        ev.compare(ev.expect([200], [w], 1.0, 200, 200, 0))
        for budget in (170, 90, 33, 1):
            ev.call(None, 0, None, 1, 1.0, budget, budget, 0, 200)
            ev.compare(ev.expect([int(cache.lens[0])], [w[:0]], 1.0, budget, budget, 0))
            cache.lens[:] = budget
            cache.d["lens"].upload(cache.lens)


def test_evict_after_a_rollback_and_lens_in_place(gpu):
    """A shorter length than the sums know (rows were rejected), then longer again; new_lens is the cache's own lens."""
    X, rng = gpu, np.random.default_rng(23)
    cache = Cache(rng, [60, 90], [1, 1], 1, 128, 32, page=16, cap=128)
    cache.push(X)
    ev = Evictor(X, cache, 128)
    for lens in ([60, 90], [55, 30], [70, 100], [64, 64]):
        w = rng.random((2, 128)).astype(np.float32)
        cache.d["lens"].upload(np.asarray(lens, np.int32))
        dw = X.DevBuf(array=w)
        ev.call(dw.ptr, 128, None, 2, 0.75, 64, 50, 9, 128, new=cache.d["lens"].ptr)
        ev.compare(ev.expect(lens, [w[:1], w[1:]], 0.75, 64, 50, 9), new=cache.d["lens"])


@pytest.mark.parametrize("known,left,budget,recent", [(60, 52, 40, 9), (60, 52, 48, 9), (60, 59, 58, 58), (1500, 1490, 20, 20),
                                                      (40000, 39000, 30000, 5000), (40000, 39999, 39998, 7)])
def test_evict_cut_after_a_rollback(gpu, known, left, budget, recent):
    """Keys are taken back, then the cache is cut: of those that are left the newest stay, though the sums want them least, and
    the keys that come next are numbered behind them."""
    X, rng = gpu, np.random.default_rng(known + budget)
    cache = Cache(rng, [known, 7], [1, 1], 1, 128, 64, page=64)
    cache.push(X)
    ev = Evictor(X, cache, known)
    w = (rng.integers(1, 9, (2, known)) / 8).astype(np.float32)
    w[0, left - recent - known // 8:] = 0
    dw = X.DevBuf(array=w)
    ev.call(dw.ptr, known, None, 2, 1.0, known, known, recent, known)
    cache.d["lens"].upload(np.array([left, 7], np.int32))
    ev.call(dw.ptr, known, None, 2, 1.0, budget, budget, recent, known)
    # no cut before: key i is the i-th that came, and the sums are twice the weights
    old = sorted(range(left - recent), key=lambda i: (-w[0, i], i))[:budget - recent]
    stays = np.zeros(left, bool)
    stays[old], stays[left - recent:] = True, True
    want = np.arange(left)
    want[np.flatnonzero(~stays[:budget])] = np.flatnonzero(stays[budget:]) + budget
    got = ev.dev[1].download(np.int32, (2, known))[0, :budget]
    assert np.array_equal(got, want[:budget])
    assert np.array_equal(ev.dev[0].download(np.float32, (2, known))[0, :budget], 2 * w[0, want[:budget]])
    k, first = cache.pull()["k"], cache.rows(0, left)
    assert np.array_equal(k[first[:budget]], cache.k[first[want[:budget]]])
    assert ev.new.download(np.int32, (2,)).tolist() == [budget, 7]
    cache.d["lens"].upload(np.array([budget + 1, 7], np.int32))
    ev.call(None, 0, None, 2, 1.0, budget + 1, budget, recent, known)
    assert ev.dev[1].download(np.int32, (2, known))[0, budget] == left
    assert ev.dev[2].download(np.int32, (2, 2)).tolist() == [[budget + 1, left + 1], [7, 7]]


def test_evict_pages_that_are_not_there(gpu):
    """Keys on missing pages are summed and ordered like the others; their rows are not copied. A table that ends early cuts
    the sequence."""
    X, rng = gpu, np.random.default_rng(24)
    cache = Cache(rng, [100, 200], [1, 1], 2, 128, 32, page=16, cap=128)
    cache.table[0, 1], cache.table[0, 5] = -1, cache.n_pages
    cache.push(X)
    ev = Evictor(X, cache, 256)
    w = rng.random((2, 256)).astype(np.float32)
    dw = X.DevBuf(array=w)
    ev.call(dw.ptr, 256, None, 2, 1.0, 50, 50, 5, 256)
    ev.compare(ev.expect([100, 128], [w[:1], w[1:]], 1.0, 50, 50, 5))


def test_writes_past_32_bits(gpu):
    """Prep and eviction on pages whose bytes lie past 4 GiB of the pool: what they do on near ones."""
    X, rng = gpu, np.random.default_rng(28)
    nq, nkv, hd, page, n, rot = 8, 8, 256, 16, 5, 64
    cache = Cache(rng, [100], [n], nkv, hd, 32, page=page, spare=0)
    n_pages = (9 << 29) // (nkv * hd * page)                       # 4.5 GiB of codes
    width = nq * hd + 2 * nkv * hd
    x, qn, kn = bf(rng.standard_normal((n, width)) * 2), bf(rng.standard_normal(hd) * 0.2), bf(rng.standard_normal(hd) * 0.2)
    cos, sin = tables(64, rot)
    w = rng.random((n, 100)).astype(np.float32)
    near = cache.push(X)
    parts = (("k", nkv * hd), ("v", nkv * hd), ("ks", nkv * hd // 32 * 4), ("vs", nkv * hd // 32 * 4))
    far = {name: X.DevBuf(n_pages * page * size) for name, size in parts}
    table = (n_pages - 1 - np.arange(cache.table.shape[1], dtype=np.int32))[None]
    for name, size in parts:
        for j, p in enumerate(cache.table[0]):
            rows = np.ascontiguousarray(getattr(cache, name)[p * page:(p + 1) * page])
            X.call("q27x_memcpy_h2d", far[name].ptr + int(table[0, j]) * page * size, rows.ctypes.data, rows.nbytes, None)
    dt = X.DevBuf(array=np.ascontiguousarray(table))
    away = X.PagedKV(k=far["k"].ptr, v=far["v"].ptr, ks=far["ks"].ptr, vs=far["vs"].ptr, kv_group=32, nkv=nkv, hd=hd, n_pages=n_pages,
                     page=page, page_stride=0, table=dt.ptr, table_stride=table.shape[1], lens=cache.d["lens"].ptr,
                     row_start=cache.d["row_start"].ptr, n_seq=1)
    dev = [X.DevBuf(array=a) for a in (x, qn, kn, cos, sin, np.arange(n, dtype=np.int32), w)]
    work = X.DevBuf(X.lib().q27x_paged_evict_work_bytes(1, 100))
    seen = []
    for kv in (near, away):
        qh, new = X.DevBuf(n * nq * hd * 2), X.DevBuf(4)
        acc, order, state = X.DevBuf(400), X.DevBuf(400), X.DevBuf(array=np.zeros(2, np.int32))
        X.call("q27x_paged_prep_rows", dev[0].ptr, width, dev[1].ptr, dev[2].ptr, dev[3].ptr, dev[4].ptr, rot, 64, dev[5].ptr, n, 1, None,
               ctypes.byref(kv), qh.ptr, nq, 0, 1e-6, n, None)
        X.call("q27x_paged_evict", ctypes.byref(kv), dev[6].ptr, 100, None, n, 1.0, acc.ptr, order.ptr, 100, state.ptr, 60, 50, 10, 100,
               work.ptr, new.ptr, None)
        X.call("q27x_device_sync")
        seen.append([b.download(np.uint8, (b.nbytes,)) for b in (qh, new, acc, order, state)])
    assert all(np.array_equal(a, b) for a, b in zip(*seen))
    got = cache.pull()
    for name, size in parts:
        assert not np.array_equal(got[name], getattr(cache, name))
        for j, p in enumerate(cache.table[0]):
            want = got[name][p * page:(p + 1) * page]
            back = np.empty_like(want)
            X.call("q27x_memcpy_d2h", back.ctypes.data, far[name].ptr + int(table[0, j]) * page * size, back.nbytes, None)
            assert np.array_equal(back.view(np.uint8), np.ascontiguousarray(want).view(np.uint8)), (name, j)
    for b in far.values():
        b.free()


# ---------------------------------------------------------------- together
def test_serving_steps(gpu):
    """Steps of a bounded batch as a server runs them: rows prepared into the pages, attention with weights, some verify
    rows rejected, eviction. Every step's attention against the float64 form over the pages as they are."""
    X, rng = gpu, np.random.default_rng(31)
    nq, nkv, hd, rot, cap = 8, 2, 128, 32, 96
    lens = np.array([70, 5, 33], np.int32)
    cache = Cache(rng, lens, [1, 1, 1], nkv, hd, 32, page=16, cap=cap)
    cache.push(X)
    ev = Evictor(X, cache, cap)
    start = np.zeros((3, cap), np.float32)
    d0 = X.DevBuf(array=start)
    ev.call(d0.ptr, cap, None, 3, 1.0, 64, 64, 8, cap)
    lens = np.array(ev.expect(lens, [start[b:b + 1] for b in range(3)], 1.0, 64, 64, 8), np.int32)
    ev.compare(lens)
    for step in range(8):
        counts = rng.integers(1, 5, 3).astype(np.int32)
        cache.counts, cache.lens = counts, lens + counts
        cache.row_start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        q, got, ref = run_prep(X, cache, rng, (nq, nkv, hd), rot, 3, [i % 3 for i in range(16)], True)
        check_prep(cache, q, got, ref, rot)
        for name, a in got.items():
            setattr(cache, name, a)
        gate = bf(rng.standard_normal(q.shape))
        res = run_attn(X, cache, q, gate, nq)
        check_attn(cache, res, q, gate, nq)
        taken = np.array([rng.integers(1, c + 1) for c in counts], np.int32)
        lens = lens + taken
        cache.lens = lens.astype(np.int32)
        kv = cache.push(X)
        w = res[3]
        full = np.zeros((len(w), cap), np.float32)
        full[:, :w.shape[1]] = w[:, :cap]
        dw, da = X.DevBuf(array=full), X.DevBuf(array=taken)
        ev.call(dw.ptr, cap, da.ptr, len(w), 1.0, 64, 60, 8, cap)
        rows = [full[cache.row_start[b]:cache.row_start[b] + taken[b]] for b in range(3)]
        lens = np.array(ev.expect(lens, rows, 1.0, 64, 60, 8), np.int32)
        ev.compare(lens)
        assert kv.n_seq == 3 and lens.max() <= 64


def test_layers_of_a_step_with_rejected_rows(gpu):
    """Two layers' caches on one table and one lens, verify rows of which some are rejected, a cut in most steps: the rejected
    rows are out of lens before a layer's eviction, and the last layer's writes it. No cache keeps a rejected key."""
    X, rng = gpu, np.random.default_rng(32)
    nq, nkv, hd, rot, cap = 8, 2, 128, 32, 96
    lens = np.array([58, 5, 33], np.int32)
    layers = [Cache(rng, lens, [1, 1, 1], nkv, hd, 32, page=16, cap=cap) for _ in range(2)]
    layers[1].table = layers[0].table
    evs = []
    for cache in layers:
        cache.push(X)
        evs.append(Evictor(X, cache, cap))
    gone, cuts = [[], []], 0
    for step in range(8):
        counts = rng.integers(1, 6, 3).astype(np.int32)
        taken = np.array([rng.integers(1, c + 1) for c in counts], np.int32)
        start = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        kept, new = X.DevBuf(array=lens + taken), None
        for i, (cache, ev) in enumerate(zip(layers, evs)):
            cache.counts, cache.lens, cache.row_start = counts, lens + counts, start
            q, got, ref = run_prep(X, cache, rng, (nq, nkv, hd), rot, 3, [j % 3 for j in range(16)], True)
            for name, a in got.items():
                setattr(cache, name, a)
            gate = bf(rng.standard_normal(q.shape))
            res = run_attn(X, cache, q, gate, nq)
            check_attn(cache, res, q, gate, nq)
            gone[i] += [cache.k[cache.slot(b, p)].copy() for b in range(3) for p in range(lens[b] + taken[b], lens[b] + counts[b])]
            full = np.zeros((len(res[3]), cap), np.float32)
            full[:, :res[3].shape[1]] = res[3][:, :cap]
            cache.push(X).lens = kept.ptr
            dw, da = X.DevBuf(array=full), X.DevBuf(array=taken)
            ev.call(dw.ptr, cap, da.ptr, len(full), 1.0, 60, 56, 8, cap, new=kept.ptr if i == 1 else None)
            rows = [full[start[b]:start[b] + taken[b]] for b in range(3)]
            new = np.array(ev.expect(lens + taken, rows, 1.0, 60, 56, 8), np.int32)
            ev.compare(new, new=kept if i == 1 else None)
        cuts += int((new < lens + taken).sum())
        lens = new
        for cache, bad in zip(layers, gone):
            held = np.concatenate([cache.k[cache.rows(b, lens[b])] for b in range(3)])
            assert not any((held == x).all(1).any() for x in bad)
    assert cuts >= 3


def test_prompts_in_steps_of_a_few_rows(gpu):
    """Two prompts behind what is there, prepared by one call: their attention sequence by sequence, eight rows at a time, and
    both together with the rows of a step side by side, has the same bits, within the bounds."""
    X, rng = gpu, np.random.default_rng(34)
    nq, nkv, hd, rot = 8, 2, 128, 32
    past, rows = [10, 0], [37, 21]
    cache = Cache(rng, [a + b for a, b in zip(past, rows)], rows, nkv, hd, 32, page=16)
    q, got, ref = run_prep(X, cache, rng, (nq, nkv, hd), rot, 3, [i % 3 for i in range(16)], True)
    check_prep(cache, q, got, ref, rot)
    for name, a in got.items():
        setattr(cache, name, a)
    gate = bf(rng.standard_normal(q.shape))
    table, start = cache.table, [0, rows[0]]

    def attend(seqs, at):
        """Rows at .. at + 7 of the sequences' prompts, those there are."""
        cache.counts = np.array([min(max(rows[b] - at, 0), 8) for b in seqs], np.int32)
        cache.lens = np.array([past[b] + min(rows[b], at + 8) for b in seqs], np.int32)
        cache.row_start = np.concatenate([[0], np.cumsum(cache.counts)]).astype(np.int32)
        cache.table = np.ascontiguousarray(table[seqs])
        pick = np.concatenate([np.arange(start[b] + at, start[b] + at + n) for b, n in zip(seqs, cache.counts)]).astype(np.int64)
        res = run_attn(X, cache, np.ascontiguousarray(q[pick]), np.ascontiguousarray(gate[pick]), nq, max_rows=8)
        check_attn(cache, res, q[pick], gate[pick], nq)
        return pick, res[0]

    alone, both = np.zeros_like(q), np.zeros_like(q)
    for b in (0, 1):
        for at in range(0, rows[b], 8):
            pick, out = attend([b], at)
            alone[pick] = out
    for at in range(0, max(rows), 8):
        pick, out = attend([0, 1], at)
        both[pick] = out
    assert np.array_equal(alone, both)


class _Graph:
    """A captured sequence of calls (HIP's graph functions, from the runtime that the library runs on)."""

    def __init__(self, X, calls):
        self.hip = ctypes.CDLL("libamdhip64.so")
        self.X, self.stream = X, ctypes.c_void_p()
        X.call("q27x_stream_create", ctypes.byref(self.stream))
        graph, self.exec = ctypes.c_void_p(), ctypes.c_void_p()
        self._ok(self.hip.hipStreamBeginCapture(self.stream, 0))
        calls(self.stream)
        self._ok(self.hip.hipStreamEndCapture(self.stream, ctypes.byref(graph)))
        self._ok(self.hip.hipGraphInstantiate(ctypes.byref(self.exec), graph, None, None, ctypes.c_size_t(0)))
        self._ok(self.hip.hipGraphDestroy(graph))

    def _ok(self, rc):
        assert rc == 0, f"HIP error {rc}"

    def replay(self):
        self._ok(self.hip.hipGraphLaunch(self.exec, self.stream))
        self.X.call("q27x_stream_sync", self.stream)

    def close(self):
        self._ok(self.hip.hipGraphExecDestroy(self.exec))
        self.X.call("q27x_stream_destroy", self.stream)


def test_streams_and_graphs(gpu):
    """A captured step (prepare, attend with weights, evict in place) replayed with eager work between, and the same calls
    on two streams with a workspace each, against the eager results of every step."""
    X = gpu
    nq, nkv, hd, rot, cap, page, steps = 8, 2, 128, 32, 640, 16, 9
    L, first = X.lib(), [601, 599, 300, 1, 17]
    seqs = len(first)
    width = 2 * nq * hd + 2 * nkv * hd
    cos, sin = tables(64, rot)

    class State:
        def __init__(self):
            rng = np.random.default_rng(33)
            self.cache = Cache(rng, first, [1] * seqs, nkv, hd, 32, page=page, cap=cap)
            self.kv = self.cache.push(X, row_start=False)
            x = {"qkv": bf(rng.standard_normal((seqs, width))), "norm": bf(rng.standard_normal(hd) * 0.1), "cos": cos, "sin": sin,
                 "pos": np.full((1, seqs), 30, np.int32), "qh": np.zeros((seqs, nq * hd), np.uint16),
                 "out": np.zeros((seqs, nq * hd), np.uint16), "w": np.zeros((seqs, cap), np.float32),
                 "acc": np.zeros((seqs, cap), np.float32), "ord": np.zeros((seqs, cap), np.int32), "state": np.zeros((seqs, 2), np.int32)}
            self.host = x
            self.d = {n: X.DevBuf(array=a) for n, a in x.items()}
            self.wa = X.DevBuf(L.q27x_paged_attn_work_bytes(nq, hd, cap, seqs, 1))
            self.we = X.DevBuf(L.q27x_paged_evict_work_bytes(seqs, cap))
            self.lens = np.array(first, np.int32)

        def grow(self):
            """A new token of every sequence, after what the eviction left."""
            self.lens = self.cache.d["lens"].download(np.int32, (seqs,)) + np.int32(1)
            self.cache.d["lens"].upload(self.lens)

        def step(self, s):
            p, kv = {n: b.ptr for n, b in self.d.items()}, ctypes.byref(self.kv)
            X.call("q27x_paged_prep_rows", p["qkv"], width, p["norm"], p["norm"], p["cos"], p["sin"], rot, 64, p["pos"], seqs, 1, None,
                   kv, p["qh"], nq, 1, 1e-6, seqs, s)
            X.call("q27x_paged_attn_rows", p["qh"], p["qkv"], width, kv, nq, 1, cap, 1, seqs, self.wa.ptr, p["out"], None, None, p["w"],
                   cap, s)
            X.call("q27x_paged_evict", kv, p["w"], cap, None, seqs, 1.0, p["acc"], p["ord"], cap, p["state"], 600, 590, 20, cap,
                   self.we.ptr, self.cache.d["lens"].ptr, s)

        def all(self):
            got = {n: self.d[n].download(self.host[n].dtype, self.host[n].shape) for n in ("qh", "out", "w", "acc", "ord", "state")}
            return {**got, **self.cache.pull(), "lens": self.cache.d["lens"].download(np.int32, (seqs,))}

    def same(a, b, what):
        for n in a:
            assert np.array_equal(a[n].view(np.uint8), b[n].view(np.uint8)), (n, what)

    eager, seen = State(), []
    for _ in range(steps):
        eager.grow()
        eager.step(None)
        X.call("q27x_device_sync")
        seen.append(eager.all())
    assert seen[-1]["lens"].tolist() != seen[0]["lens"].tolist() and (seen[0]["lens"][:2] == [590, 600]).all()

    st = State()
    graph = _Graph(X, st.step)
    for i in range(steps):
        st.grow()                                                   # (copies on the null stream between the replays)
        X.call("q27x_device_sync")
        graph.replay()
        same(st.all(), seen[i], f"replay {i}")
    graph.close()

    # two streams at once, a state and a workspace each
    pair = [(State(), ctypes.c_void_p()) for _ in range(2)]
    for _, s in pair:
        X.call("q27x_stream_create", ctypes.byref(s))
    for i in range(steps):
        for u, _ in pair:
            u.grow()
        X.call("q27x_device_sync")
        for u, s in pair:
            u.step(s)
        X.call("q27x_device_sync")
        for u, _ in pair:
            same(u.all(), seen[i], f"two streams, step {i}")
    for _, s in pair:
        X.call("q27x_stream_destroy", s)
