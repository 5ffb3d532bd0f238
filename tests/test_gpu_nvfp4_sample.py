"""A decode step's end on NVFP4 weights with sampled tokens, as a server runs it: norm, gate | up, down on the residual in place, norm,
head, a token a row, acceptance of the drafts. Every call against its float64 form on what it read; captured and replayed, and on two
streams at once, bit for bit as one after another."""
import ctypes

import numpy as np
import pytest

import test_gpu_nvfp4 as nvfp4
import test_gpu_sample as sampling
from ref64 import bf16_rne, bf2f, rmsnorm
from test_gpu_nvfp4 import Matrix
from test_gpu_paged import _Graph

pytestmark = pytest.mark.gpu
HID, MID, VOCAB, ROWS, EPS, IN_SCALE = 1024, 2064, 5003, 5, 1e-6, 0.6
U = 2.0 ** -24


class Step:
    def __init__(self, X, bf16_logits):
        rng = np.random.default_rng(12)
        self.X, self.bf16 = X, bf16_logits
        alpha = 0.05 / np.sqrt(HID)
        self.gate, self.up = (Matrix(X, rng, MID, HID, alpha=a) for a in (alpha, -alpha))
        self.down = Matrix(X, rng, HID, MID, alpha=0.01 / np.sqrt(MID))
        self.head = Matrix(X, rng, VOCAB, HID, alpha=0.004)
        i32, f32, u16 = (lambda *s: np.zeros(s, np.int32)), (lambda *s: np.zeros(s, np.float32)), (lambda *s: np.zeros(s, np.uint16))
        self.host = {
            "x": u16(ROWS, HID), "norm": bf16_rne((rng.standard_normal((2, HID)) * 0.1).astype(np.float32)),
            "xq": np.zeros((ROWS, HID), np.int8), "xs": f32(ROWS, HID // 16), "zq": np.zeros((ROWS, HID), np.int8), "zs": f32(ROWS, HID // 16),
            "oq": np.zeros((ROWS, MID), np.int8), "os": f32(ROWS, MID // 16),
            "logits": (u16 if bf16_logits else f32)(ROWS, VOCAB), "u": f32(ROWS), "idx": i32(ROWS), "prob": f32(ROWS), "drafts": i32(ROWS - 1),
            "t": np.array([0.8, 1.3, 0.0, 1.0, 0.6], np.float32), "k": np.array([50, 0, 0, 700, 0], np.int32),
            "p": np.array([0.95, 1, 1, 0.99, 0.5], np.float32), "m": np.array([0, 0.01, 0, 0, 0.02], np.float32),
            "nacc": i32(2), "committed": i32(8)}
        self.d = {n: X.DevBuf(array=a) for n, a in self.host.items()}
        self.work = X.DevBuf(X.lib().q27x_sample_work_bytes(VOCAB, ROWS))

    def feed(self, i):
        """Inputs of step i."""
        rng = np.random.default_rng(100 + i)
        self.x = bf16_rne(rng.standard_normal((ROWS, HID)).astype(np.float32) * 2)
        self.drafts = rng.integers(0, VOCAB, ROWS - 1).astype(np.int32)
        self.u = rng.random(ROWS).astype(np.float32)
        for n, a in (("x", self.x), ("drafts", self.drafts), ("u", self.u)):
            self.d[n].upload(a)

    def run(self, s):
        X, p = self.X, {n: b.ptr for n, b in self.d.items()}
        ref = lambda m: ctypes.byref(m.handle)
        X.call("q27x_rmsnorm_quant_rows", p["x"], 1, HID, p["norm"], 1.0, EPS, HID, None, None, 0, p["xq"], p["xs"], 0, 1.0, ROWS, s)
        X.call("q27x_swiglu_nvfp4_rows", ref(self.gate), ref(self.up), p["xq"], HID, p["xs"], p["oq"], p["os"], IN_SCALE, ROWS, s)
        X.call("q27x_proj_nvfp4_rows", ref(self.down), p["oq"], MID, p["os"], p["x"], HID, 1, p["x"], 1, HID, 1.0, ROWS, s)
        X.call("q27x_rmsnorm_quant_rows", p["x"], 1, HID, p["norm"] + 2 * HID, 1.0, EPS, HID, None, None, 0, p["zq"], p["zs"], 0, 1.0, ROWS, s)
        X.call("q27x_proj_nvfp4_rows", ref(self.head), p["zq"], HID, p["zs"], p["logits"], VOCAB, int(self.bf16), None, 0, 0, 0.0, ROWS, s)
        X.call("q27x_sample_rows", p["logits"], int(self.bf16), VOCAB, VOCAB, ROWS, p["t"], p["k"], p["p"], p["m"], p["u"], self.work.ptr,
               p["idx"], p["prob"], s)
        X.call("q27x_accept", p["idx"], p["drafts"], ROWS - 1, p["nacc"], p["committed"], s)

    def all(self):
        got = {n: self.d[n].download(self.host[n].dtype, self.host[n].shape) for n in self.host}
        got["committed"] = got["committed"][:got["nacc"][1]]        # (nothing behind is written)
        return got


def check_norm(q, s, x, w):
    """Codes and scales of a normed row: the norm in fp32, some 1100 roundings at most (its sum's half of them), and the code's own half step."""
    v = rmsnorm(bf2f(x).astype(np.float64), bf2f(w).astype(np.float64), 1.0, EPS).reshape(ROWS, -1, 16)
    rel, s = 1100 * U, s.astype(np.float64)
    top = np.abs(v).max(-1) / 127
    assert (np.abs(s - top) <= rel * top).all()
    off = np.abs(q.reshape(v.shape) * s[..., None] - v)
    assert (off <= (0.5 + 127 * 4 * U) * s[..., None] + rel * np.abs(v) + rel * 127 * top[..., None]).all()


@pytest.mark.parametrize("bf16", [False, True])
def test_every_call_on_what_it_read(gpu, bf16):
    st = Step(gpu, bf16)
    for i in range(3):
        st.feed(i)
        st.run(None)
        gpu.call("q27x_device_sync")
        g = st.all()
        check_norm(g["xq"], g["xs"], st.x, st.host["norm"][0])
        nvfp4.check_swiglu(g["oq"], g["os"], st.gate, st.up, g["xq"], g["xs"], IN_SCALE)
        nvfp4.check(g["x"], st.down, g["oq"], g["os"], st.x, 1.0)
        assert not np.array_equal(g["x"], st.x)
        check_norm(g["zq"], g["zs"], g["x"], st.host["norm"][1])
        nvfp4.check(g["logits"], st.head, g["zq"], g["zs"])
        v = (bf2f(g["logits"]) if bf16 else g["logits"]).astype(np.float32)
        for r in range(ROWS):
            want = sampling.answers(v[r], *(float(st.host[n][r]) for n in "t"), int(st.host["k"][r]), float(st.host["p"][r]),
                                    float(st.host["m"][r]), float(st.u[r]))
            assert g["idx"][r] in want, (i, r, want)
        hit = g["idx"][:-1] == st.drafts
        nacc = int(np.argmin(hit)) if not hit.all() else ROWS - 1
        assert g["nacc"].tolist() == [nacc, nacc + 1] and np.array_equal(g["committed"], g["idx"][:nacc + 1])


def test_drafts_that_the_sample_meets(gpu):
    """Drafts equal to what is drawn are accepted as far as they are, for every length."""
    X, st = gpu, Step(gpu, False)
    st.feed(0)
    st.run(None)
    X.call("q27x_device_sync")
    idx = st.all()["idx"]
    for n in range(ROWS):
        st.feed(0)
        drafts = idx[:-1].copy()
        drafts[n:] = (drafts[n:] + 1) % VOCAB
        st.d["drafts"].upload(drafts)
        st.run(None)
        X.call("q27x_device_sync")
        g = st.all()
        assert g["nacc"].tolist() == [n, n + 1] and np.array_equal(g["committed"], idx[:n + 1])


def same(a, b, what):
    for n in a:
        assert np.array_equal(np.ascontiguousarray(a[n]).view(np.uint8), np.ascontiguousarray(b[n]).view(np.uint8)), (n, what)


def test_streams_and_graphs(gpu):
    """Captured, and replayed with eager work between; and on two streams, a workspace each."""
    X, steps = gpu, 5
    eager, seen = Step(X, False), []
    for i in range(steps):
        eager.feed(i)
        eager.run(None)
        X.call("q27x_device_sync")
        seen.append(eager.all())
    assert len({s["idx"].tobytes() for s in seen}) == steps

    st = Step(X, False)
    graph = _Graph(X, st.run)
    for i in range(steps):
        eager.feed(steps - i)                                       # (other calls of the same kernels between the replays)
        eager.run(None)
        st.feed(i)
        X.call("q27x_device_sync")
        graph.replay()
        same(st.all(), seen[i], f"replay {i}")
    graph.close()

    pair = [(Step(X, False), ctypes.c_void_p()) for _ in range(2)]
    for _, s in pair:
        X.call("q27x_stream_create", ctypes.byref(s))
    for i in range(steps):
        for j, (u, _) in enumerate(pair):
            u.feed((i + j) % steps)
        X.call("q27x_device_sync")
        for u, s in pair:
            u.run(s)
        X.call("q27x_device_sync")
        for j, (u, _) in enumerate(pair):
            same(u.all(), seen[(i + j) % steps], f"two streams, step {i}")
    for _, s in pair:
        X.call("q27x_stream_destroy", s)


@pytest.mark.parametrize("rows,K,nr", [(5121, 272, 8), (5120, 272, 2), (100, 528, 5), (5121, 17424, 6), (300, 20496, 3)])
def test_residual_in_place(gpu, rows, K, nr):
    """y over res, bf16, in every kernel: the bits of the call that writes elsewhere."""
    X, rng = gpu, np.random.default_rng(rows + nr)
    m = Matrix(X, rng, rows, K, alpha=0.01)
    xq, xs = nvfp4.rows_of(rng, nr, K)
    res = bf16_rne(rng.standard_normal((nr, rows + 3)).astype(np.float32))
    apart = nvfp4.project(X, m, xq, xs, True, res, 1.0, pad=3)
    y, dq, ds = X.DevBuf(array=res), X.DevBuf(array=xq), X.DevBuf(array=xs)
    X.call("q27x_proj_nvfp4_rows", ctypes.byref(m.handle), dq.ptr, K, ds.ptr, y.ptr, rows + 3, 1, y.ptr, 1, rows + 3, 1.0, nr, None)
    X.call("q27x_device_sync")
    got = y.download(np.uint16, res.shape)
    assert np.array_equal(got[:, :rows], apart) and np.array_equal(got[:, rows:], res[:, rows:])


def test_one_row_needs_no_strides(gpu):
    X, rng = gpu, np.random.default_rng(1)
    m = Matrix(X, rng, 99, 400)
    xq, xs = nvfp4.rows_of(rng, 1, 400)
    want = nvfp4.project(X, m, xq, xs)
    dq, ds, y = X.DevBuf(array=xq), X.DevBuf(array=xs), X.DevBuf(4 * 99)
    X.call("q27x_proj_nvfp4_rows", ctypes.byref(m.handle), dq.ptr, 0, ds.ptr, y.ptr, -1, 0, None, 0, 0, 0.0, 1, None)
    X.call("q27x_device_sync")
    assert np.array_equal(y.download(np.float32, (1, 99)), want)


def test_one_workspace_for_calls_in_turn(gpu):
    """Calls of many sizes one behind another on a stream, with the largest one's workspace and no wait between."""
    X, rng = gpu, np.random.default_rng(2)
    sizes = [(62080, 3), (300, 40), (62080, 20), (5000, 7), (140000, 2), (4096, 1), (62080, 1), (20000, 30)]
    work = X.DevBuf(max(X.lib().q27x_sample_work_bytes(n, nr) for n, nr in sizes))
    calls = []
    for n, nr in sizes:
        x, u = sampling.logits(rng, nr, n), rng.random(nr).astype(np.float32)
        calls.append((x, u, X.DevBuf(array=x), X.DevBuf(array=u), X.DevBuf(4 * nr), X.DevBuf(4 * nr)))
    for (n, nr), (_, _, x, u, idx, prob) in zip(sizes, calls):
        X.call("q27x_sample_rows", x.ptr, 0, n, n, nr, None, None, None, None, u.ptr, work.ptr, idx.ptr, prob.ptr, None)
    X.call("q27x_device_sync")
    for (n, nr), (x, u, _, _, idx, prob) in zip(sizes, calls):
        want = sampling.sample(X, x, u=u)
        assert np.array_equal(idx.download(np.int32, (nr,)), want[0]) and np.array_equal(prob.download(np.float32, (nr,)), want[1])
