"""Decode on four-bit weights, and the token that it answers with: the operators, their plain forms and results.

- `proj`: a projection of 1 to 8 rows through NVFP4 weights (E2M1 codes, an E4M3 scale per 16 of them), as the reference's
  checkpoint holds its MLP and its head, on the rows that the activation quantizers give (q27x_proj_nvfp4_rows).
- `swiglu`: gate and up of an MLP on such weights, SwiGLU and the per-16 quantizer of what the down projection reads
  (q27x_swiglu_nvfp4_rows).
- `sample`: a token a row from its logits by temperature, top-k, top-p and min-p, with given random numbers
  (q27x_sample_rows).

Sizes are the repository's own: the 5120-wide model (17408 intermediate, 62080 logits), the 1024-wide one, the
248320 tokens of the whole vocabulary. Calls go to the null stream.
"""
import ctypes
import importlib.util
import math
import os
import sys

import numpy as np
import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_LIB = os.path.join(_ROOT, "qwen3.8-27b-mi50-cpp-engine_amd", "q27x.py")

HIDDEN, INTER, VOCAB, WHOLE = 5120, 17408, 62080, 248320
E2M1 = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def listed():
    return [
        # the 1024-wide model's out_proj on one row, residual: launch latency
        {"name": "proj_tiny", "kind": "proj", "rows": 1024, "K": 768, "nr": 1, "bf16": True, "res": "bf16"},
        # the down projection of a K=2 verify
        {"name": "proj_down", "kind": "proj", "rows": HIDDEN, "K": INTER, "nr": 3, "bf16": False, "res": "bf16"},
        # widths that no tile divides, rows that end inside one
        {"name": "proj_ragged", "kind": "proj", "rows": 9001, "K": 5136, "nr": 5, "bf16": True, "res": "f32"},
        # the head of a plain decode step
        {"name": "proj_head", "kind": "proj", "rows": VOCAB, "K": HIDDEN, "nr": 1, "bf16": False, "res": "none"},
        # a small MLP's gate and up
        {"name": "swiglu_small", "kind": "swiglu", "rows": 2048, "K": 1024, "nr": 2},
        # gate and up of a plain decode step
        {"name": "swiglu_1", "kind": "swiglu", "rows": INTER, "K": HIDDEN, "nr": 1},
        # gate and up on the most rows that a verify has
        {"name": "swiglu_8", "kind": "swiglu", "rows": INTER, "K": HIDDEN, "nr": 8},
        # one conversation's next token: latency
        {"name": "sample_1", "kind": "sample", "n": VOCAB, "nr": 1, "bf16": False, "how": "all"},
        # the rows of a K=2 verify, nucleus alone
        {"name": "sample_verify", "kind": "sample", "n": VOCAB, "nr": 3, "bf16": False, "how": "top_p"},
        # a served batch, each request with settings of its own, some of them greedy
        {"name": "sample_batch", "kind": "sample", "n": VOCAB, "nr": 64, "bf16": False, "how": "mixed"},
        # the whole vocabulary's logits in bf16, where many are equal
        {"name": "sample_whole", "kind": "sample", "n": WHOLE, "nr": 8, "bf16": True, "how": "min_p"},
        # nothing cut: every token counts
        {"name": "sample_plain", "kind": "sample", "n": VOCAB, "nr": 16, "bf16": False, "how": "plain"},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["proj", "proj", "swiglu", "sample", "sample"])
    if kind == "sample":
        n = _log(rng, 100, WHOLE)
        return {"kind": kind, "n": n, "nr": _log(rng, 1, min(64, 64 * VOCAB // n)), "bf16": rng.random() < 0.4,
                "how": rng.choice(["all", "top_k", "top_p", "min_p", "plain", "mixed", "mixed"])}
    K = 16 * _log(rng, 4, 1280)
    rows = min(_log(rng, 16, VOCAB), VOCAB * HIDDEN // K)
    if kind == "swiglu":
        return {"kind": kind, "rows": max(16, rows // 32 * 16), "K": K, "nr": rng.randint(1, 8)}
    return {"kind": kind, "rows": rows, "K": K, "nr": rng.randint(1, 8), "bf16": rng.random() < 0.5,
            "res": rng.choice(["none", "bf16", "f32"])}


# ---------------------------------------------------------------- inputs
class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda") * (hi - lo) + lo

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda")

    def pick(self, values, n, dtype):
        return torch.tensor(values, dtype=dtype, device="cuda")[self.ints(0, len(values), n)]


def _matrix(g, rows, K):
    """Codes as the quantizer leaves normal weights (the largest of 16 at 6 or 4), and scales of such groups."""
    v = g.normal(8192, 16)
    v = v / v.abs().amax(1, keepdim=True) * 6
    grid = torch.tensor(E2M1, device="cuda")
    code = (v.abs()[..., None] - grid).abs().argmin(-1) + 8 * (v < 0)
    pool = (code[:, ::2] | code[:, 1::2] << 4).to(torch.uint8).reshape(-1)
    w = torch.empty(rows, K // 2, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // K)
    for r in range(0, rows, step):
        part = w[r:r + step]
        part.copy_(pool[torch.randint(0, pool.numel(), part.shape, generator=g.g, device="cuda")])
    s = torch.empty(rows, K // 16, device="cuda").uniform_(0.3, 1.0, generator=g.g)
    return w, (s * 240).to(torch.float8_e4m3fn).view(torch.uint8)


def _rows_of(g, nr, K):
    """Activation rows as the per-16 quantizer leaves them: codes, scales."""
    x = g.normal(nr, K // 16, 16)
    s = x.abs().amax(-1) / 127
    return torch.round(x / s[..., None]).to(torch.int8).view(nr, K), s


def _settings(g, how, nr):
    """Temperature, top-k, top-p and min-p of each row (0, 0, 1 and 0 where it has none)."""
    t, k = g.uniform(0.6, 1.2, nr), torch.zeros(nr, dtype=torch.int32, device="cuda")
    p, m = torch.ones(nr, device="cuda"), torch.zeros(nr, device="cuda")
    if how in ("all", "top_k"):
        k = g.pick([20, 40, 50, 100], nr, torch.int32)
    if how in ("all", "top_p"):
        p = g.pick([0.8, 0.9, 0.95], nr, torch.float32)
    if how in ("all", "min_p"):
        m = g.pick([0.02, 0.05, 0.1], nr, torch.float32)
    if how == "mixed":
        t = t * g.pick([0.0, 1.0, 1.0, 1.0], nr, torch.float32)
        k = g.pick([0, 0, 1, 20, 50, 1000], nr, torch.int32)
        p = g.pick([1.0, 1.0, 0.5, 0.9, 0.95, 0.99], nr, torch.float32)
        m = g.pick([0.0, 0.0, 0.01, 0.05], nr, torch.float32)
    return t, k, p, m


def prepare(case, seed):
    g, nr = _Gen(seed), case["nr"]
    t = {}
    if case["kind"] == "sample":
        n = case["n"]
        # the bulk of a vocabulary, and the tokens that the context makes likely
        x = g.normal(nr, n, std=2.0)
        likely = g.ints(0, n, nr, 200)
        x.scatter_add_(1, likely, -torch.log(g.uniform(1e-6, 1.0, nr, 200)) * 2.5 + 2)
        t["logits"] = x.bfloat16() if case["bf16"] else x
        t["t"], t["k"], t["p"], t["m"] = _settings(g, case["how"], nr)
        t["u"] = g.uniform(0, 1, nr).clamp_max(1 - 2.0 ** -24)
        t["idx"] = torch.empty(nr, dtype=torch.int32, device="cuda")
        t["prob"] = torch.empty(nr, device="cuda")
        return {"case": case, "t": t}
    rows, K = case["rows"], case["K"]
    t["xq"], t["xs"] = _rows_of(g, nr, K)
    t["w"], t["s"] = _matrix(g, rows, K)
    if case["kind"] == "swiglu":
        t["w2"], t["s2"] = _matrix(g, rows, K)
        t["oq"] = torch.empty(nr, rows, dtype=torch.int8, device="cuda")
        t["os"] = torch.empty(nr, rows // 16, device="cuda")
        t["h"] = torch.empty(nr, rows // 16, 16, dtype=torch.bfloat16, device="cuda")
        # outputs of gate and up near 1, the down projection's input scale
        return {"case": case, "t": t, "alpha": 1 / (240 * 1.6 * math.sqrt(K)), "alpha2": 0.9 / (240 * 1.6 * math.sqrt(K)), "in_scale": 0.75}
    t["y"] = torch.empty(nr, rows, dtype=torch.bfloat16 if case["bf16"] else torch.float32, device="cuda")
    if case["res"] != "none":
        t["res"] = g.normal(nr, rows)
        if case["res"] == "bf16":
            t["res"] = t["res"].bfloat16()
    return {"case": case, "t": t, "alpha": 1 / (240 * 1.6 * math.sqrt(K))}


# ---------------------------------------------------------------- the framework's calls
def _load():
    if "q27x" not in sys.modules:
        spec = importlib.util.spec_from_file_location("q27x", _LIB)
        mod = importlib.util.module_from_spec(spec)
        sys.modules["q27x"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["q27x"]


def _p(x):
    return None if x is None else x.data_ptr()


def _handle(state):
    """What a program builds once for its buffers: the weights' handles, the workspace, the call's arguments."""
    X, case, t = _load(), state["case"], state["t"]
    L, nr = X.lib(), case["nr"]
    state["check"] = X.check
    if case["kind"] == "sample":
        t["work"] = torch.empty(L.q27x_sample_work_bytes(case["n"], nr), dtype=torch.uint8, device="cuda")
        return L.q27x_sample_rows, (_p(t["logits"]), int(case["bf16"]), case["n"], case["n"], nr, _p(t["t"]), _p(t["k"]),
                                    _p(t["p"]), _p(t["m"]), _p(t["u"]), _p(t["work"]), _p(t["idx"]), _p(t["prob"]), None)
    rows, K = case["rows"], case["K"]
    state["h"] = X.NVFP4(_p(t["w"]), _p(t["s"]), state["alpha"], rows, K)
    if case["kind"] == "swiglu":
        state["h2"] = X.NVFP4(_p(t["w2"]), _p(t["s2"]), state["alpha2"], rows, K)
        return L.q27x_swiglu_nvfp4_rows, (ctypes.byref(state["h"]), ctypes.byref(state["h2"]), _p(t["xq"]), K, _p(t["xs"]),
                                          _p(t["oq"]), _p(t["os"]), state["in_scale"], nr, None)
    return L.q27x_proj_nvfp4_rows, (ctypes.byref(state["h"]), _p(t["xq"]), K, _p(t["xs"]), _p(t["y"]), rows, int(case["bf16"]),
                                    _p(t.get("res")), int(case["res"] == "bf16"), rows, 1.0, nr, None)


def run(state):
    case, t = state["case"], state["t"]
    if own:
        if "call" not in state:
            state["call"] = _handle(state)
        fn, args = state["call"]
        rc = fn(*args)
        if rc:
            state["check"](rc)
    else:
        {"proj": _plain_proj, "swiglu": _plain_swiglu, "sample": _plain_sample}[case["kind"]](state)
    if case["kind"] == "proj":
        return {"y": t["y"]}
    if case["kind"] == "sample":
        return {"idx": t["idx"], "prob": t["prob"]}
    # the codes as the values that the down projection reads
    torch.mul(t["oq"].view_as(t["h"]), t["os"][..., None], out=t["h"])
    return {"h": t["h"], "scales": t["os"]}


# ---------------------------------------------------------------- plain forms
def _product(t, w, s, alpha, K):
    """alpha x W for the rows x, in fp32, some rows of W at a time."""
    x = (t["xq"].float().view(-1, K // 16, 16) * t["xs"][..., None]).view(-1, K)
    grid = torch.tensor(E2M1 + [-v for v in E2M1], device="cuda")
    y = torch.empty(x.shape[0], w.shape[0], device="cuda")
    step = max(1, (1 << 27) // K)
    for r in range(0, w.shape[0], step):
        b = w[r:r + step]
        v = torch.stack([grid[(b & 15).int()], grid[(b >> 4).int()]], -1).view(b.shape[0], K // 16, 16)
        v = v * s[r:r + step].view(torch.float8_e4m3fn).float()[..., None]
        y[:, r:r + step] = torch.matmul(x, v.view(b.shape[0], K).t())
    return y * alpha


def _plain_proj(state):
    case, t = state["case"], state["t"]
    y = _product(t, t["w"], t["s"], state["alpha"], case["K"])
    if "res" in t:
        y = y + t["res"].float()
    t["y"].copy_(y)


def _plain_swiglu(state):
    case, t = state["case"], state["t"]
    gate = _product(t, t["w"], t["s"], state["alpha"], case["K"])
    up = _product(t, t["w2"], t["s2"], state["alpha2"], case["K"])
    v = (gate / (1 + torch.exp(-gate)) * up * (1 / state["in_scale"])).view(case["nr"], -1, 16)
    s = v.abs().amax(-1) * (1 / 127)
    inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    t["oq"].copy_(torch.round(v * inv[..., None]).clamp(-127, 127).view(case["nr"], -1))
    t["os"].copy_(s)


def _plain_sample(state):
    # in 64 bits: a sum next to a random number decides between two tokens
    t = state["t"]
    x = t["logits"].double()
    n = x.shape[1]
    x, order = torch.sort(torch.where(torch.isfinite(x), x, -math.inf), dim=1, descending=True, stable=True)
    temp, k = t["t"].double()[:, None], t["k"].long()[:, None]
    k = torch.where(temp > 0, torch.where(k > 0, k, n), 1)
    rank = torch.arange(n, device="cuda")
    w = torch.exp((x - x[:, :1]) / torch.where(temp > 0, temp, 1.0)) * (rank < k)
    p = t["p"].double()[:, None]
    c = torch.cumsum(w, 1)
    w = w * ((p >= 1) | (rank == 0) | (c - w < p * c[:, -1:])) * ((rank == 0) | (w >= t["m"].double()[:, None]))
    c = torch.cumsum(w, 1)
    at = (c <= t["u"].double()[:, None] * c[:, -1:]).sum(1, keepdim=True)
    at = torch.minimum(at, (w > 0).sum(1, keepdim=True) - 1)
    t["idx"].copy_(torch.gather(order, 1, at)[:, 0])
    t["prob"].copy_((torch.gather(w, 1, at) / c[:, -1:])[:, 0])


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    nr = case["nr"]
    if case["kind"] == "sample":
        return {"bytes": nr * (case["n"] * (2.0 if case["bf16"] else 4.0) + 28), "flops": 4.0 * nr * case["n"]}
    rows, K = case["rows"], case["K"]
    x = nr * K * 1.25
    if case["kind"] == "swiglu":
        return {"bytes": 2 * rows * K * 9 / 16 + x + nr * rows * 1.25, "flops": 4.0 * nr * rows * K}
    out = (2 if case["bf16"] else 4) + {"none": 0, "bf16": 2, "f32": 4}[case["res"]]
    return {"bytes": rows * K * 9 / 16 + x + nr * rows * float(out), "flops": 2.0 * nr * rows * K}


# ---------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    t = state["t"]
    if case["kind"] == "sample":
        got = [_exact_token(state, r) for r in range(case["nr"])]
        return {"idx": torch.tensor([i for i, _ in got], dtype=torch.int32), "prob": torch.tensor([p for _, p in got], dtype=torch.float64)}
    y = _exact_product(t, t["w"], t["s"], state["alpha"])
    if case["kind"] == "proj":
        return {"y": y + t["res"].double() if "res" in t else y}
    u = _exact_product(t, t["w2"], t["s2"], state["alpha2"])
    v = (y * torch.sigmoid(y) * u / state["in_scale"]).unflatten(1, (-1, 16))
    step = v.abs().amax(-1, keepdim=True) / 127
    return {"h": torch.round(v / step.clamp_min(1e-300)) * step, "scales": step[..., 0]}


def _exact_product(t, w, s, alpha):
    """Each output as the sum over 16-wide slabs of (integer dot of doubled codes) x scales."""
    nr, K = t["xq"].shape
    x = t["xq"].double().view(nr, K // 16, 16)
    sign_mag = torch.tensor([0, 1, 2, 3, 4, 6, 8, 12, 0, -1, -2, -3, -4, -6, -8, -12], dtype=torch.float64, device="cuda")
    out = torch.zeros(nr, w.shape[0], dtype=torch.float64, device="cuda")
    step = max(1, (1 << 24) // K)
    for r in range(0, w.shape[0], step):
        b = w[r:r + step].long()
        codes = torch.zeros(b.shape[0], K, dtype=torch.float64, device="cuda")
        codes[:, 0::2], codes[:, 1::2] = sign_mag[b % 16], sign_mag[b // 16]
        scale = s[r:r + step].view(torch.float8_e4m3fn).double()
        for i in range(nr):
            dots = (codes.view(-1, K // 16, 16) * x[i]).sum(-1)
            out[i, r:r + step] = (dots * scale * t["xs"][i].double()).sum(-1) * (alpha / 2)
    return out


def _exact_token(state, r):
    t = state["t"]
    x = t["logits"][r].double().cpu().numpy()
    temp, k, p, m, u = (float(t[c][r]) for c in ("t", "k", "p", "m", "u"))
    ids = np.flatnonzero(np.isfinite(x))
    ids = ids[np.lexsort((ids, -x[ids]))]
    if temp <= 0:
        return int(ids[0]), 1.0
    w = np.exp((x[ids] - x[ids[0]]) / temp)
    if k >= 1:
        w = w[:int(k)]
    if p < 1:
        sums = np.cumsum(w)
        w = w[:max(1, int(np.searchsorted(sums, p * sums[-1], side="left")) + 1)]
    w = w[:max(1, int((w >= m).sum()))]
    sums = np.cumsum(w)
    i = min(int(np.searchsorted(sums, u * sums[-1], side="right")), len(w) - 1)
    return int(ids[i]), float(w[i] / sums[-1])
