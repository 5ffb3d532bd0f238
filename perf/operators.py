"""Serving many sequences from one paged key/value cache: the operators of a decode step, their plain forms and results.

- `prep`: per-head RMSNorm and rotary positions of up to four axes (time, height, width) for a batch's new rows, their
  keys and values appended to each sequence's pages (q27x_paged_prep_rows).
- `attn`: attention of each sequence's new tokens over its pages, optionally with the weight that every key got
  (q27x_paged_attn_rows).
- `evict`: those weights added up per key, and the cache of a sequence that has grown past its limit cut back to its
  newest and its heaviest keys (q27x_paged_evict).

Head layouts are the repository's own: 32 query / 8 kv heads of 128 (32 rotary dims), and the checkpoint's 24 / 4 heads
of 256 (64 rotary dims), both with the gate beside each query head. Calls go to the null stream.
"""
import ctypes
import functools
import importlib.util
import math
import os
import random
import sys

import torch

own = False

_ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
_LIB = os.path.join(_ROOT, "qwen3.8-27b-mi50-cpp-engine_amd", "q27x.py")

# (query heads, kv heads, head dim, rotary dims)
GEOMS = {"base": (32, 8, 128, 32), "trunk": (24, 4, 256, 64)}
EPS, THETA = 1e-6, 1e7
TABLE = 32768                                                 # rows of the rotary tables


def listed():
    return [
        # one sequence's next token on the checkpoint's heads, bf16 pages: latency
        {"name": "prep_1", "kind": "prep", "geom": "trunk", "group": 0, "page": 16, "seqs": 1, "rows": 1, "past": 777},
        # a decode step of a full batch: one token of each of 64 sequences
        {"name": "prep_64", "kind": "prep", "geom": "base", "group": 32, "page": 16, "seqs": 64, "rows": 1, "past": 4000},
        # prompts with images arriving: rows that share a time position and differ in height and width
        {"name": "prep_prompt", "kind": "prep", "geom": "trunk", "group": 32, "page": 64, "seqs": 3, "rows": 1531, "past": 100},
        # a single short conversation: latency
        {"name": "attn_short", "kind": "attn", "geom": "base", "group": 32, "page": 16, "seqs": 1, "rows": 1, "len": 203,
         "mix": 0, "weights": False},
        # a single long document on the checkpoint's heads
        {"name": "attn_long", "kind": "attn", "geom": "trunk", "group": 32, "page": 64, "seqs": 1, "rows": 1, "len": 32003,
         "mix": 0, "weights": False},
        # a served batch of ragged lengths
        {"name": "attn_ragged", "kind": "attn", "geom": "base", "group": 32, "page": 16, "seqs": 48, "rows": 1, "len": 8190,
         "mix": 7, "weights": False},
        # the verify rows of K=2 speculation, a batch of even lengths
        {"name": "attn_verify", "kind": "attn", "geom": "trunk", "group": 32, "page": 32, "seqs": 16, "rows": 3, "len": 4099,
         "mix": 0, "weights": False},
        # a large batch on bf16 pages
        {"name": "attn_bf16", "kind": "attn", "geom": "base", "group": 0, "page": 32, "seqs": 64, "rows": 1, "len": 4000,
         "mix": 0, "weights": False},
        # a batch whose keys' weights the eviction below needs
        {"name": "attn_weights", "kind": "attn", "geom": "base", "group": 32, "page": 16, "seqs": 32, "rows": 1, "len": 4097,
         "mix": 0, "weights": True},
        # the steady state of a bounded cache: a token came, one goes
        {"name": "evict_step", "kind": "evict", "geom": "base", "group": 32, "page": 16, "seqs": 32, "rows": 1, "len": 4097,
         "mix": 0, "budget": 4096, "high": 4096, "recent": 256, "decay": 1.0},
        # weights of accepted verify rows added up, no sequence past its limit
        {"name": "evict_add", "kind": "evict", "geom": "trunk", "group": 32, "page": 32, "seqs": 24, "rows": 3, "len": 8000,
         "mix": 5, "budget": 8192, "high": 8192, "recent": 1024, "decay": 1.0},
        # long prompts cut to half: the copy counts
        {"name": "evict_half", "kind": "evict", "geom": "base", "group": 32, "page": 64, "seqs": 6, "rows": 1, "len": 32001,
         "mix": 0, "budget": 16000, "high": 20000, "recent": 2000, "decay": 0.875},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["prep", "attn", "attn", "attn", "evict"])
    case = {"kind": kind, "geom": rng.choice(["base", "trunk"]), "group": rng.choice([0, 16, 32, 32, 64]),
            "page": rng.choice([8, 16, 16, 32, 64, 128])}
    if kind == "prep":
        case["seqs"] = _log(rng, 1, 64)
        return {**case, "rows": _log(rng, 1, 4600 // case["seqs"]), "past": _log(rng, 1, 8000)}
    case["seqs"] = _log(rng, 1, 64)
    case["rows"] = rng.choice([1, 1, 2, 3, 5, 8])
    case["mix"] = rng.choice([0, rng.randint(1, 999)])
    if kind == "attn":
        case["len"] = _log(rng, 8, min(32003, 256000 // case["seqs"] // (1 if case["group"] else 2)))
        return {**case, "weights": rng.random() < 0.3}
    case["len"] = _log(rng, 64, min(32001, 192006 // case["seqs"] // (1 if case["group"] else 2)))
    budget = max(1, int(case["len"] * rng.choice([0.5, 0.9, 0.999, 1.0])))
    return {**case, "budget": budget, "high": budget + rng.choice([0, 0, 3]), "recent": int(budget * rng.choice([0.0, 0.1, 0.5])),
            "decay": rng.choice([1.0, 1.0, 0.875, 0.5])}


def _lens(case):
    """Positions that each sequence's cache holds, the new rows included: all alike (mix 0), or spread over the range."""
    n, rows, most = case["seqs"], case["rows"], max(case["len"], case["rows"])
    if not case["mix"]:
        return [most] * n
    r = random.Random(case["mix"])
    got = [max(rows, _log(r, rows, most)) for _ in range(n)]
    got[r.randrange(n)] = most
    return got


# ---------------------------------------------------------------- inputs
class _Gen:
    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(seed)

    def normal(self, *shape, std=1.0):
        return torch.randn(*shape, generator=self.g, device="cuda") * std

    def bf16(self, *shape, std=1.0):
        return self.normal(*shape, std=std).bfloat16()

    def ints(self, lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=self.g, device="cuda", dtype=torch.int32)

    def uniform(self, lo, hi, *shape):
        return torch.rand(*shape, generator=self.g, device="cuda") * (hi - lo) + lo

    def perm(self, n):
        return torch.randperm(n, generator=self.g, device="cuda").to(torch.int32)


def _pages(g, case, lens, filled):
    """The two pools of a layer and each sequence's page table; `filled`: with keys and values in them."""
    nq, nkv, hd, _ = GEOMS[case["geom"]]
    G, page, width = case["group"], case["page"], nkv * hd
    per = -(-max(lens) // page)
    n = sum(-(-x // page) for x in lens) + 3
    t = {"table": torch.zeros(len(lens), per, dtype=torch.int32, device="cuda")}
    order, used = g.perm(n), 0
    for b, x in enumerate(lens):
        k = -(-x // page)
        t["table"][b, :k] = order[used:used + k]
        used += k
    # the pool holds the pages of keys, then those of values: one allocation, two pointers
    if G:
        t["codes"] = torch.zeros(2, n * page, width, dtype=torch.int8, device="cuda")
        t["scales"] = torch.zeros(2, n * page, width // G, device="cuda")
    else:
        t["codes"] = torch.zeros(2, n * page, width, dtype=torch.bfloat16, device="cuda")
    for i in range(2 if filled else 0):
        if G:
            t["codes"][i].random_(-127, 128, generator=g.g)
            t["scales"][i].uniform_(0.005, 0.03, generator=g.g)
        else:
            t["codes"][i].normal_(generator=g.g)
    return t


def _positions(case, nrows):
    """Time, height and width of every new row: text, and in it images of 24 x 31 that share a time."""
    past, rows = case["past"], case["rows"]
    i = torch.arange(rows, dtype=torch.int64)
    at, image = i % 1000, (i % 1000 >= 200) & (i % 1000 < 200 + 24 * 31)
    cell = at - 200
    base = past + (i // 1000) * 300
    text = torch.where(at < 200, base + at, base + 231 + at - 200 - 24 * 31)
    tm = torch.where(image, base + 200, text)
    h = torch.where(image, base + 200 + cell // 31, text)
    w = torch.where(image, base + 200 + cell % 31, text)
    return torch.stack([tm, h, w])[:, None].expand(3, case["seqs"], rows).reshape(3, nrows).to(torch.int32).cuda()


def _axes(rot):
    """The axis of each rotary pair: time, height and width in turn, time alone at the end of the range."""
    return [(i % 3) if i < rot // 2 - 2 else 0 for i in range(rot // 2)]


def prepare(case, seed):
    g = _Gen(seed)
    nq, nkv, hd, rot = GEOMS[case["geom"]]
    kind, seqs, rows = case["kind"], case["seqs"], case["rows"]
    lens = [case["past"] + rows] * seqs if kind == "prep" else _lens(case)
    nrows = seqs * rows
    t = _pages(g, case, lens, kind != "prep")
    t["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    t["row_start"] = torch.arange(seqs + 1, dtype=torch.int32, device="cuda") * rows
    state = {"case": case, "t": t, "max_len": max(lens), "nrows": nrows}
    if kind == "prep":
        t["qkv"] = g.bf16(nrows, 2 * nq * hd + 2 * nkv * hd)
        t["qn"], t["kn"] = g.bf16(hd, std=0.1), g.bf16(hd, std=0.1)
        ang = torch.arange(TABLE, dtype=torch.float64, device="cuda")[:, None] * \
            THETA ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / rot)
        t["cos"], t["sin"] = ang.cos().float(), ang.sin().float()
        t["pos"] = _positions(case, nrows)
        state["axes"] = _axes(rot)
        t["axes"] = torch.tensor(state["axes"], device="cuda")
        t["qh"] = torch.empty(nrows, nq * hd, dtype=torch.bfloat16, device="cuda")
        # the pool rows that the new keys and values go to: what a caller of the plain form has, and a reader of the pages
        i = t["lens"][:, None].long() - rows + torch.arange(rows, device="cuda")
        t["slot"] = (torch.gather(t["table"].long(), 1, i // case["page"]) * case["page"] + i % case["page"]).reshape(-1)
    elif kind == "attn":
        t["q"] = g.bf16(nrows, nq * hd)
        t["qkv"] = g.bf16(nrows, 2 * nq * hd + 2 * nkv * hd)
        t["out"] = torch.empty(nrows, nq * hd, dtype=torch.bfloat16, device="cuda")
        if case["weights"]:
            t["w"] = torch.zeros(nrows, state["max_len"], device="cuda")
    else:
        # weights and sums in steps of 2^-20, so that equal ones are there and sums are exact
        t["w"] = (g.uniform(0, 1, nrows, state["max_len"]) ** 8 * 65536).round() * 2.0 ** -20
        t["acc"] = (g.uniform(0, 1, seqs, state["max_len"]) ** 4 * 2.0 ** 20).round() * 2.0 ** -20
        known = (t["lens"] - rows).clamp_min(0)
        t["state"] = torch.stack([known, known + 50], 1).contiguous()
        # the order in which the keys came, shuffled by earlier evictions, which took 50 of each sequence
        mixed = g.uniform(0, 1, seqs, state["max_len"])
        mixed += torch.arange(state["max_len"], device="cuda") >= known[:, None]
        t["ord"] = torch.argsort(torch.argsort(mixed, 1), 1).to(torch.int32) + 50
        t["taken"] = g.ints(1, rows + 1, seqs) if rows > 1 else torch.ones(seqs, dtype=torch.int32, device="cuda")
        t["new_lens"] = torch.empty(seqs, dtype=torch.int32, device="cuda")
    return state


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
    """What a program builds once for its buffers: the cache's handle, the workspace, the call's arguments."""
    X, case, t = _load(), state["case"], state["t"]
    L = X.lib()
    nq, nkv, hd, rot = GEOMS[case["geom"]]
    s = t.get("scales")
    kv = X.PagedKV(k=_p(t["codes"][0]), v=_p(t["codes"][1]), ks=_p(s[0]) if s is not None else None,
                   vs=_p(s[1]) if s is not None else None, kv_group=case["group"], nkv=nkv, hd=hd,
                   n_pages=t["codes"].shape[1] // case["page"], page=case["page"], page_stride=case["page"],
                   table=_p(t["table"]), table_stride=t["table"].shape[1], lens=_p(t["lens"]), row_start=_p(t["row_start"]),
                   n_seq=case["seqs"])
    state["kv"], state["check"] = kv, X.check
    width = 2 * nq * hd + 2 * nkv * hd
    if case["kind"] == "prep":
        state["pair_axis"] = (ctypes.c_uint8 * (rot // 2))(*state["axes"])
        return L.q27x_paged_prep_rows, (
            _p(t["qkv"]), width, _p(t["qn"]), _p(t["kn"]), _p(t["cos"]), _p(t["sin"]), rot, TABLE, _p(t["pos"]),
            state["nrows"], 3, state["pair_axis"], ctypes.byref(kv), _p(t["qh"]), nq, 1, EPS, state["nrows"], None)
    if case["kind"] == "attn":
        n = L.q27x_paged_attn_work_bytes(nq, hd, state["max_len"], state["nrows"], int(case["weights"]))
        t["work"] = torch.empty(n, dtype=torch.uint8, device="cuda")
        return L.q27x_paged_attn_rows, (
            _p(t["q"]), _p(t["qkv"]), width, ctypes.byref(kv), nq, 1, state["max_len"], case["rows"], state["nrows"],
            _p(t["work"]), _p(t["out"]), None, None, _p(t.get("w")), state["max_len"] if case["weights"] else 0, None)
    n = L.q27x_paged_evict_work_bytes(case["seqs"], state["max_len"])
    t["work"] = torch.empty(n, dtype=torch.uint8, device="cuda")
    return L.q27x_paged_evict, (
        ctypes.byref(kv), _p(t["w"]), state["max_len"], _p(t["taken"]), state["nrows"], case["decay"], _p(t["acc"]),
        _p(t["ord"]), state["max_len"], _p(t["state"]), case["high"], case["budget"], case["recent"], state["max_len"],
        _p(t["work"]), _p(t["new_lens"]), None)


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
        {"prep": _plain_prep, "attn": _plain_attn, "evict": _plain_evict}[case["kind"]](state)
    if case["kind"] == "prep":
        return {"q": t["qh"], **_written(case, t)}
    if case["kind"] == "attn":
        return {"out": t["out"], **({"w": t["w"]} if case["weights"] else {})}
    return {n: t[n] for n in ("new_lens", "acc", "ord", "state", "codes", "scales") if n in t}


def _written(case, t):
    """The new keys and values as the attention reads them: bf16 pages as they are, codes as the values they stand for."""
    kv = t["codes"][:, t["slot"]]
    if not case["group"]:
        return {"kv": kv}
    s = t["scales"][:, t["slot"]]
    return {"kv": (kv.view(*s.shape, case["group"]) * s[..., None]).bfloat16(), "scales": s}


# ---------------------------------------------------------------- plain forms
def _plain_prep(state):
    case, t = state["case"], state["t"]
    nq, nkv, hd, rot = GEOMS[case["geom"]]
    n, half = state["nrows"], rot // 2
    x = t["qkv"].float()
    q, k = x[:, :2 * nq * hd].view(n, nq, 2, hd)[:, :, 0], x[:, 2 * nq * hd:2 * nq * hd + nkv * hd].view(n, nkv, hd)
    v = x[:, 2 * nq * hd + nkv * hd:]
    at = t["pos"].long()[t["axes"]].t()                                   # [row][pair]
    pair = torch.arange(half, device="cuda")
    cos, sin = t["cos"][at, pair][:, None], t["sin"][at, pair][:, None]

    def turn(y, w):
        y = y * (1 / torch.sqrt(y.square().mean(-1, keepdim=True) + EPS)) * (1 + w.float())
        a, b = y[..., :half], y[..., half:rot]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., rot:]], -1)

    t["qh"].copy_(turn(q, t["qn"]).reshape(n, -1))
    kv = torch.stack([turn(k, t["kn"]).reshape(n, -1), v])
    if not case["group"]:
        t["codes"][:, t["slot"]] = kv.bfloat16()
        return
    kv = kv.view(2, n, -1, case["group"])
    s = kv.abs().amax(-1) * (1 / 127)
    inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
    t["codes"][:, t["slot"]] = torch.round(kv * inv[..., None]).clamp(-127, 127).to(torch.int8).view(2, n, -1)
    t["scales"][:, t["slot"]] = s


def _plain_attn(state):
    case, t, L = state["case"], state["t"], state["max_len"]
    nq, nkv, hd, _ = GEOMS[case["geom"]]
    seqs, rows, g = case["seqs"], case["rows"], nq // nkv
    i = torch.arange(L, device="cuda")
    slot = t["table"].long()[:, i // case["page"]] * case["page"] + i % case["page"]        # [seq][key]

    def values(which):
        x = t["codes"][which, slot].float()
        if case["group"]:
            x = (x.view(seqs, L, -1, case["group"]) * t["scales"][which, slot][..., None])
        return x.view(seqs, L, nkv, hd)

    q = t["q"].float().view(seqs, rows, nkv, g, hd).permute(0, 2, 1, 3, 4).reshape(seqs, nkv, rows * g, hd)
    s = torch.matmul(q, values(0).permute(0, 2, 3, 1)) * (1 / math.sqrt(hd))               # [seq][kv head][row, head][key]
    last = t["lens"].long()[:, None] - rows + torch.arange(rows, device="cuda")             # [seq][row]
    seen = (i <= last[..., None])[:, None, :, None]                                         # [seq][1][row][1][key]
    s = s.view(seqs, nkv, rows, g, L).masked_fill(~seen, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(seqs, nkv, rows * g, L), values(1).permute(0, 2, 1, 3)).view(seqs, nkv, rows, g, hd)
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs * rows, nq, hd)
    gate = t["qkv"][:, :2 * nq * hd].view(-1, nq, 2, hd)[:, :, 1].float()
    t["out"].copy_((o * (1 / (1 + torch.exp(-gate)))).view(-1, nq * hd))
    if case["weights"]:
        w = p.sum((1, 3))                                                                   # [seq][row][key]
        t["w"].copy_(torch.where((i < t["lens"].long()[:, None])[:, None], w, t["w"].view(seqs, rows, L)).view(-1, L))


def _plain_evict(state):
    case, t, L = state["case"], state["t"], state["max_len"]
    seqs, rows = case["seqs"], case["rows"]
    lens, i = t["lens"].long()[:, None], torch.arange(L, device="cuda")
    known, total = torch.minimum(t["state"][:, :1].long(), lens), t["state"][:, 1:].long()
    now = total + lens - known
    held = i < lens
    # the sums: rows that were not accepted add nothing
    taken = torch.arange(rows, device="cuda")[None] < t["taken"][:, None]
    w = t["w"].view(seqs, rows, L) * taken[..., None]
    acc = functools.reduce(torch.add, w.unbind(1), torch.where(i < known, t["acc"] * case["decay"], torch.zeros_like(t["acc"])))
    came = torch.where(i < known, t["ord"].long(), total + i - known)
    t["acc"].copy_(torch.where(held, acc, t["acc"]))
    t["ord"].copy_(torch.where(held, came, t["ord"].long()))
    # what stays: the newest, then the heaviest, ties to the lowest index
    over = lens > case["high"]
    newest = held & (came >= now - case["recent"])
    rank = torch.where(newest, math.inf, torch.where(held, t["acc"], -math.inf))
    order = torch.sort(rank, dim=1, descending=True, stable=True).indices
    stays = torch.zeros_like(held).scatter_(1, order[:, :case["budget"]], True)
    hole, moved = (over & held & ~stays & (i < case["budget"])).nonzero(), (over & stays & (i >= case["budget"])).nonzero()
    b, to, fro = hole[:, 0], hole[:, 1], moved[:, 1]
    t["acc"][b, to], t["ord"][b, to] = t["acc"][b, fro], t["ord"][b, fro]
    slot = t["table"].long()[:, i // case["page"]] * case["page"] + i % case["page"]
    t["codes"][:, slot[b, to]] = t["codes"][:, slot[b, fro]]
    if case["group"]:
        t["scales"][:, slot[b, to]] = t["scales"][:, slot[b, fro]]
    t["new_lens"].copy_(torch.where(over, case["budget"], lens)[:, 0])
    t["state"].copy_(torch.cat([t["new_lens"][:, None].long(), now], 1))


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    nq, nkv, hd, rot = GEOMS[case["geom"]]
    G, seqs, rows = case["group"], case["seqs"], case["rows"]
    n = seqs * rows
    position = 2 * nkv * hd * ((1 + 4 / G) if G else 2)                   # a position's key and value in the pages
    if case["kind"] == "prep":
        return {"bytes": n * (4 * nq * hd + 4 * nkv * hd + position + 12) + min(n, TABLE) * 4.0 * rot,
                "flops": n * (nq + nkv) * (4.0 * hd + 3 * rot)}
    lens = _lens(case)
    if case["kind"] == "attn":
        return {"bytes": sum(lens) * (position + (4.0 * rows if case["weights"] else 0)) + n * 6.0 * nq * hd,
                "flops": 4.0 * rows * nq * hd * sum(lens)}
    cut = [x - case["budget"] if x > case["high"] else 0 for x in lens]
    # every key's weights, sum and order; the moved ones' cache rows, about the share of the tail that stays
    moves = sum(c * case["budget"] / x for c, x in zip(cut, lens))
    return {"bytes": sum(lens) * (8.0 + 4 * rows + 4) + moves * 2 * position, "flops": sum(lens) * (rows + 1.0)}


# ---------------------------------------------------------------- the same in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    return {"prep": _exact_prep, "attn": _exact_attn, "evict": _exact_evict}[case["kind"]](state)


def _exact_prep(state):
    case, t = state["case"], state["t"]
    nq, nkv, hd, rot = GEOMS[case["geom"]]
    G, half = case["group"], rot // 2
    x = t["qkv"].double()
    c = torch.stack([t["cos"].double()[t["pos"][a].long(), i] for i, a in enumerate(state["axes"])], 1)
    s = torch.stack([t["sin"].double()[t["pos"][a].long(), i] for i, a in enumerate(state["axes"])], 1)

    def head(y, w):
        y = y / (y.pow(2).sum(-1, keepdim=True) / hd + EPS).sqrt() * (1.0 + w.double())
        z = torch.complex(y[:, :half], y[:, half:rot]) * torch.complex(c, s)
        return torch.cat([z.real, z.imag, y[:, rot:]], 1)

    q = [head(x[:, 2 * h * hd:(2 * h + 1) * hd], t["qn"]) for h in range(nq)]
    k0 = 2 * nq * hd
    k = [head(x[:, k0 + h * hd:k0 + (h + 1) * hd], t["kn"]) for h in range(nkv)]
    kv = torch.stack([torch.cat(k, 1), x[:, k0 + nkv * hd:]])
    if not G:
        return {"q": torch.cat(q, 1), "kv": kv}
    kv = kv.unflatten(-1, (-1, G))
    step = kv.abs().amax(-1) / 127
    codes = torch.round(kv / step.clamp_min(1e-300)[..., None])
    return {"q": torch.cat(q, 1), "kv": codes * step[..., None], "scales": step}


def _exact_attn(state):
    case, t = state["case"], state["t"]
    nq, nkv, hd, _ = GEOMS[case["geom"]]
    rows, G, page, g = case["rows"], case["group"], case["page"], nq // nkv
    if sum(_lens(case)) * nkv * hd > 400_000_000:
        return None
    out = torch.zeros(state["nrows"], nq, hd, dtype=torch.float64, device="cuda")
    w = torch.zeros(state["nrows"], state["max_len"], dtype=torch.float64, device="cuda")
    for b, n in enumerate(_lens(case)):
        ids = t["table"][b, :-(-n // page)].long()
        kv = t["codes"].view(2, -1, page, nkv * hd)[:, ids].reshape(2, -1, nkv * hd)[:, :n].double()
        if G:
            sc = t["scales"].view(2, -1, page, nkv * hd // G)[:, ids].reshape(2, -1, nkv * hd // G)[:, :n].double()
            kv = kv * sc.repeat_interleave(G, 2)
        for r in range(rows):
            m, row = n - rows + r + 1, b * rows + r
            for h in range(nkv):
                k, v = kv[0, :m, h * hd:(h + 1) * hd], kv[1, :m, h * hd:(h + 1) * hd]
                q = t["q"][row].double().view(nq, hd)[h * g:(h + 1) * g]
                p = torch.softmax(q @ k.t() / math.sqrt(hd), 1)
                out[row, h * g:(h + 1) * g] = p @ v
                w[row, :m] += p.sum(0)
    gate = t["qkv"].double()[:, :2 * nq * hd].view(-1, nq, 2, hd)[:, :, 1]
    got = {"out": (out * torch.sigmoid(gate)).view(-1, nq * hd)}
    return {**got, "w": w} if case["weights"] else got


def _exact_evict(state):
    case, t = state["case"], state["t"]
    page, budget = case["page"], case["budget"]
    acc, scales = t["acc"].double(), t["scales"].double() if "scales" in t else None
    for b, n in enumerate(_lens(case)):
        known, total = min(int(t["state"][b, 0]), n), int(t["state"][b, 1])
        rows = range(b * case["rows"], b * case["rows"] + int(t["taken"][b]))
        acc[b, known:n] = 0
        acc[b, :n] = acc[b, :n] * case["decay"] + t["w"][list(rows), :n].double().sum(0)
        if n <= case["high"]:
            continue
        came = torch.cat([t["ord"][b, :known].long(), total + torch.arange(n - known, device="cuda")])
        old = (came < total + n - known - case["recent"]).nonzero()[:, 0]
        goes = old[torch.sort(acc[b, old], stable=True, descending=True).indices[budget - (n - len(old)):]]
        stays = torch.ones(n, dtype=torch.bool, device="cuda")
        stays[goes] = False
        to, fro = goes[goes < budget].sort().values, stays[budget:].nonzero()[:, 0] + budget
        acc[b, to] = acc[b, fro]
        if scales is not None:
            at = t["table"][b].long()
            scales[:, at[to // page] * page + to % page] = scales[:, at[fro // page] * page + fro % page]
    got = {"new_lens": None, "acc": acc, "ord": None, "state": None, "codes": None}
    return {**got, "scales": scales} if scales is not None else got
