"""Float64 forms of the paged-cache operators (rows of many sequences, rotary positions of several axes, attention over
pages, eviction by accumulated weight), written from their definitions in include/q27x.h, and a device cache to run them
on. A batch is (lens, counts): keys that each sequence holds, rows of it in the call."""
import numpy as np

from ref64 import bf16_rne, bf2f

INT8_GROUPS = (16, 32, 64)


def bf(x):
    return bf16_rne(np.asarray(x, np.float32))


class Cache:
    """Host copy of a pool of pages and its tables; `push` puts it on the device, `pull` reads it back."""

    def __init__(self, rng, lens, counts, nkv=2, hd=128, group=32, page=16, spare=3, page_stride=0, cap=None, fill=True):
        self.nkv, self.hd, self.group, self.page = nkv, hd, group, page
        self.lens, self.counts = np.asarray(lens, np.int32), np.asarray(counts, np.int32)
        self.row_start = np.concatenate([[0], np.cumsum(self.counts)]).astype(np.int32)
        self.stride = page_stride or page
        self.page_stride = page_stride
        cap = max(max(lens), 1) if cap is None else cap
        per = -(-cap // page)
        need = [-(-max(int(x), 1) // page) for x in lens] if cap is None else [per] * len(lens)
        need = [min(per, max(n, 1)) for n in need]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(lens), per), -1, np.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order[at:at + n]
            at += n
        width, rows = nkv * hd, self.n_pages * self.stride
        if group:
            self.k, self.v = (rng.integers(-127, 128, (rows, width)).astype(np.int8) if fill else np.full((rows, width), 77, np.int8)
                              for _ in range(2))
            self.ks, self.vs = (rng.uniform(0.002, 0.03, (rows, width // group)).astype(np.float32) if fill else
                                np.full((rows, width // group), 0.5, np.float32) for _ in range(2))
        else:
            self.k, self.v = (bf(rng.standard_normal((rows, width))) if fill else np.full((rows, width), 0x4242, np.uint16) for _ in range(2))
            self.ks = self.vs = None

    def slot(self, b, key):
        """The pool row of a key, or -1."""
        if key < 0 or key // self.page >= self.table.shape[1]:
            return -1
        p = self.table[b, key // self.page]
        return -1 if p < 0 or p >= self.n_pages else int(p) * self.stride + key % self.page

    def rows(self, b, n):
        """Pool rows of keys 0 .. n - 1."""
        return np.array([self.slot(b, i) for i in range(n)], np.int64)

    def values(self, which, slots):
        """[key][kv head][dim] in float64."""
        x = (self.k, self.v)[which][slots]
        if not self.group:
            return bf2f(x).astype(np.float64).reshape(-1, self.nkv, self.hd)
        s = (self.ks, self.vs)[which][slots].astype(np.float64)
        return (x.reshape(len(slots), -1, self.group).astype(np.float64) * s[..., None]).reshape(-1, self.nkv, self.hd)

    def push(self, X, row_start=True):
        self.X = X
        self.d = {n: X.DevBuf(array=getattr(self, n)) for n in ("k", "v", "ks", "vs", "table", "lens", "row_start")
                  if getattr(self, n) is not None}
        p = {n: b.ptr for n, b in self.d.items()}
        self.kv = X.PagedKV(k=p["k"], v=p["v"], ks=p.get("ks"), vs=p.get("vs"), kv_group=self.group, nkv=self.nkv, hd=self.hd,
                            n_pages=self.n_pages, page=self.page, page_stride=self.page_stride, table=p["table"],
                            table_stride=self.table.shape[1], lens=p["lens"], row_start=p["row_start"] if row_start else None,
                            n_seq=len(self.lens))
        return self.kv

    def pull(self):
        got = {}
        for n in ("k", "v", "ks", "vs"):
            a = getattr(self, n)
            if a is not None:
                got[n] = self.d[n].download(a.dtype, a.shape)
        return got


def rotate(y, pos, axes, rot, theta=1e4):
    """Rotate-half of the first rot dims: y [row][head][dim], pos [axis][row]."""
    half = rot // 2
    ang = np.stack([pos[axes[i]].astype(np.float64) * theta ** (-2.0 * i / rot) for i in range(half)], 1)[:, None]
    a, b = y[..., :half], y[..., half:rot]
    return np.concatenate([a * np.cos(ang) - b * np.sin(ang), b * np.cos(ang) + a * np.sin(ang), y[..., rot:]], -1)


def tables(n_pos, rot, theta=1e4):
    ang = np.arange(n_pos, dtype=np.float64)[:, None] * theta ** (-2.0 * np.arange(rot // 2) / rot)
    return np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32)


def rmsnorm(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1.0 + w)


def attention(cache, q, nq, max_len=None):
    """q [row][head][dim] float64 -> (out before the gate, sum p|v|, weights per key, largest sum |q k| / sqrt(hd)) of every
    row; rows that see nothing 0. Weights [row][longest]."""
    nrow, g, hd = len(q), nq // cache.nkv, cache.hd
    longest = int(max(max(cache.lens), 1))
    out, mag = np.zeros((nrow, nq, hd)), np.zeros((nrow, nq, hd))
    w, big = np.zeros((nrow, longest)), np.zeros(nrow)
    for b, (n, cnt) in enumerate(zip(cache.lens, cache.counts)):
        slots = cache.rows(b, min(int(n), max_len or int(n)))
        there = np.flatnonzero(slots >= 0)
        if not len(there):
            continue
        K, V = cache.values(0, slots[there]), cache.values(1, slots[there])
        for i in range(cnt):
            row = cache.row_start[b] + i
            see = there <= n - cnt + i
            if not see.any():
                continue
            for h in range(nq):
                k, v, idx = K[see, h // g], V[see, h // g], there[see]
                with np.errstate(invalid="ignore", over="ignore"):
                    x = k @ q[row, h] / np.sqrt(hd)
                    big[row] = max(big[row], np.nan_to_num((np.abs(k) @ np.abs(q[row, h])).max() / np.sqrt(hd)))
                    p = np.exp(x - x.max())
                    p /= p.sum()
                    out[row, h] = p @ v
                    mag[row, h] = p @ np.abs(v)
                w[row, idx] += p
    return out, mag, w, big


def evict(acc, ord_, state, n, w_rows, decay, high, budget, recent):
    """One sequence: acc, ord_ float32 / int32 rows, changed in place; w_rows the accepted rows' weights. Returns the new
    length and the moves [(from, to)]."""
    known = min(max(int(state[0]), 0), n)
    total = int(state[1]) - (max(int(state[0]), 0) - known)        # (keys taken back are the last that came)
    now = total + n - known
    acc[:known] = acc[:known] * np.float32(decay)
    acc[known:n] = 0
    for r in w_rows:
        acc[:n] = acc[:n] + r[:n].astype(np.float32)
    ord_[known:n] = total + np.arange(n - known)
    state[1] = now
    if n <= high:
        state[0] = n
        return n, []
    new = np.zeros(n, bool)
    new[np.argsort(-ord_[:n].astype(np.int64), kind="stable")[:recent]] = True
    key = [(-2, 0.0, i) if new[i] else (0, 0.0, i) if np.isnan(acc[i]) else (-1, -float(acc[i]), i) for i in range(n)]
    stays = np.zeros(n, bool)
    stays[[k[2] for k in sorted(key)[:budget]]] = True
    moves = list(zip((np.flatnonzero(stays[budget:]) + budget).tolist(), np.flatnonzero(~stays[:budget]).tolist()))
    for src, dst in moves:
        acc[dst], ord_[dst] = acc[src], ord_[src]
    state[0] = budget
    return budget, moves
