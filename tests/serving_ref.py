"""Plain 64-bit numpy forms of the serving operators (rotary positions, paged cache, attention over
it, sampling) and a paged cache on the device, for the tests of the kernels behind them."""
import ctypes as C
import math

import numpy as np

F32, BF16, I8, F8 = 0, 3, 4, 5  # jas_dtype
QMAX = {I8: 127.0, F8: 448.0}
STORE = {F32: np.float32, BF16: np.uint16, I8: np.int8, F8: np.uint8}


def to_bf16(x):
    """bf16 bit patterns of fp32 values, to nearest even."""
    x = np.ascontiguousarray(x, np.float32)
    u = x.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def from_bf16(u):
    return (u.astype(np.uint32) << 16).view(np.float32)


def _e4m3():
    c = np.arange(256)
    e, m = (c >> 3) & 15, c & 7
    v = np.where(e == 0, m * 2.0 ** -9, (8 + m) * 2.0 ** (e - 10.0))
    v[(c & 127) == 127] = np.nan
    return np.where(c >> 7, -v, v)


E4M3 = _e4m3()


def stored(x, dtype):
    """Rows of fp32 values as an 8-bit cache holds them: (the codes' values, scales)."""
    with np.errstate(all="ignore"):
        s = (np.abs(x).max(-1) / np.float32(QMAX[dtype])).astype(np.float32)
        s = np.where(np.isfinite(x).all(-1), np.where(s < np.float32(2.0 ** -126), np.float32(0), s), np.float32(np.nan))
        t = x.astype(np.float64) / s.astype(np.float64)[..., None]
        t = np.where((s > 0)[..., None], t, 0.0)
        if dtype == I8:
            t = np.clip(np.rint(t), -127, 127)
        else:
            step = np.ldexp(1.0, np.maximum(np.frexp(t)[1] - 4, -9))
            t = np.clip(np.rint(t / step) * step, -448, 448)
    return t, s


class Cache:
    """A paged cache on the device and its plain copy: k, v [pages, heads, page, dh] as values."""

    def __init__(self, jas, dtype, pages, heads, page, dh, table, token_major=False, pad=0, fill=0.0):
        self.jas, self.dtype, self.shape = jas, dtype, (pages, heads, page, dh)
        es = np.dtype(STORE[dtype]).itemsize
        pad = pad * 16 // es
        row = dh + pad
        if token_major:
            self.strides = (page * heads * row, row, heads * row)
        else:
            self.strides = (heads * page * row, page * row, row)
        n = pages * heads * page * row
        raw = np.full(n, fill, np.float32)
        raw = to_bf16(raw) if dtype == BF16 else raw.astype(STORE[dtype]) if dtype != F8 else np.full(n, 127 if np.isnan(fill) else 0, np.uint8)
        self.raw = raw
        self.k, self.v = jas.to_device(raw.view(np.uint8)), jas.to_device(raw.view(np.uint8))
        self.ks = self.vs = None
        if dtype in QMAX:
            self.ks, self.vs = (jas.to_device(np.full((pages, heads, page), fill, np.float32)) for _ in range(2))
        self.table_h = np.ascontiguousarray(table, np.int32)
        self.table = jas.to_device(self.table_h)
        self.plain = {n: np.full(self.shape, fill, np.float64) for n in "kv"}
        self.view = jas.PagedKv(self.k.ptr, self.v.ptr, self.ks.ptr if self.ks else None, self.vs.ptr if self.vs else None, self.table.ptr,
                                *self.strides, self.table_h.shape[1], self.table_h.shape[1], dtype, pages, page, heads, dh)

    @property
    def ref(self):
        return C.byref(self.view)

    def slots(self, cu, lens):
        """(row, page, slot) of every row of the batch that has a place."""
        page, cap = self.shape[2], self.table_h.shape[1] * self.shape[2]
        for b in range(len(lens)):
            for i in range(cu[b], cu[b + 1]):
                t = lens[b] - cu[b + 1] + i
                if 0 <= t < cap and 0 <= self.table_h[b, t // page] < self.shape[0]:
                    yield i, self.table_h[b, t // page], t % page

    def put(self, k, v, cu, lens):
        """The plain copy's append of fp32 rows k, v [n, heads, dh]."""
        for name, x in (("k", k), ("v", v)):
            if self.dtype in QMAX:
                t, s = stored(x, self.dtype)
                t = t * s.astype(np.float64)[..., None]
            else:
                t = from_bf16(to_bf16(x)) if self.dtype == BF16 else x
            for i, pg, sl in self.slots(cu, lens):
                self.plain[name][pg, :, sl] = t[i]

    def rows(self, b, n):
        """Keys and values of positions below n of sequence b, and which of them have a page."""
        t = np.arange(n)
        pg = self.table_h[b, t // self.shape[2]]
        ok = (pg >= 0) & (pg < self.shape[0])
        pg = np.where(ok, pg, 0)
        return self.plain["k"][pg, :, t % self.shape[2]], self.plain["v"][pg, :, t % self.shape[2]], ok


def attention(cache, q, cu, lens, scale, causal, n_rows, rss=None):
    """Rows of the batch in 64 bits: (o, sum of p |v|, largest sum of |q||k| scale of a row).
    rss: an array of o's shape for the root of the sum of (p v)^2."""
    H, D = q.shape[1:]
    g = H // cache.shape[1]
    o, mag, big = np.full((n_rows, H, D), np.nan), np.zeros((n_rows, H, D)), np.zeros((n_rows, H, 1))
    cap = cache.table_h.shape[1] * cache.shape[2]
    for b in range(len(lens)):
        L = min(lens[b], cap)
        if cu[b + 1] == cu[b]:
            continue
        k, v, ok = cache.rows(b, L)
        new = cu[b + 1] - cu[b]
        for i in range(new):
            pos = L - new + i
            n = max(0, min(L, pos + 1)) if causal else L
            see = np.flatnonzero(ok[:n])
            for h in range(H):
                kk, vv = k[see, h // g], v[see, h // g]
                qq = q[cu[b] + i, h].astype(np.float64)
                if len(see) == 0:
                    o[cu[b] + i, h] = 0
                    continue
                with np.errstate(all="ignore"):
                    s = kk @ qq * scale
                    p = np.exp(s - s.max())
                    l = p.sum()
                    o[cu[b] + i, h], mag[cu[b] + i, h] = p @ vv / l, p @ np.abs(vv) / l
                    if rss is not None:
                        rss[cu[b] + i, h] = np.sqrt((p / l) ** 2 @ vv ** 2)
                    big[cu[b] + i, h] = (np.abs(kk) @ np.abs(qq)).max() * abs(scale)
    return o, mag, big


def rope(x, pos, freq, mscale, rot, halves):
    """x [n, heads, dh] in 64 bits."""
    x = x.astype(np.float64)
    y = x.copy()
    a = pos.astype(np.float64)[:, None] * freq
    c, s = (np.cos(a) * mscale)[:, None], (np.sin(a) * mscale)[:, None]
    i = np.arange(rot // 2) if halves else np.arange(0, rot, 2)
    j = i + (rot // 2 if halves else 1)
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., i] * s + x[..., j] * c
    return y


def sample(x, temp, top_k, top_p, min_p, u):
    """(id, log of its share) of one row, by the definition."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, -np.inf
    if not temp > 0:
        return int(np.argmax(x)), 0.0
    order = np.argsort(-x, kind="stable")
    if 0 < top_k < len(x):
        order = order[:top_k]
    top = x[order[0]]
    with np.errstate(all="ignore"):
        w = np.where(x[order] == top, 1.0, 0.0) if np.isinf(top) else np.exp((x[order] - top) / temp)
    w = np.where(np.isnan(w), 0.0, w)
    if top_p < 1:
        count = max(1, 1 + int(np.searchsorted(np.cumsum(w), top_p * w.sum(), side="left")))
        order, w = order[:count], w[:count]
    keep = w >= (min(min_p, 1.0) if min_p > 0 else 0.0)
    order, w = order[keep], w[keep]
    by = np.argsort(order)
    order, w = order[by], w[by]
    upto = np.cumsum(w)
    u = min(max(u, 0.0), 1 - 2.0 ** -24) if u == u else 0.0
    k = int(np.searchsorted(upto, u * upto[-1], side="right"))
    return int(order[k]), math.log(w[k] / upto[-1])


class Hip:
    """Streams and graphs of the HIP runtime that the library runs on."""

    def __init__(self):
        with open("/proc/self/maps") as f:
            path = next(line.split()[-1] for line in f if "libamdhip64" in line)
        self.lib = C.CDLL(path)

    def __call__(self, name, *args):
        rc = getattr(self.lib, name)(*args)
        assert rc == 0, (name, rc)

    def stream(self):
        s = C.c_void_p()
        self("hipStreamCreateWithFlags", C.byref(s), C.c_uint(1))  # non-blocking, default priority
        return s

    def capture(self, stream, work):
        """The launches that work() makes on `stream`, as a graph that can be launched."""
        self("hipStreamBeginCapture", stream, C.c_int(1))  # (calls of other threads may go on)
        work()
        graph, ready = C.c_void_p(), C.c_void_p()
        self("hipStreamEndCapture", stream, C.byref(graph))
        self("hipGraphInstantiate", C.byref(ready), graph, None, None, C.c_size_t(0))
        self("hipGraphDestroy", graph)
        return ready
