"""Plain restatements of the paged cache's rules (include/janas_attn.h, Part 4)
in numpy, in 64 bits, and the pools that the tests make."""
import math

import numpy as np

KV_I8, KV_I16, KV_F16, KV_F32 = 0, 1, 2, 3
DTYPE = {KV_I8: np.int8, KV_I16: np.int16, KV_F16: np.float16, KV_F32: np.float32}
TOP = {KV_I8: 127.0, KV_I16: 32767.0}
NONE = -1


def blocks(n, page):
    return -(-n // page)


def plan(table, free, n_free, lens, n_new, page, max_tokens):
    """janas_attn_pages_plan, sequence after sequence. Returns a dict of what it
    writes; table and free are copies."""
    table, free = table.copy(), free.copy()
    lens, news = [int(x) for x in lens], [int(x) for x in n_new]
    n_pages, room = len(free), table.shape[1] * page
    top = min(int(n_free), n_pages)
    for i, x in enumerate(news):
        if x == NONE:
            b = min(blocks(lens[i], page), table.shape[1])
            m = min(b, n_pages - top)
            free[top:top + m] = table[i, :m]
            top, lens[i], news[i] = top + m, 0, 0
    slot = np.full(max_tokens, NONE, np.int32)
    pos, seq = np.zeros(max_tokens, np.int32), np.zeros(max_tokens, np.int32)
    granted, start, taken, asked, at = [], [0], [0], 0, top
    for i, x in enumerate(news):
        t0 = start[-1]
        start.append(t0 + x)
        seq[min(t0, max_tokens):t0 + x] = i
        b0, b1 = blocks(lens[i], page), blocks(lens[i] + x, page)
        fits = lens[i] + x <= room and t0 + x <= max_tokens
        asked += b1 - b0 if fits else 0
        if not fits or (b1 > b0 and asked > top):
            granted.append(0)
            taken.append(taken[-1])
            continue
        for b in range(b0, b1):
            at -= 1
            table[i, b] = free[at]
        for t in range(x):
            p = lens[i] + t
            pos[t0 + t] = p
            slot[t0 + t] = table[i, p // page] * page + p % page
        granted.append(x)
        taken.append(taken[-1] + b1 - b0)
        lens[i] += x
    a = lambda x: np.array(x, np.int32)  # noqa: E731
    return dict(table=table, free=free, n_free=a([at]), length=a(lens), granted=a(granted),
                start=a(start), taken=a(taken), slot=slot, pos=pos, seq=seq)


def quantize(x, kv):
    """Rows at 8 or 16 bits with a scale each (the cache write's rule)."""
    top = np.float32(TOP[kv])
    mx = np.abs(x).max(-1).astype(np.float32)
    inv = np.where(mx > 0, top / np.where(mx > 0, mx, 1), np.float32(0)).astype(np.float32)
    return np.rint(x * inv[..., None]).astype(DTYPE[kv]), (mx / top).astype(np.float32)


class Pool:
    """A pool with sequences of `lens` positions in shuffled pages. What no
    sequence holds - free pages, rows past a sequence's end, table entries past
    its blocks - is filled with what must not be used: NaN where the type has
    it, the largest numbers and NaN scales where not, entries far outside."""

    def __init__(self, rng, kv, lens, page, n_kv, hd, spare=3, extra=2, key_shift=0.0):
        self.kv, self.lens, self.page, self.n_kv, self.hd = kv, list(lens), page, n_kv, hd
        need = [blocks(n, page) for n in lens]
        self.n_pages = sum(need) + spare
        order = rng.permutation(self.n_pages).astype(np.int32)
        self.table = np.full((len(lens), max(need) + extra), 0x7FFFFFF0, np.int32)
        self.n_free = spare
        self.free = np.full(self.n_pages, 0x7FFFFFF0, np.int32)
        self.free[:spare] = order[:spare]
        shape = (self.n_pages, n_kv, page, hd)
        self.ks = self.vs = None
        bad = np.nan if kv in (KV_F16, KV_F32) else (127 if kv == KV_I8 else 32767)
        self.k, self.v = (np.full(shape, bad, DTYPE[kv]) for _ in range(2))
        if kv in TOP:
            self.ks, self.vs = (np.full(shape[:3], np.nan, np.float32) for _ in range(2))
        at = spare
        for i, n in enumerate(lens):
            self.table[i, :need[i]] = order[at:at + need[i]]
            at += need[i]
            if n == 0:
                continue
            x = rng.standard_normal((2, n, n_kv, hd)).astype(np.float32)
            # neighbouring keys alike, so that blocks differ
            drift = rng.standard_normal((need[i], n_kv, hd)).astype(np.float32)
            x[0] += key_shift * np.repeat(drift, page, axis=0)[:n]
            for p in range(n):
                pg, r = self.table[i, p // page], p % page
                for dst, z, y in ((self.k, self.ks, x[0, p]), (self.v, self.vs, x[1, p])):
                    if kv in TOP:
                        dst[pg, :, r], z[pg, :, r] = quantize(y, kv)
                    else:
                        dst[pg, :, r] = y.astype(DTYPE[kv])

    def rows(self, which, i, n=None):
        """Sequence i's first n rows in 64 bits: (n, n_kv, hd)."""
        n = self.lens[i] if n is None else n
        p = np.arange(n)
        pg, r = self.table[i, p // self.page], p % self.page
        x = (self.k if which == "k" else self.v)[pg, :, r].astype(np.float64)
        z = self.ks if which == "k" else self.vs
        return x if z is None else x * z[pg, :, r].astype(np.float64)[..., None]


def sigmoid(x):
    return 1.0 / (1.0 + np.exp(-np.asarray(x, np.float64)))


def attend(q, k, v, scale, seen):
    """One token's (h, hd) attention of k, v (n, n_kv, hd), where seen[kv head]
    are positions (they may repeat); and how far f32-accurate arithmetic may be
    from it. Bound: a score's error dx (in units of the exponent) is the query's
    second plane's rounding, 2^-23 of each product, f32 sums over the head
    dimension in products of 16 at least and two plane sums, (hd / 16 + 8)
    2^-23 of the sum of the products' sizes, and the roundings of the scaled
    score and of the exponential, 8 x 2^-24 of 1 + its size (log2 e and the key
    scale among them); a weight's second plane and the value scale 2^-22. A
    weighted mean moves by at most 2 (dx + ...) of the largest value, and the
    sums of n weights and products by (n / 16 + 32) 2^-23 of it: a unit of 16
    positions is one addition."""
    h, hd = q.shape
    g = h // k.shape[1]
    out, bar = np.zeros((h, hd)), np.zeros(h)
    for i in range(h):
        p = np.asarray(seen[i // g], np.int64)
        if len(p) == 0:
            continue
        kk, vv = k[p, i // g], v[p, i // g]
        qi = q[i].astype(np.float64)
        x = scale * (kk @ qi)
        size = abs(scale) * (np.abs(kk) @ np.abs(qi)).max()
        w = np.exp(x - x.max())
        out[i] = (w @ vv) / w.sum()
        dx = size * (hd / 16 + 9) * 2.0 ** -23 + (1 + np.abs(x).max()) * 2.0 ** -21 + 2.0 ** -22
        bar[i] = np.abs(vv).max() * (2 * dx + (len(p) / 16 + 32) * 2.0 ** -23)
    return out, bar


def in_sight(n, window):
    return np.arange(max(0, n - window) if window else 0, n)


def outward(x, up):
    """Halves not inside of x, within their range."""
    x = np.clip(x.astype(np.float64), -65504, 65504)
    h = x.astype(np.float16)
    short = h.astype(np.float64) < x if up else h.astype(np.float64) > x
    with np.errstate(over="ignore"):
        return np.where(short, np.nextafter(h, np.float16(np.inf if up else -np.inf)), h)


def key_bounds(pool, i, b):
    """(n_kv, 2, hd) halves: block b of sequence i, of the f32 numbers."""
    k = pool.rows("k", i)[b * pool.page:(b + 1) * pool.page].astype(np.float32)
    with np.errstate(all="ignore"):
        lo = np.fmin.reduce(k, axis=0, initial=np.inf)
        hi = np.fmax.reduce(k, axis=0, initial=-np.inf)
    return np.stack((outward(lo, False), outward(hi, True)), 1)


def choose(q, boxes, n, window, page, n_sel, first, last):
    """One KV head's blocks: q (g, hd), boxes (blocks, 2, hd)."""
    row = np.full(n_sel, NONE, np.int32)
    if n == 0:
        return row
    b0, nb = (max(0, n - window) // page if window else 0), blocks(n, page)
    if nb - b0 <= n_sel:
        row[:nb - b0] = np.arange(b0, nb)
        return row
    q = q.astype(np.float64)
    box = boxes.astype(np.float64)
    score = np.maximum(q, 0) @ box[:, 1].T + np.minimum(q, 0) @ box[:, 0].T
    score = score.max(0).astype(np.float32)
    forced = list(range(b0, b0 + first)) + list(range(nb - last, nb))
    rest = [b for b in range(b0 + first, nb - last)]
    rest.sort(key=lambda b: (-score[b], b))
    row[:] = sorted(forced + rest[:n_sel - first - last])
    return row


def rotation(n_tab, n_rot, base=1e6):
    half = max(n_rot // 2, 1)
    ang = np.outer(np.arange(n_tab), base ** (-2.0 * np.arange(half) / max(n_rot, 2)))
    return (np.cos(ang).astype(np.float32), np.sin(ang).astype(np.float32))


def default_scale(hd):
    return float(np.float32(1.0) / np.float32(math.sqrt(hd)))
