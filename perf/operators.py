"""The operators of a paged KV cache whose speed is measured, through the
package's public entry points (``own`` true) and in their plain form.

A case is one of four kinds:

  plan    a serving step's pages and slots from the sequences' lengths
          (``pages_plan``): block tables, slot map, free list, releases
  write   the step's key and value rows, normalized, turned and quantized, into
          their slots, and its query rows (``pages_write``)
  decode  attention of one new token of every sequence over its pages
          (``Attention.run_pages``)
  sparse  the key bounds of the blocks that changed, the blocks each KV head's
          queries select, and the attention over those (``pages_bounds``,
          ``Attention.select``, ``Attention.run_pages``); ``attend`` false:
          without the attention

Head shapes, cache types and lengths are the ones of the repository's benchmark
and tests (32 / 8 / 128, 16 / 2 / 256, 16 / 2 / 512 ...). All calls go to the
default stream.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda:0"
DTYPE = {"i8": torch.int8, "i16": torch.int16, "f16": torch.float16,
         "f32": torch.float32}
KIND = {"i8": 0, "i16": 1, "f16": 2, "f32": 3}
BYTES = {"i8": 1, "i16": 2, "f16": 2, "f32": 4}
TOP = {"i8": 127.0, "i16": 32767.0}
# head shapes (query heads, KV heads, head size)
HEADS = ((32, 8, 128), (32, 4, 128), (12, 4, 64), (16, 2, 256), (16, 4, 256))
WIDE = (16, 2, 512)
PAGES = (16, 32, 64, 128)
RELEASE = -1
MOST_BYTES = 1.05e9
TABLE_ROWS = 40960        # positions of the rotation's table


def _case(kind, **more):
    c = dict(kind=kind, h=32, n_kv=8, hd=128, kv="f16", page=64, seqs=1,
             length=1024, new=1, even=False, release=0, spare=64, pad=0,
             window=0, gate=False, n_sel=0, first=1, last=1, attend=True,
             fresh=1)
    c.update(more)
    return c


def listed():
    return [
        # the smallest: a decode step's bookkeeping for 48 users
        _case("plan", seqs=48, length=6000, name="plan-decode-48"),
        # prompts of unlike lengths admitted in one step, in small pages, while
        # five finished users give theirs back
        _case("plan", seqs=61, length=4000, new=1400, release=5, page=16,
              spare=4500, name="plan-prompts-61"),
        # a decode step's rows: 64 users' new token over the engine's int8 cache
        _case("write", seqs=64, length=4000, kv="i8", name="write-decode-64-i8"),
        # a packed batch of prompts' rows, large heads
        _case("write", h=16, n_kv=2, hd=256, seqs=7, length=8000, new=900,
              page=32, pad=33, name="write-prompts-f16"),
        # one user at a short context: latency
        _case("decode", kv="i8", page=16, length=1023, name="decode-1k-i8"),
        # a serving step of a gated layer: users at unlike lengths
        _case("decode", seqs=24, length=16000, gate=True,
              name="decode-ragged24-gated-f16"),
        # a full batch: the largest
        _case("decode", seqs=60, length=4170, page=32, even=True,
              name="decode-60x4k-f16"),
        # a long document with the widest heads over a 16-bit integer cache
        _case("decode", h=16, n_kv=2, hd=512, kv="i16", page=128, length=90000,
              name="decode-90k-hd512-i16"),
        # a sliding-window layer over a float cache
        _case("decode", h=16, n_kv=4, hd=256, kv="f32", seqs=9, length=20000,
              window=1024, name="decode-window-f32"),
        # one user far into a document: 64 of 2000 blocks attended
        _case("sparse", length=127931, n_sel=64, last=2, name="sparse-128k-f16"),
        # a batch over the engine's int8 cache: a sixteenth of it attended
        _case("sparse", seqs=16, length=32000, kv="i8", page=32, n_sel=64,
              last=4, name="sparse-16x32k-i8"),
        # prompts just written: their blocks' bounds made, the first selection
        _case("sparse", h=16, n_kv=2, hd=256, seqs=5, length=24000, n_sel=40,
              attend=False, fresh=6000, name="select-prompts-f16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    while True:
        c = _draw(rng)
        # (the pool itself, its rows in 32 bits, is made each time)
        if work(c)["bytes"] <= MOST_BYTES and \
                (c["kind"] == "plan" or _pool_bytes(c) <= 2 * MOST_BYTES):
            return c


def _draw(rng):
    kind = rng.choice(("plan", "write", "decode", "decode", "sparse"))
    seqs = _log(rng, 1, 100)
    page = rng.choice(PAGES)
    if kind == "plan":
        decode = rng.random() < 0.5
        return _case("plan", seqs=_log(rng, 1, 400), page=page,
                     length=_log(rng, 20, 30000), new=1 if decode else _log(rng, 2, 2000),
                     release=rng.choice((0, 0, 1, 3)),
                     spare=rng.choice((0, 5, 64, 4000)), even=rng.random() < 0.2)
    h, n_kv, hd = rng.choice(HEADS)
    kv = rng.choice(("f16", "f16", "i8", "i8", "i16", "f32"))
    if kind == "write":
        new = 1 if rng.random() < 0.5 else _log(rng, 2, 1500)
        return _case("write", h=h, n_kv=n_kv, hd=hd, kv=kv, page=page,
                     seqs=seqs if new == 1 else _log(rng, 1, 12),
                     length=_log(rng, 20, 16000), new=new, pad=rng.choice((0, 0, 3, 40)),
                     even=rng.random() < 0.2)
    if kind == "decode":
        if kv != "f32" and rng.random() < 0.2:
            h, n_kv, hd = WIDE
        return _case("decode", h=h, n_kv=n_kv, hd=hd, kv=kv, page=page, seqs=seqs,
                     length=_log(rng, 1, 100000), even=rng.random() < 0.3,
                     gate=rng.random() < 0.4, window=rng.choice((0, 0, 0, 1024)))
    length = _log(rng, 200, 130000)
    blocks = -(-length // page)
    first, last = rng.choice((0, 1, 2)), rng.choice((1, 1, 4))
    return _case("sparse", h=h, n_kv=n_kv, hd=hd, kv=kv, page=page,
                 seqs=_log(rng, 1, 24), length=length, first=first, last=last,
                 n_sel=max(first + last, min(_log(rng, 4, 256), blocks)),
                 fresh=rng.choice((1, 1, 1, 700)), attend=rng.random() < 0.8,
                 even=rng.random() < 0.3)


def _lengths(c):
    """Positions in the cache of each sequence."""
    n = c["seqs"]
    if c["even"] or n == 1:
        return [c["length"]] * n
    # spread over [1/12, 1] of the longest, in no order
    p = c["length"]
    return [max(1, p // 12 + (p - p // 12) * ((i * 37 + 11) % n) // max(1, n - 1))
            for i in range(n)]


def _news(c):
    """New tokens of each sequence in a step (RELEASE: finished)."""
    n, w = c["seqs"], c["new"]
    if w == 1:
        res = [1] * n
        for i in range(2, n, 7):
            res[i] = 0          # waits this step
    else:
        res = [1 + (w * ((i * 23 + 5) % 9)) // 4 if i % 3 else i % 2 for i in range(n)]
        res[0] = w
    for i in range(c["release"]):
        res[(3 * i + 1) % n] = RELEASE
    return res


def _blocks(length, page):
    return -(-length // page)


def _row(c):
    """Bytes of a position's keys and values."""
    return 2 * c["n_kv"] * (c["hd"] * BYTES[c["kv"]] + (4 if c["kv"] in TOP else 0))


def _pool_bytes(c):
    return sum(_blocks(n, c["page"]) for n in _lengths(c)) * c["page"] * _row(c)


def _seen(c):
    """Positions that each sequence's token sees."""
    return [min(n, c["window"]) if c["window"] else n for n in _lengths(c)]


def work(case):
    c = case
    h, n_kv, hd, page = c["h"], c["n_kv"], c["hd"], c["page"]
    lens = _lengths(c)
    if c["kind"] == "plan":
        news = _news(c)
        tokens = sum(max(0, x) for x in news)
        took = sum(_blocks(n + x, page) - _blocks(n, page)
                   for n, x in zip(lens, news) if x > 0)
        gave = sum(_blocks(n, page) for n, x in zip(lens, news) if x < 0)
        return {"bytes": 12.0 * tokens + 8.0 * (took + gave) + 24.0 * len(lens), "flops": 0.0}
    if c["kind"] == "write":
        t = sum(x for x in _news(c) if x > 0)
        return {"bytes": float(t) * (4 * hd * 2 * (n_kv + h) + 4 * hd + _row(c) + 8),
                "flops": 9.0 * t * hd * (h + 2 * n_kv)}
    total = flops = 0.0
    attended = _seen(c)
    if c["kind"] == "sparse":
        for n in lens:
            b = _blocks(n, page)
            changed = b - max(0, n - c["fresh"]) // page
            rows = changed * page * n_kv * (hd * BYTES[c["kv"]] + (4 if c["kv"] in TOP else 0))
            total += rows + changed * n_kv * 4 * hd
            flops += 2.0 * changed * page * n_kv * hd
            total += b * n_kv * 4 * hd + 4 * n_kv * c["n_sel"] + 4 * h * hd
            flops += 2.0 * b * h * hd
        attended = [min(n, c["n_sel"] * page) for n in lens]
        if not c["attend"]:
            return {"bytes": total, "flops": flops}
    for n in attended:
        total += n * _row(c) + 2 * 4 * h * hd + (4 * h * hd if c["gate"] else 0)
        flops += 4.0 * hd * h * n
    return {"bytes": total, "flops": flops}


# ---- inputs ---------------------------------------------------------------

def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed((int(seed) * 1000003 + salt) & 0x7FFFFFFF)
    return g


def _randn(seed, salt, *shape):
    return torch.randn(*shape, generator=_gen(seed, salt), device=DEV)


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _quant(x, kv):
    """Rows at 8 or 16 bits with a scale each, as the cache write makes them:
    the multiplier and the scale are one quotient each, rounded once. (A number
    over a tensor is the number times the reciprocal, rounded twice, and so on
    the GPU is a tensor over a number: quotients of two tensors.)"""
    mx = x.abs().amax(-1)
    top = torch.full_like(mx, TOP[kv])
    inv = torch.where(mx > 0, top / mx, torch.zeros_like(mx))
    return torch.round(x * inv[..., None]).to(DTYPE[kv]), mx / top


def _pool(c, seed, n_pages):
    """A resident pool: k, v (n_pages, n_kv, page, hd), ks, vs or None. A page's
    keys share a direction, as neighbouring tokens' do."""
    res = []
    for i in range(2):
        shape = (n_pages, c["n_kv"], c["page"], c["hd"])
        x = _randn(seed, 10 + i, *shape)
        if i == 0:
            x += _randn(seed, 12, n_pages, c["n_kv"], 1, c["hd"])
        if c["kv"] in TOP:
            res += list(_quant(x, c["kv"]))
        else:
            res += [x.to(DTYPE[c["kv"]]), None]
        del x
    return dict(k=res[0], ks=res[1], v=res[2], vs=res[3])


def _tables(c, seed, lens, extra=0):
    """Block tables over a shuffled pool (rows as long as the longest, plus
    `extra` blocks), the free pages, and how many there are."""
    page = c["page"]
    need = [_blocks(n, page) for n in lens]
    width = max(need) + extra
    n_pages = sum(need) + c["spare"]
    order = torch.randperm(n_pages, generator=_gen(seed, 5), device=DEV).int()
    table = torch.zeros(len(lens), width, dtype=torch.int32, device=DEV)
    at = 0
    for i, b in enumerate(need):
        table[i, :b] = order[at:at + b]
        at += b
    free = torch.zeros(n_pages, dtype=torch.int32, device=DEV)
    free[:n_pages - at] = order[at:]
    return table, free, n_pages - at, n_pages


def _rotation(c):
    half = c["hd"] // 2
    f = 1e6 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)
    a = torch.arange(TABLE_ROWS, dtype=torch.float64, device=DEV)[:, None] * f
    return a.cos().float().contiguous(), a.sin().float().contiguous()


def _prepare_plan(c, seed):
    lens, news = _lengths(c), _news(c)
    # rows of the table with room for the step, for all but the longest
    grow = max(0, _blocks(max(lens) + max(1, c["new"] // 2), c["page"]) -
               _blocks(max(lens), c["page"]))
    table, free, n_free, n_pages = _tables(c, seed, lens, grow)
    t = sum(max(0, x) for x in news)
    cap = t + 7                         # the step's buffers hold a few more
    return dict(case=c, table=table, free=free, n_free=_ints([n_free]),
                length=_ints(lens), n_new=_ints(news), cap=cap,
                out=dict(length=_ints(lens), n_free=_ints([0]),
                         granted=_ints([0] * len(lens)),
                         start=_ints([0] * (len(lens) + 1)),
                         taken=_ints([0] * (len(lens) + 1)),
                         slot=_ints([0] * cap), pos=_ints([0] * cap),
                         seq=_ints([0] * cap)))


def _prepare_write(c, seed):
    h, n_kv, hd, page = c["h"], c["n_kv"], c["hd"], c["page"]
    lens = _lengths(c)
    news = [max(0, x) for x in _news(c)]
    table, _, _, n_pages = _tables(c, seed, [n + x for n, x in zip(lens, news)])
    pool = _pool(c, seed, n_pages)
    rows = table.cpu()
    slot, pos = [], []
    for i, (n, x) in enumerate(zip(lens, news)):
        for p in range(n, n + x):
            slot.append(int(rows[i, p // page]) * page + p % page)
            pos.append(p % TABLE_ROWS)
    live, t = len(slot), len(slot) + c["pad"]
    slot += [-1] * c["pad"]
    pos += [0] * c["pad"]
    cs, sn = _rotation(c)
    s = dict(case=c, pool=pool, slot=_ints(slot), pos=_ints(pos), live=live,
             cs=cs, sn=sn, q=2.0 * _randn(seed, 30, t, h, hd),
             k=1.5 * _randn(seed, 31, t, n_kv, hd), v=_randn(seed, 32, t, n_kv, hd),
             qn=1.0 + 0.2 * _randn(seed, 33, hd), kn=1.0 + 0.2 * _randn(seed, 34, hd),
             table=table, length=_ints(lens))
    s["q_out"] = torch.zeros_like(s["q"])
    return s


def _prepare_attend(c, seed):
    h, hd = c["h"], c["hd"]
    lens = _lengths(c)
    table, _, _, n_pages = _tables(c, seed, lens)
    # some heads sharper than others
    sharp = 1.0 + torch.arange(h, device=DEV) % 4 * 0.5
    s = dict(case=c, pool=_pool(c, seed, n_pages), lens=lens, table=table,
             length=_ints(lens), q=_randn(seed, 20, len(lens), h, hd) * sharp[:, None],
             gate=_randn(seed, 21, len(lens), h, hd) if c["gate"] else None)
    s["out"] = torch.zeros_like(s["q"])
    if c["kind"] == "sparse":
        s["n_new"] = _ints([min(n, c["fresh"]) for n in lens])
        s["bounds"] = torch.zeros(n_pages, c["n_kv"], 2, hd, dtype=torch.float16, device=DEV)
        # the blocks that no token of the step touched have theirs
        _bounds(s, [(0, max(0, n - c["fresh"]) // c["page"]) for n in lens])
        s["sel"] = torch.zeros(len(lens), c["n_kv"], c["n_sel"], dtype=torch.int32, device=DEV)
    return s


def prepare(case, seed):
    c = case
    s = {"plan": _prepare_plan, "write": _prepare_write}.get(c["kind"], _prepare_attend)(c, seed)
    if own:
        s["calls"] = _calls(s)
    torch.cuda.synchronize()
    return s


# ---- the framework's calls --------------------------------------------------

def _calls(s):
    """The case's calls with their arguments built once, as a program that
    makes them every step keeps them."""
    import janas_amd as jm
    from janas_amd import attention as at

    c = s["case"]
    if c["kind"] == "plan":
        pool = at.page_tables(s["table"], s["length"], page=c["page"], free=s["free"],
                              n_free=s["n_free"])
        o = s["out"]
        return [at.prepare_pages_plan(
            pool, s["n_new"], slot=o["slot"], pos=o["pos"], seq=o["seq"], start=o["start"],
            granted=o["granted"], taken=o["taken"], length=o["length"], n_free=o["n_free"])]
    p = s["pool"]
    pool = at.pages(p["k"], p["v"], p["ks"], p["vs"], kv_type=KIND[c["kv"]], table=s["table"],
                    length=s["length"], bounds=s.get("bounds"))
    if c["kind"] == "write":
        return [at.prepare_pages_write(
            pool, s["k"], s["v"], slot=s["slot"], pos=s["pos"], cs=s["cs"], sn=s["sn"],
            n_rot=c["hd"], k_norm=s["kn"], q=s["q"], q_out=s["q_out"], q_norm=s["qn"])]
    a = jm.Attention(c["h"], c["n_kv"], c["hd"], 256, 1, jm.FLOAT)
    if c["window"]:
        a.set_window(c["window"])
    s["a"] = a
    n_work = a.pages_work_bytes(pool)
    s["work"] = torch.empty(n_work, dtype=torch.uint8, device=DEV)
    calls, sel = [], None
    if c["kind"] == "sparse":
        sel = s["sel"]
        calls += [at.prepare_pages_bounds(pool, s["n_new"], max_new=c["fresh"]),
                  a.prepare_select(pool, s["q"], sel, first=c["first"], last=c["last"],
                                   work=s["work"])]
    if c["attend"]:
        calls.append(a.prepare_pages(
            pool, s["q"], s["out"], gate=s["gate"],
            gate_mode=jm.GATE_ELEM if c["gate"] else jm.GATE_NONE, sel=sel, work=s["work"]))
    return calls


def run(state):
    s, c = state, state["case"]
    if own:
        for call in s["calls"]:
            call()
    elif c["kind"] == "plan":
        return _plain_plan(s)
    elif c["kind"] == "write":
        _plain_write(s)
    else:
        if c["kind"] == "sparse":
            _bounds(s, [(max(0, n - c["fresh"]) // c["page"], _blocks(n, c["page"]))
                        for n in s["lens"]])
            s["sel"] = _plain_select(s)
        if c["attend"]:
            s["out"] = _plain_attend(s)
    if c["kind"] == "plan":
        o = s["out"]
        return [s["table"], s["free"], o["n_free"], o["length"], o["granted"], o["start"],
                o["taken"], o["slot"], o["pos"], o["seq"]]
    if c["kind"] == "write":
        p = s["pool"]
        return [x for x in (p["k"], p["v"], p["ks"], p["vs"], s["q_out"]) if x is not None]
    res = [s["bounds"], s["sel"]] if c["kind"] == "sparse" else []
    return res + ([s["out"]] if c["attend"] else [])


# ---- the plain forms --------------------------------------------------------

def _plain_plan(s):
    c, page = s["case"], s["case"]["page"]
    table, free, cap = s["table"], s["free"], s["cap"]
    n_seqs, width = table.shape
    old, new = s["length"].long(), s["n_new"].long()
    b = torch.arange(width, device=DEV)
    gone = new == RELEASE
    # released pages go on top of the free ones, in the sequences' order
    gave = torch.where(gone, (old + page - 1) // page, 0)
    at = s["n_free"].long() + gave.cumsum(0) - gave
    dest = torch.where(b < gave[:, None], at[:, None] + b, len(free))
    stack = torch.cat((free, free.new_zeros(1)))
    stack.scatter_(0, dest.flatten(), table.flatten())
    top = s["n_free"].long() + gave.sum()
    old, new = torch.where(gone, 0, old), torch.where(gone, 0, new)
    end = new.cumsum(0)
    start = end - new
    have = (old + page - 1) // page
    fits = (old + new <= width * page) & (end <= cap)
    need = torch.where(fits, (old + new + page - 1) // page - have, 0)
    ok = fits & ((need == 0) | (need.cumsum(0) <= top))
    need, granted = torch.where(ok, need, 0), torch.where(ok, new, 0)
    taken = need.cumsum(0) - need
    k = b - have[:, None]
    fresh = (k >= 0) & (k < need[:, None])
    pick = (top - 1 - taken[:, None] - k).clamp(0, len(free) - 1)
    table2 = torch.where(fresh, stack[pick], table)
    t = torch.arange(cap, device=DEV)
    seq = torch.searchsorted(end, t, right=True)
    live = seq < n_seqs
    seq = torch.where(live, seq, 0)
    live = live & ok[seq]
    pos = torch.where(live, old[seq] + t - start[seq], 0)
    slot = table2[seq, pos // page].long() * page + pos % page
    zero = new.new_zeros(1)
    i32 = lambda x: x.to(torch.int32)  # noqa: E731
    return [table2, stack[:-1], i32(top - need.sum()).reshape(1), i32(old + granted),
            i32(granted), i32(torch.cat((zero, end))), i32(torch.cat((zero, need.cumsum(0)))),
            i32(torch.where(live, slot, -1)), i32(pos),
            i32(torch.where(t < end[-1], seq, 0))]


def _norm32(x, w):
    """The root mean square norm: squares summed in 64 bits, the rest in 32."""
    ms = x.double().square().sum(-1, keepdim=True) / x.shape[-1]
    inv = 1.0 / torch.sqrt(ms.float() + torch.tensor(1e-6, device=DEV))
    return x * inv * w


def _turn(x, cs, sn):
    half = x.shape[-1] // 2
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cs - b * sn, a * sn + b * cs), -1)


def _plain_write(s):
    c, n, p = s["case"], s["live"], s["pool"]
    at = s["pos"][:n].long()
    cs, sn = s["cs"][at][:, None], s["sn"][at][:, None]
    s["q_out"][:n] = _turn(_norm32(s["q"][:n], s["qn"]), cs, sn)
    slot = s["slot"][:n].long()
    page, off = slot // c["page"], slot % c["page"]
    heads = torch.arange(c["n_kv"], device=DEV)
    at = (page[:, None], heads[None], off[:, None])
    for x, name, z in ((_turn(_norm32(s["k"][:n], s["kn"]), cs, sn), "k", "ks"),
                       (s["v"][:n], "v", "vs")):
        if c["kv"] in TOP:
            x, scale = _quant(x, c["kv"])
            p[z][at] = scale
        p[name][at] = x.to(DTYPE[c["kv"]])


def _numbers(p, which, scale, pages):
    """Cached rows of some pages in 32 bits."""
    x = p[which][pages].float()
    return x if p[scale] is None else x * p[scale][pages][..., None]


def _outward(x, up):
    """To f16, never inside of x."""
    h = x.clamp(-65504.0, 65504.0).half()
    short = h.float() < x if up else h.float() > x
    bits = h.view(torch.int16)
    away = (h > 0) if up else (h < 0)
    nxt = torch.where(away, bits + 1, bits - 1)
    # from zero the step is to the smallest number of that sign
    tiny = torch.full_like(bits, 1 if up else -32767)
    nxt = torch.where(h == 0, tiny, nxt)
    return torch.where(short & (h.abs() < 65504), nxt, bits).view(torch.float16)


def _bounds(s, spans):
    """The key bounds of blocks [b0, b1) of each sequence, into their pages."""
    c, page = s["case"], s["case"]["page"]
    for i, (b0, b1) in enumerate(spans):
        if b1 <= b0:
            continue
        pages = s["table"][i, b0:b1].long()
        x = _numbers(s["pool"], "k", "ks", pages)
        p = torch.arange(b0 * page, b1 * page, device=DEV).reshape(-1, 1, page, 1)
        unseen = p >= s["lens"][i]
        lo = x.masked_fill(unseen, math.inf).amin(2)
        hi = x.masked_fill(unseen, -math.inf).amax(2)
        s["bounds"][pages] = torch.stack((_outward(lo, False), _outward(hi, True)), 2)


def _plain_select(s):
    c, page, n_sel = s["case"], s["case"]["page"], s["case"]["n_sel"]
    n_kv, g = c["n_kv"], c["h"] // c["n_kv"]
    res = []
    for i, n in enumerate(s["lens"]):
        nb = _blocks(n, page)
        row = torch.full((n_kv, n_sel), -1, dtype=torch.int32, device=DEV)
        if nb <= n_sel:
            row[:, :nb] = torch.arange(nb, device=DEV)
            res.append(row)
            continue
        q = s["q"][i].reshape(n_kv, g, -1).double()
        box = s["bounds"][s["table"][i, :nb].long()].double()     # nb, n_kv, 2, hd
        lo, hi = (box[:, :, j].permute(1, 2, 0).contiguous() for j in (0, 1))
        score = q.clamp(min=0) @ hi + q.clamp(max=0) @ lo
        score = score.amax(1).float()
        score[:, :c["first"]] = math.inf
        score[:, nb - c["last"]:] = math.inf
        order = torch.sort(score, dim=-1, descending=True, stable=True).indices[:, :n_sel]
        res.append(torch.sort(order, dim=-1).values.int())
    return torch.stack(res)


def _plain_attend(s):
    """A padded batch at once: every sequence's rows gathered by its table (its
    selected blocks), masked past its length."""
    c, page, p = s["case"], s["case"]["page"], s["pool"]
    n_seqs, h, hd = s["q"].shape
    n_kv, g = c["n_kv"], h // c["n_kv"]
    lens = s["length"].long()
    heads = torch.arange(n_kv, device=DEV)[None, :, None]
    if c["kind"] == "sparse":
        blocks = s["sel"].long()
        known = blocks >= 0
        blocks = blocks.clamp(min=0)
    else:
        blocks = torch.arange(s["table"].shape[1], device=DEV).expand(n_seqs, n_kv, -1)
        known = torch.ones_like(blocks, dtype=torch.bool)
    pages = s["table"].long()[torch.arange(n_seqs, device=DEV)[:, None, None], blocks]
    pos = blocks[..., None] * page + torch.arange(page, device=DEV)
    seen = known[..., None] & (pos < lens[:, None, None, None])
    if c["window"]:
        seen &= pos + c["window"] >= lens[:, None, None, None]
    seen = seen.reshape(n_seqs, n_kv, 1, -1)

    def rows(which, scale):
        x = p[which][pages, heads].float()
        if p[scale] is not None:
            x = x * p[scale][pages, heads][..., None]
        return x.reshape(n_seqs, n_kv, -1, hd)
    k = rows("k", "ks")
    q = s["q"].reshape(n_seqs, n_kv, g, hd) * (1.0 / math.sqrt(hd))
    x = (q @ k.transpose(-1, -2).contiguous()).masked_fill_(~seen, -math.inf)
    del k
    w = torch.exp(x - x.amax(-1, keepdim=True))
    o = (w @ rows("v", "vs")) / w.sum(-1, keepdim=True)
    o = o.reshape(n_seqs, h, hd)
    if s["gate"] is not None:
        o = o * (1.0 / (1.0 + torch.exp(-s["gate"])))
    return o


# ---- from the definitions, in 64 bits ---------------------------------------

def exact(case, seed):
    c = case
    global own
    was, own = own, False
    try:
        s = prepare(c, seed)
    finally:
        own = was
    if c["kind"] == "plan":
        return _exact_plan(s)
    if c["kind"] == "write":
        return _exact_write(s)
    return _exact_attend(s)


def _exact_plan(s):
    """Sequence after sequence."""
    page, cap = s["case"]["page"], s["cap"]
    table, free = s["table"].cpu().numpy().copy(), s["free"].cpu().numpy().copy()
    lens, news = s["length"].tolist(), s["n_new"].tolist()
    room = table.shape[1] * page
    top = int(s["n_free"][0])
    for i, x in enumerate(news):
        if x == RELEASE:
            b = _blocks(lens[i], page)
            free[top:top + b] = table[i, :b]
            top, lens[i], news[i] = top + b, 0, 0
    slot, pos, seq = (np.full(cap, v, np.int32) for v in (-1, 0, 0))
    granted, start, taken, asked, at = [], [0], [0], 0, top
    for i, x in enumerate(news):
        t0 = start[-1]
        start.append(t0 + x)
        seq[t0:t0 + x] = i
        b0, b1 = _blocks(lens[i], page), _blocks(lens[i] + x, page)
        fits = lens[i] + x <= room and t0 + x <= cap
        asked += b1 - b0 if fits else 0
        if not fits or (b1 > b0 and asked > top):
            granted.append(0)
            taken.append(taken[-1])
            continue
        for b in range(b0, b1):
            at -= 1
            table[i, b] = free[at]
        p = np.arange(lens[i], lens[i] + x)
        pos[t0:t0 + x] = p
        slot[t0:t0 + x] = table[i, p // page] * page + p % page
        granted.append(x)
        taken.append(taken[-1] + b1 - b0)
        lens[i] += x
    arr = lambda x: np.array(x, np.int32)  # noqa: E731
    return [table, free, arr([at]), arr(lens), arr(granted), arr(start), arr(taken), slot, pos, seq]


def _exact_write(s):
    c, n, p = s["case"], s["live"], s["pool"]
    ang = s["pos"][:n].long()
    cs, sn = s["cs"].double()[ang], s["sn"].double()[ang]

    def turned(x, w):
        x = x.double()
        y = x / (x.pow(2).mean(-1, keepdim=True) + 1e-6).sqrt() * w.double()
        half = y.shape[-1] // 2
        z = torch.empty_like(y)
        z[..., :half] = y[..., :half] * cs[:, None] - y[..., half:] * sn[:, None]
        z[..., half:] = y[..., :half] * sn[:, None] + y[..., half:] * cs[:, None]
        return z
    q = torch.zeros_like(s["q"], dtype=torch.float64)
    q[:n] = turned(s["q"][:n], s["qn"])
    new = dict(k=turned(s["k"][:n], s["kn"]), v=s["v"][:n].double())
    page, off = (s["slot"][:n].long() // c["page"]), (s["slot"][:n].long() % c["page"])
    res, scales = [], []
    for name, z in (("k", "ks"), ("v", "vs")):
        x = new[name]
        if c["kv"] in TOP:
            top = torch.tensor(TOP[c["kv"]], dtype=torch.float64, device=DEV)
            mx = x.abs().amax(-1)
            full = p[z].double().transpose(1, 2).contiguous()
            full[page, off] = mx / top
            scales.append(full.transpose(1, 2))
            if name == "k":
                # whole numbers beside their scale: a tie's side is the 32-bit
                # arithmetic's, of the norm and the rotation too
                res.append(None)
                continue
            # the values' are the rule's own: a quotient and a product, each
            # rounded once to 32 bits (from 64, where either is near enough
            # exact), and the nearest whole number
            inv = torch.where(mx > 0, torch.full_like(mx, TOP[c["kv"]]) / mx, 0.0).float()
            full = p[name].transpose(1, 2).contiguous()
            full[page, off] = (x * inv.double()[..., None]).float().round().to(full.dtype)
            res.append(full.transpose(1, 2))
        else:
            full = p[name].double().transpose(1, 2).contiguous()
            full[page, off] = x
            res.append(full.transpose(1, 2))
    return res + scales + [q]


def _exact_attend(s):
    c, p, page = s["case"], s["pool"], s["case"]["page"]
    n_kv, g, hd = c["n_kv"], c["h"] // c["n_kv"], c["hd"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    bounds = s["bounds"].double() if c["kind"] == "sparse" else None
    sel = torch.full((len(s["lens"]), n_kv, max(1, c["n_sel"])), -1, dtype=torch.int32)
    for i, n in enumerate(s["lens"]):
        nb = _blocks(n, page)
        pages = s["table"][i, :nb].long()
        for kh in range(n_kv):
            at = torch.arange(n, device=DEV)
            if c["window"]:
                at = at[-c["window"]:]
            k32 = p["k"][pages, kh].reshape(-1, hd)[:n].double()
            if p["ks"] is not None:
                k32 = k32 * p["ks"][pages, kh].reshape(-1)[:n, None].double()
            q = s["q"][i, kh * g:(kh + 1) * g].double()
            if c["kind"] == "sparse":
                b0 = max(0, n - c["fresh"]) // page
                for b in range(b0, nb):
                    x = k32[b * page:min(n, (b + 1) * page)]
                    bounds[pages[b], kh, 0] = x.min(0).values
                    bounds[pages[b], kh, 1] = x.max(0).values
                sel[i, kh] = _exact_choice(c, q, k32, n, nb)
                if not c["attend"]:
                    continue
                chosen = sel[i, kh][sel[i, kh] >= 0].to(DEV).long()
                at = (chosen[:, None] * page + torch.arange(page, device=DEV)).flatten()
                at = at[at < n]
            v = p["v"][pages, kh].reshape(-1, hd)[at].double()
            if p["vs"] is not None:
                v = v * p["vs"][pages, kh].reshape(-1)[at, None].double()
            x = q @ k32[at].t().contiguous() / math.sqrt(hd)
            w = torch.softmax(x, -1)
            out[i, kh * g:(kh + 1) * g] = w @ v
    if s["gate"] is not None:
        out *= torch.sigmoid(s["gate"].double())
    res = [bounds, sel] if c["kind"] == "sparse" else []
    return res + ([out] if c["attend"] else [])


def _exact_choice(c, q, k, n, nb):
    """One KV head's blocks: the forced ones, then the largest by score."""
    page, n_sel = c["page"], c["n_sel"]
    row = torch.full((n_sel,), -1, dtype=torch.int32)
    if nb <= n_sel:
        row[:nb] = torch.arange(nb)
        return row
    full = torch.nn.functional.pad(k, (0, 0, 0, nb * page - n), value=math.nan)
    full = full.reshape(nb, page, -1)
    rounded = []
    for up in (False, True):
        x = full.nan_to_num(nan=-math.inf if up else math.inf)
        x = (x.amax(1) if up else x.amin(1)).cpu().numpy().astype(np.float32).astype(np.float64)
        x = np.clip(x, -65504, 65504)
        h = x.astype(np.float16)
        short = h.astype(np.float64) < x if up else h.astype(np.float64) > x
        h = np.where(short, np.nextafter(h, np.float16(np.inf if up else -np.inf)), h)
        rounded.append(h.astype(np.float64))
    qn = q.cpu().numpy()
    score = np.where(qn > 0, qn, 0) @ rounded[1].T + np.where(qn < 0, qn, 0) @ rounded[0].T
    score = score.max(0).astype(np.float32)
    free = list(range(c["first"], nb - c["last"]))
    best = sorted(free, key=lambda b: (-score[b], b))[:n_sel - c["first"] - c["last"]]
    forced = list(range(c["first"])) + list(range(nb - c["last"], nb))
    row[:] = torch.tensor(sorted(best + forced))
    return row
