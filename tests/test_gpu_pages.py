"""The paged cache on the GPU (include/janas_attn.h, Part 4) against the plain
rules of pages_helpers.py in 64 bits:

* janas_attn_pages_plan: every array it writes, number for number, over steps
  small and large, with releases, too few pages and refused sequences;
* janas_attn_pages_write: the rows, scales and queries bit for bit those of
  janas_attn_cache_write and janas_attn_q_prep;
* janas_attn_pages_run: within the bound that attend() derives, in pools whose
  unused numbers are NaN and whose unused table entries lie outside;
* janas_attn_pages_bounds and _select: number for number;
* all of them together, a step after another, against the contiguous cache, and
  captured once and replayed.
"""
import numpy as np
import pytest
import torch

import janas_amd as jm
import pages_helpers as ph
from attn_helpers import TOL_FLOAT_ABS, within
from janas_amd import attention as at
from oracle import orc

pytestmark = pytest.mark.gpu

KV_I8, KV_I16, KV_F16, KV_F32 = jm.KV_I8, jm.KV_I16, jm.KV_F16, jm.KV_F32
NAMES = {KV_I8: "i8", KV_I16: "i16", KV_F16: "f16", KV_F32: "f32"}
CANARY = -77777777


def dev(x, gpu):
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x)).to(gpu)


def guarded(gpu, n, fill=0):
    """n int32 between canaries: the whole, and the middle."""
    whole = torch.full((n + 16,), CANARY, dtype=torch.int32, device=gpu)
    whole[8:8 + n] = fill
    return whole, whole[8:8 + n]


def canaries_whole(*wholes):
    return all(bool((w[:8] == CANARY).all() and (w[-8:] == CANARY).all()) for w in wholes)


class OnGpu:
    """A pages_helpers.Pool's arrays on the device."""

    def __init__(self, pool, gpu, bounds=None):
        self.k, self.v, self.ks, self.vs = (dev(x, gpu) for x in
                                            (pool.k, pool.v, pool.ks, pool.vs))
        self.table, self.length = dev(pool.table, gpu), dev(np.array(pool.lens, np.int32), gpu)
        self.bounds = bounds
        self.p = at.pages(self.k, self.v, self.ks, self.vs, kv_type=pool.kv, table=self.table,
                          length=self.length, bounds=bounds)


def work_for(a, p, gpu):
    n = a.pages_work_bytes(p)
    assert n > 0
    return torch.empty(n, dtype=torch.uint8, device=gpu).fill_(0xFF)  # (NaN as floats)


# ---- plan -------------------------------------------------------------------

# (sequences, longest, most new, page, table columns beyond the longest's, free
# pages, released, packed rows: of all that are asked for)
PLANS = [(1, 0, 1, 16, 1, 1, 0, 1.0), (1, 16, 1, 16, 1, 1, 0, 1.0), (48, 500, 1, 64, 2, 64, 0, 1.2),
         (70, 300, 1, 16, 2, 20, 9, 1.0), (33, 90, 40, 16, 3, 500, 4, 1.0),
         (33, 90, 40, 16, 3, 30, 0, 1.0), (33, 90, 40, 32, 0, 300, 2, 0.6),
         (9, 4000, 2000, 16, 200, 2000, 2, 1.1), (61, 700, 900, 128, 9, 100, 5, 1.0),
         (61, 700, 900, 256, 1, 1000, 60, 0.8), (1300, 100, 1, 16, 1, 1500, 50, 1.0),
         (2100, 60, 9, 32, 1, 900, 100, 1.0), (3, 20, 0, 16, 1, 2, 0, 1.0),
         (64, 40, 5, 16, 1, 90, 7, 1.0), (65, 40, 5, 16, 1, 90, 7, 1.0),
         (12, 90, 200, 16, 8, 60, 3, 1.0)]


@pytest.mark.parametrize("case", range(len(PLANS)))
@pytest.mark.parametrize("in_place", [False, True])
def test_plan(gpu, case, in_place):
    n, longest, most, page, more, n_free, gone, part = PLANS[case]
    rng = np.random.default_rng(500 + case)
    lens = rng.integers(0, longest + 1, n).astype(np.int32)
    n_new = rng.integers(0, most + 1, n).astype(np.int32)
    n_new[rng.permutation(n)[:gone]] = ph.NONE
    need = [ph.blocks(int(x), page) for x in lens]
    n_pages = sum(need) + n_free
    order = rng.permutation(n_pages).astype(np.int32)
    table = np.full((n, max(need) + more), 0x7FFFFFF0, np.int32)
    at0 = n_free
    for i, b in enumerate(need):
        table[i, :b] = order[at0:at0 + b]
        at0 += b
    free = np.full(n_pages, 0x7FFFFFF0, np.int32)
    free[:n_free] = order[:n_free]
    cap = int(part * np.maximum(n_new, 0).sum())
    want = ph.plan(table, free, n_free, lens, n_new, page, cap)
    size = dict(length=n, n_free=1, granted=n, start=n + 1, taken=n + 1, slot=cap, pos=cap, seq=cap)
    whole, got = {}, {}
    for name, m in size.items():
        whole[name], got[name] = guarded(gpu, m, 5)
    wt, gt = guarded(gpu, table.size)
    gt.copy_(dev(table.ravel(), gpu))
    wf, gf = guarded(gpu, n_pages)
    gf.copy_(dev(free, gpu))
    new, old_len, old_free = dev(n_new, gpu), dev(lens, gpu), dev(np.array([n_free], np.int32), gpu)
    if in_place:
        got["length"].copy_(old_len)
        got["n_free"].copy_(old_free)
        got["granted"].copy_(new)
        old_len, old_free, new = got["length"], got["n_free"], got["granted"]
    p = at.page_tables(gt.view(n, -1), old_len, page=page, free=gf, n_free=old_free)
    at.pages_plan(p, new, **got)
    torch.cuda.synchronize()
    got.update(table=gt.view(n, -1), free=gf)
    for name, x in want.items():
        y = got[name].cpu().numpy()
        assert np.array_equal(x, y), (name, np.argwhere(x != y)[:5])
    assert canaries_whole(wt, wf, *whole.values())
    if not in_place:
        assert np.array_equal(old_len.cpu().numpy(), lens) and int(old_free[0]) == n_free


def test_plan_bad_counts_stay_in_the_arrays(gpu):
    """A free count above the pool, a length past the table row, an n_new near
    2^32: nothing is written outside, and such sequences are refused."""
    n, page, n_pages = 4, 16, 6
    wt, gt = guarded(gpu, n * 2, 3)
    wf, gf = guarded(gpu, n_pages)
    gf.copy_(torch.arange(n_pages, dtype=torch.int32, device=gpu))
    lens = dev(np.array([100, 5, 33, 0], np.int32), gpu)
    new = dev(np.array([1, 0x7FFFFFFF, -1, -2], np.int32), gpu)
    nf = dev(np.array([1000], np.int32), gpu)
    whole, got = {}, {}
    for name, m in dict(length=n, n_free=1, granted=n, start=n + 1, taken=n + 1, slot=9, pos=9,
                        seq=9).items():
        whole[name], got[name] = guarded(gpu, m)
    at.pages_plan(at.page_tables(gt.view(n, 2), lens, page=page, free=gf, n_free=nf), new, **got)
    torch.cuda.synchronize()
    assert got["granted"].tolist() == [0, 0, 0, 0]
    assert got["length"].tolist() == [100, 5, 0, 0]
    assert got["slot"].tolist() == [-1] * 9
    assert int(got["n_free"][0]) == n_pages
    assert canaries_whole(wt, wf, *whole.values())


@pytest.mark.parametrize("tokens", [1, 3, 70])
@pytest.mark.parametrize("rows", [100, 5000])
def test_plan_pages_outside_the_pool_have_no_slots(gpu, tokens, rows):
    """Pages whose slots would be another's in 32 bits (2^28 pages of 16 are 2^32
    slots), named by the table or on the stack: the tokens that would lie there
    have none, the others theirs. In one launch and in two."""
    page, n_pages = 16, 12
    wild = 1 << 28
    table = torch.tensor([[wild, 1, 0, 0, 0, 0], [2, wild + 1, 0, 0, 0, 0], [3, 0, 0, 0, 0, 0],
                          [4, 5, 0, 0, 0, 0]], dtype=torch.int32, device=gpu)
    lens = [7, 20, 16, 17]
    free = torch.zeros(n_pages, dtype=torch.int32, device=gpu)
    # (from the top: the third page that the step takes is outside)
    free[:6] = torch.tensor([9, 8, 7, wild + 2, 6, 10], dtype=torch.int32)
    out = {name: torch.full((m,), CANARY, dtype=torch.int32, device=gpu)
           for name, m in dict(length=4, n_free=1, granted=4, start=5, taken=5, slot=rows, pos=rows,
                               seq=rows).items()}
    n_new = [tokens if tokens < 70 else x for x in (20, 3, 30, 0)]
    p = at.page_tables(table, dev(np.array(lens, np.int32), gpu), page=page, free=free,
                       n_free=torch.full((1,), 6, dtype=torch.int32, device=gpu))
    at.pages_plan(p, dev(np.array(n_new, np.int32), gpu), **out)
    torch.cuda.synchronize()
    assert out["granted"].tolist() == n_new
    at_ = [(pos, int(table[i, pos // page])) for i, n in enumerate(n_new)
           for pos in range(lens[i], lens[i] + n)]
    want = [pg * page + pos % page if pg < n_pages else -1 for pos, pg in at_]
    behind = rows - len(want)
    assert out["slot"].tolist() == want + [-1] * behind
    assert out["pos"].tolist() == [pos if pg < n_pages else 0 for pos, pg in at_] + [0] * behind
    assert -1 in want and max(want) >= 0


# ---- write ------------------------------------------------------------------

# tokens, query heads, KV heads, hd, n_rot, norms, v_norm, page
WRITES = [(1, 4, 2, 64, 64, True, False, 16), (7, 32, 8, 128, 128, True, False, 64),
          (37, 8, 1, 256, 128, False, True, 32), (5, 3, 3, 512, 512, True, True, 128),
          (9, 4, 2, 96, 0, True, False, 16), (6, 2, 1, 40, 36, True, True, 16),
          (300, 2, 2, 8, 8, False, False, 256)]


@pytest.mark.parametrize("kv", [KV_I8, KV_I16, KV_F16, KV_F32], ids=NAMES.get)
@pytest.mark.parametrize("case", range(len(WRITES)))
@pytest.mark.parametrize("how", ["packed", "strided", "unaligned", "in place", "no queries"])
def test_write_is_the_contiguous_write(gpu, kv, case, how):
    n, h, n_kv, hd, n_rot, norms, v_norm, page = WRITES[case]
    rng = np.random.default_rng(700 + case)
    n_tab, n_pages = 50, 3 + 2 * n // page
    cs, sn = (dev(x, gpu) for x in ph.rotation(n_tab, n_rot))
    x = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(gpu)  # noqa: E731
    q, k, v = 2 * x(n, h, hd), 1.5 * x(n, n_kv, hd), x(n, n_kv, hd)
    qn, kn = (x(hd) if norms else None for _ in range(2))
    slot = rng.permutation(n_pages * page)[:n].astype(np.int32)
    pos = rng.integers(0, n_tab, n).astype(np.int32)
    # rows left out: none, outside the pool, no row of the table
    out = np.zeros(n, bool)
    if n > 4:
        slot[1], slot[3] = ph.NONE, n_pages * page
        out[[1, 3]] = True
        if n_rot:
            pos[4] = n_tab
            out[4] = True
    # the contiguous calls, a token at a time at its position's table row
    dt = {KV_I8: torch.int8, KV_I16: torch.int16, KV_F16: torch.float16, KV_F32: torch.float32}[kv]
    ck, cv = (torch.zeros(n_kv, n, hd, dtype=dt, device=gpu) for _ in range(2))
    cks, cvs = (torch.zeros(n_kv, n, device=gpu) for _ in range(2))
    cache = at.cache(ck, cv, cks, cvs, kv_type=kv)
    turn = torch.from_numpy(np.minimum(pos, n_tab - 1)).to(gpu).long()
    tc, ts = (t[turn].contiguous() if n_rot else None for t in (cs, sn))
    at.cache_write(cache, k, v, cs=tc, sn=ts, n_rot=n_rot, pos0=0, k_norm=kn, v_norm=v_norm)
    want_q = q.clone()
    at.q_prep(want_q, cs=tc, sn=ts, n_rot=n_rot, q_norm=qn)
    # the pool
    mark = torch.zeros(1, dtype=dt, device=gpu).fill_(77)[0]
    pk, pv = (torch.full((n_pages, n_kv, page, hd), 77, dtype=dt, device=gpu) for _ in range(2))
    pks, pvs = (torch.full((n_pages, n_kv, page), 7.5, device=gpu) for _ in range(2))
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu)
    p = at.pages(pk, pv, pks, pvs, kv_type=kv, table=table, length=table[0])
    given = dict(q=q, k=k, v=v)
    if how == "strided":     # one product's rows: q, k, v side by side, and some
        wide = x(n, h + 2 * n_kv + 1, hd)
        for name, a, b in (("q", 0, h), ("k", h, h + n_kv), ("v", h + n_kv, h + 2 * n_kv)):
            wide[:, a:b] = given[name]
            given[name] = wide[:, a:b]
    elif how == "unaligned":
        for name, y in given.items():
            flat = torch.zeros(y.numel() + 1, device=gpu)
            flat[1:] = y.ravel()
            given[name] = flat[1:].view(y.shape)
    q_out = torch.full((n, h, hd), 3.25, device=gpu)
    if how == "in place":
        q_out = given["q"]
    more = {} if how == "no queries" else dict(q=given["q"], q_out=q_out, q_norm=qn)
    at.pages_write(p, given["k"], given["v"], slot=dev(slot, gpu), pos=dev(pos, gpu), cs=cs, sn=sn,
                   n_rot=n_rot, k_norm=kn, v_norm=v_norm, **more)
    torch.cuda.synchronize()
    at_page, at_row = slot // page, slot % page
    scaled = kv in ph.TOP
    left = q if how == "in place" else torch.full_like(q, 3.25)
    for t in range(n):
        if out[t]:
            assert torch.equal(q_out[t], left[t]) or how in ("in place", "no queries")
            continue
        b, r = int(at_page[t]), int(at_row[t])
        assert torch.equal(pk[b, :, r], ck[:, t]) and torch.equal(pv[b, :, r], cv[:, t])
        if scaled:
            assert torch.equal(pks[b, :, r], cks[:, t]) and torch.equal(pvs[b, :, r], cvs[:, t])
        if how != "no queries":
            assert torch.equal(q_out[t], want_q[t])
    # nothing else
    kept = np.ones(n_pages * page, bool)
    kept[slot[~out]] = False
    kept = torch.from_numpy(kept).to(gpu).view(n_pages, page)
    for y in (pk, pv):
        assert bool((y.transpose(1, 2)[kept] == mark).all())
    assert bool((pks.transpose(1, 2)[kept] == 7.5).all())


@pytest.mark.parametrize("kv", [KV_I8, KV_I16, KV_F16, KV_F32], ids=NAMES.get)
@pytest.mark.parametrize("hd,n_rot", [(128, 128), (128, 0), (40, 36)])
@pytest.mark.parametrize("how", ["in place", "apart", "no queries"])
def test_write_leaves_rows_out(gpu, kv, hd, n_rot, how):
    """Rows without a slot, with one outside the pool, or at a position that the
    table does not have: nothing of them is written, their queries neither, which
    in place are the caller's own; the other rows are those of a call without
    them."""
    n, h, n_kv, page, n_pages, n_tab = 9, 4, 2, 16, 3, 50
    rng = np.random.default_rng([kv, hd, n_rot])
    cs, sn = (dev(x, gpu) for x in ph.rotation(n_tab, n_rot))
    x = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).to(gpu)  # noqa: E731
    q, k, v, kn, qn = x(n, h, hd), x(n, n_kv, hd), x(n, n_kv, hd), x(hd), x(hd)
    slot = torch.from_numpy(rng.permutation(n_pages * page)[:n].astype(np.int32)).to(gpu)
    pos = torch.arange(n, dtype=torch.int32, device=gpu)
    slot[1], slot[4], slot[8] = ph.NONE, n_pages * page, 0x7FFFFFFF
    left = [1, 4, 8]
    if n_rot:
        pos[5], pos[6] = n_tab, -1
        left += [5, 6]
    kept = [t for t in range(n) if t not in left]
    dt = {KV_I8: torch.int8, KV_I16: torch.int16, KV_F16: torch.float16, KV_F32: torch.float32}[kv]
    table = torch.zeros(1, 1, dtype=torch.int32, device=gpu)

    def written(rows):
        pool = [torch.full((n_pages, n_kv, page, hd), 77, dtype=dt, device=gpu) for _ in range(2)]
        pool += [torch.full((n_pages, n_kv, page), 7.5, device=gpu) for _ in range(2)]
        p = at.pages(*pool, kv_type=kv, table=table, length=table[0])
        qq = q[rows].clone()
        out = qq if how == "in place" else torch.full_like(qq, 3.25)
        more = {} if how == "no queries" else dict(q=qq, q_out=out, q_norm=qn)
        at.pages_write(p, k[rows].clone(), v[rows].clone(), slot=slot[rows].clone(),
                       pos=pos[rows].clone(), cs=cs, sn=sn, n_rot=n_rot, k_norm=kn, **more)
        torch.cuda.synchronize()
        return pool, out
    (pool, out), (pool2, out2) = written(list(range(n))), written(kept)
    for y, z in zip(pool, pool2):
        assert torch.equal(y, z)
    assert torch.equal(out[kept], out2)
    before = q if how == "in place" else torch.full_like(q, 3.25)
    assert torch.equal(out[left], before[left])
    if how == "no queries":
        assert bool((out == 3.25).all())
    else:
        assert not bool((out[kept] == before[kept]).flatten(1).all(1).any())


# ---- attention --------------------------------------------------------------

def run_pages(gpu, pool, h, q, *, window=0, gate=None, mode=jm.GATE_NONE, sel=None, scale=None,
              times=1, **more):
    g = OnGpu(pool, gpu)
    out = torch.full((q.shape[0], h, pool.hd), float("nan"), device=gpu)
    with jm.Attention(h, pool.n_kv, pool.hd, 256) as a:
        a.set_window(window)
        if scale is not None:
            a.set_scale(scale)
        work = work_for(a, g.p, gpu)
        call = a.prepare_pages(g.p, dev(q, gpu), out, work=work, gate=dev(gate, gpu),
                               gate_mode=mode, sel=dev(sel, gpu), **more)
        first = None
        for _ in range(times):
            call()
            torch.cuda.synchronize()
            assert first is None or np.array_equal(first, out.cpu().numpy(), equal_nan=True)
            first = out.cpu().numpy().copy()
        assert a.status() == 0
    return first


def check_run(pool, h, q, out, *, window=0, gate=None, sel=None, scale=None, what=""):
    scale = ph.default_scale(pool.hd) if scale is None else scale
    g = h // pool.n_kv
    for i, n in enumerate(pool.lens):
        k, v = pool.rows("k", i), pool.rows("v", i)
        near = ph.in_sight(n, window)
        seen = [near] * pool.n_kv
        if sel is not None:
            cnt = min(sel.shape[2], ph.blocks(n, pool.page))
            seen = [np.array([p for b in sel[i, kh, :cnt] if 0 <= b for p in
                              range(b * pool.page, (b + 1) * pool.page)
                              if p < n and (not window or p >= n - window)], np.int64)
                    for kh in range(pool.n_kv)]
        want, bar = ph.attend(q[i], k, v, scale, seen)
        if gate is not None:
            want = want * ph.sigmoid(gate[i]).reshape(h, -1)
            bar = bar + np.abs(want).max(1) * 2.0 ** -20
        err = np.abs(out[i].astype(np.float64) - want).max(1)
        worst = int(np.argmax(err / np.maximum(bar, 1e-30)))
        assert within(err[worst], max(bar[worst], 1e-30), f"{what} len {n} head {worst}"), \
            (i, n, g, err, bar)


SHAPES = [(32, 8, 128), (4, 4, 64), (12, 4, 64), (16, 2, 256), (20, 1, 128), (9, 1, 72), (6, 2, 8),
          (16, 2, 512), (5, 1, 200), (34, 2, 264)]


# (other head sizes are refused: test_refusals)
RUNS = [(kv, s) for kv in (KV_I8, KV_I16, KV_F16, KV_F32) for s in SHAPES
        if (16 if kv == KV_I8 else 8) <= s[2] <= (256 if kv == KV_F32 else 512)]


@pytest.mark.parametrize("kv,shape", RUNS, ids=lambda x: NAMES.get(x) if isinstance(x, int) else
                         "-".join(map(str, x)))
@pytest.mark.parametrize("page", [16, 64, 256])
def test_run(gpu, kv, shape, page):
    h, n_kv, hd = shape
    rng = np.random.default_rng([kv, h, hd, page])
    lens = [1, 2, 15, 16, 17, page - 1, page, page + 1, 0, 3 * page + 5, 700, 333]
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    q = (rng.standard_normal((len(lens), h, hd)) *
         (1 + np.arange(h) % 4 * 0.5)[:, None]).astype(np.float32)
    out = run_pages(gpu, pool, h, q, times=2)
    check_run(pool, h, q, out, what=f"{NAMES[kv]} {shape} page {page}")
    assert not out[lens.index(0)].any()


@pytest.mark.parametrize("kv", [KV_I8, KV_I16, KV_F16, KV_F32], ids=NAMES.get)
@pytest.mark.parametrize("window,mode", [(1, 0), (16, 1), (77, 2), (100000, 1)])
def test_run_windows_and_gates(gpu, kv, window, mode):
    h, n_kv, hd, page = 8, 2, 128, 32
    rng = np.random.default_rng([kv, window])
    lens = [1, 16, 17, 76, 77, 78, 400, 1025, 0]
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    # what lies before the window may be gone: other pages, other numbers
    for i, n in enumerate(lens):
        for b in range(max(0, n - window) // page):
            pool.table[i, b] = 0x7FFFFF00
    q = rng.standard_normal((len(lens), h, hd)).astype(np.float32)
    gate = rng.standard_normal((len(lens), h, hd) if mode == 1 else (len(lens), h))
    gate = gate.astype(np.float32) if mode else None
    out = run_pages(gpu, pool, h, q, window=window, gate=gate, mode=mode, scale=0.11)
    for i, n in enumerate(lens):
        for b in range(max(0, n - window) // page):
            pool.table[i, b] = 0
    shaped = gate if mode != 2 else gate[..., None]
    if mode == 2:
        shaped = np.repeat(shaped, hd, axis=2)
    check_run(pool, h, q, out, window=window, gate=shaped, scale=float(np.float32(0.11)),
              what=f"window {window} gate {mode}")


@pytest.mark.parametrize("kv", [KV_I8, KV_F16, KV_F32], ids=NAMES.get)
def test_run_long_and_many(gpu, kv):
    """Sequences of one and of many thousand positions in one call, more than a
    wave's lanes of them, and table rows of more entries than a wave holds."""
    h, n_kv, hd, page = 4, 1, 64, 16
    rng = np.random.default_rng(kv)
    lens = [int(x) for x in rng.integers(0, 40, 130)] + [9001, 3, 20011]
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    q = (2 * rng.standard_normal((len(lens), h, hd))).astype(np.float32)
    out = run_pages(gpu, pool, h, q, times=2)
    check_run(pool, h, q, out, what="long and many")


@pytest.mark.parametrize("kv,hd", [(KV_I8, 64), (KV_I8, 128), (KV_I16, 128), (KV_F16, 128),
                                   (KV_F32, 64), (KV_F16, 256)])
@pytest.mark.parametrize("picked", [False, True])
def test_run_more_sequences_than_workgroups(gpu, kv, hd, picked):
    """Workgroups that go from a sequence into the next, and on: more short
    sequences than there are workgroups, among them empty and a long one."""
    h, n_kv, page = 16, 8, 16
    rng = np.random.default_rng([kv, hd])
    lens = [int(x) for x in rng.integers(0, 90, 300)] + [3000] + [17] * 20
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    q = rng.standard_normal((len(lens), h, hd)).astype(np.float32)
    sel = None
    if picked:
        sel = np.full((len(lens), n_kv, 4), ph.NONE, np.int32)
        for i, n in enumerate(lens):
            nb = ph.blocks(n, page)
            for kh in range(n_kv):
                m = min(nb, 4)
                sel[i, kh, :m] = np.sort(rng.permutation(nb)[:m])
    out = run_pages(gpu, pool, h, q, sel=sel, times=2)
    check_run(pool, h, q, out, sel=sel, what="many sequences")


def test_run_shared_pages(gpu):
    """Sequences that begin with the same pages."""
    h, n_kv, hd, page = 4, 2, 64, 16
    rng = np.random.default_rng(12)
    pool = ph.Pool(rng, KV_F16, [100, 77, 64], page, n_kv, hd)
    pool.table[1, :3] = pool.table[0, :3]
    pool.table[2, :4] = pool.table[0, :4]
    q = rng.standard_normal((3, h, hd)).astype(np.float32)
    check_run(pool, h, q, run_pages(gpu, pool, h, q), what="shared pages")


@pytest.mark.parametrize("kv", [KV_I8, KV_I16], ids=NAMES.get)
def test_run_value_scales_of_unlike_size(gpu, kv):
    """Value scales from 2^-60 to 2^20, growing, falling and mixed along a
    sequence: the weights' planes follow the largest. Keys alike, so that every
    position weighs about the same."""
    h, n_kv, hd, page = 2, 1, 64, 16
    rng = np.random.default_rng(kv)
    lens = [300, 300, 300, 60]
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    e = [np.linspace(-60, 20, 300), np.linspace(20, -60, 300), rng.uniform(-60, 20, 300),
         np.full(60, -58.0)]
    for i, n in enumerate(lens):
        for t in range(n):
            at_ = pool.table[i, t // page], 0, t % page
            pool.vs[at_] = np.float32(2.0 ** e[i][t])
            pool.ks[at_] *= np.float32(0.05)
    q = rng.standard_normal((len(lens), h, hd)).astype(np.float32)
    out = run_pages(gpu, pool, h, q)
    check_run(pool, h, q, out, what="value scales")


def test_run_scores_that_climb(gpu):
    """Scores that rise by hundreds along the sequence (each unit renews the
    row's reference), fall, or are all far below zero."""
    h, n_kv, hd, page = 2, 1, 64, 16
    rng = np.random.default_rng(1)
    lens = [500, 500, 500]
    pool = ph.Pool(rng, KV_F32, lens, page, n_kv, hd)
    for i, slope in enumerate((1.0, -1.0, 0.0)):
        for t in range(500):
            pool.k[pool.table[i, t // page], 0, t % page] = slope * t - (900 if i == 2 else 0)
    q = np.full((3, h, hd), 1 / 64, np.float32)
    q[:, 1] = 1 / 512
    out = run_pages(gpu, pool, h, q, scale=1.0)
    check_run(pool, h, q, out, scale=1.0, what="climbing scores")


def test_run_rows_that_take_part(gpu):
    """With a step's start and granted: packed rows, those of sequences that
    wait or bring a prompt left as they were; a row outside the tensor takes no
    part."""
    h, n_kv, hd, page = 4, 2, 64, 16
    rng = np.random.default_rng(2)
    lens = [40, 33, 0, 100, 17, 5]
    granted = np.array([1, 0, 1, 3, 1, 1], np.int32)
    start = np.array([0, 1, 1, 2, 5, 6, 7], np.int32)
    pool = ph.Pool(rng, KV_F16, lens, page, n_kv, hd)
    q = rng.standard_normal((6, h, hd)).astype(np.float32)   # (start[5] = 6 is outside)
    g = OnGpu(pool, gpu)
    out = torch.full((6, h, hd), 5.0, device=gpu)
    with jm.Attention(h, n_kv, hd, 256) as a:
        a.run_pages(g.p, dev(q, gpu), out, work=work_for(a, g.p, gpu), rows=dev(start, gpu),
                    granted=dev(granted, gpu))
    torch.cuda.synchronize()
    out = out.cpu().numpy()
    for i, r in ((0, 0), (2, 1), (4, 5)):
        want, bar = ph.attend(q[r], pool.rows("k", i), pool.rows("v", i), ph.default_scale(hd),
                              [np.arange(lens[i])] * n_kv)
        assert (np.abs(out[r] - want).max(1) <= np.maximum(bar, 1e-30)).all()
    assert (out[2:5] == 5.0).all()


def test_calls_without_rows(gpu):
    """A step in which nobody has a token: empty tensors, which have no address."""
    rng = np.random.default_rng(43)
    pool = ph.Pool(rng, KV_F16, [40, 20], 16, 1, 64)
    g = OnGpu(pool, gpu, torch.zeros(pool.n_pages, 1, 2, 64, dtype=torch.float16, device=gpu))
    zero = torch.zeros(2, dtype=torch.int32, device=gpu)
    q = torch.zeros(0, 4, 64, device=gpu)
    sel = torch.full((2, 1, 2), 7, dtype=torch.int32, device=gpu)
    with jm.Attention(4, 1, 64, 64) as a:
        part = dict(work=work_for(a, g.p, gpu), rows=zero, granted=zero)
        blocks = torch.zeros(0, dtype=torch.uint8, device=gpu)
        a.run_pages(g.p, q, q.clone(), out_q8k=blocks, **part)
        a.select(g.p, q, sel, **part)
        at.pages_write(g.p, q[:, :1], q[:, :1], slot=zero[:0])
        assert a.status() == 0
    torch.cuda.synchronize()
    assert bool((sel == 7).all())


def test_run_strided_queries_and_q8k(gpu):
    h, n_kv, hd, page = 8, 2, 128, 64
    rng = np.random.default_rng(3)
    lens = [100, 64, 1]
    pool = ph.Pool(rng, KV_I8, lens, page, n_kv, hd)
    wide = rng.standard_normal((3, h + 2 * n_kv, hd)).astype(np.float32)
    g = OnGpu(pool, gpu)
    out = torch.empty(3, h, hd, device=gpu)
    blocks = torch.zeros(3, h * hd // 256, at.Q8K_BYTES, dtype=torch.uint8, device=gpu)
    with jm.Attention(h, n_kv, hd, 256) as a:
        a.run_pages(g.p, dev(wide, gpu)[:, :h], out, work=work_for(a, g.p, gpu), out_q8k=blocks)
    torch.cuda.synchronize()
    check_run(pool, h, wide[:, :h], out.cpu().numpy(), what="strided queries")
    want = orc.q8k_quantize(out.cpu().numpy().reshape(3, h * hd))
    assert blocks.cpu().numpy().tobytes() == want.tobytes()


def test_run_bad_tables(gpu):
    """A page outside the pool, or a length past the table row: that row is NaN,
    the others are what they are."""
    h, n_kv, hd, page = 4, 2, 64, 16
    rng = np.random.default_rng(4)
    lens = [40, 3000, 50, 60]
    pool = ph.Pool(rng, KV_F16, lens, page, n_kv, hd, extra=0)
    q = rng.standard_normal((4, h, hd)).astype(np.float32)
    good = run_pages(gpu, pool, h, q)
    for entry in (pool.n_pages, -1, 0x7FFFFFF0):
        table = pool.table.copy()
        pool.table[1, 93] = entry
        pool.table[2, 0] = entry
        bad = run_pages(gpu, pool, h, q)
        assert np.isnan(bad[1]).all() and np.isnan(bad[2]).all()
        # (the splits are the same: the lengths are)
        assert np.array_equal(bad[0], good[0]) and np.array_equal(bad[3], good[3])
        pool.table = table
    pool.lens[1] = pool.table.shape[1] * page + 1
    bad = run_pages(gpu, pool, h, q)
    assert np.isnan(bad[1]).all() and np.isfinite(bad[[0, 2, 3]]).all()


@pytest.mark.parametrize("kv", [KV_I8, KV_I16, KV_F16, KV_F32], ids=NAMES.get)
@pytest.mark.parametrize("window", [0, 150])
def test_run_selected(gpu, kv, window):
    """Lists as a selection makes them, and others: out of order, with entries
    that are none, past the sequence, before the window, or named twice; a list
    that names nothing."""
    h, n_kv, hd, page = 8, 2, 64, 32
    rng = np.random.default_rng([kv, window])
    lens = [500, 33, 0, 1025, 320, 700]
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    n_sel = 7
    sel = np.full((len(lens), n_kv, n_sel), ph.NONE, np.int32)
    for i, n in enumerate(lens):
        nb = ph.blocks(n, page)
        for kh in range(n_kv):
            m = min(nb, n_sel)
            sel[i, kh, :m] = rng.permutation(nb)[:m]
    sel[0, 0] = [15, 3, ph.NONE, 3, 15, 900, 0]
    sel[3, 1] = [0x7FFFFFFF, 33, 32, 31, ph.NONE, 30, 29]
    sel[4, 0] = ph.NONE
    q = rng.standard_normal((len(lens), h, hd)).astype(np.float32)
    out = run_pages(gpu, pool, h, q, window=window, sel=sel, times=2)
    check = sel.copy()
    for i, n in enumerate(lens):
        nb = ph.blocks(n, page)
        check[i][(check[i] >= nb)] = ph.NONE
    check_run(pool, h, q, out, window=window, sel=check, what="selected")
    assert not out[4, :h // n_kv].any() and not out[2].any()


@pytest.mark.parametrize("kv", [KV_I8, KV_I16, KV_F16, KV_F32], ids=NAMES.get)
@pytest.mark.parametrize("window", [1, 16, 77, 150])
def test_run_selected_blocks_before_the_window(gpu, kv, window):
    """A list kept for some steps while the window goes on: the pages of the
    blocks that it has left may be gone, and their table entries anything. A
    block that the window begins in is still read, and is bad if its page is."""
    h, n_kv, hd, page = 8, 2, 64, 32
    rng = np.random.default_rng([kv, window])
    lens = [500, 33, 0, 1025, 320, 700, 64]
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    n_sel = 9
    sel = np.full((len(lens), n_kv, n_sel), ph.NONE, np.int32)
    for i, n in enumerate(lens):
        nb = ph.blocks(n, page)
        for kh in range(n_kv):
            m = min(nb, n_sel)
            sel[i, kh, :m] = rng.permutation(nb)[:m]
            sel[i, kh, :min(m, 2)] = [nb - 1, 0][:min(m, 2)]
    q = rng.standard_normal((len(lens), h, hd)).astype(np.float32)
    whole = pool.table.copy()
    for i, n in enumerate(lens):
        for b in range(max(0, n - window) // page):
            pool.table[i, b] = (0x7FFFFF00, -1, pool.n_pages)[b % 3]
    gone = pool.table.copy()
    out = run_pages(gpu, pool, h, q, window=window, sel=sel, times=2)
    pool.table = whole
    check_run(pool, h, q, out, window=window, sel=sel, what="blocks before the window")
    # the first block in sight of the longest sequence, gone too
    b = (1025 - window) // page
    pool.table = gone
    pool.table[3, b] = -1
    sel[3, 0, 1] = b
    bad = run_pages(gpu, pool, h, q, window=window, sel=sel)
    assert np.isnan(bad[3, :h // n_kv]).all()
    assert np.array_equal(bad[[0, 1, 2, 4, 5, 6]], out[[0, 1, 2, 4, 5, 6]])


# ---- bounds and selection ---------------------------------------------------

@pytest.mark.parametrize("kv", [KV_I8, KV_I16, KV_F16, KV_F32], ids=NAMES.get)
@pytest.mark.parametrize("hd,page", [(64, 16), (128, 64), (256, 128), (512, 256), (72, 32),
                                     (200, 64), (136, 16), (8, 64)])
def test_bounds(gpu, kv, hd, page):
    n_kv = 2
    rng = np.random.default_rng([kv, hd])
    lens = [1, page, page + 1, 0, 3 * page - 1, 700]
    pool = ph.Pool(rng, kv, lens, page, n_kv, hd)
    if kv == KV_F32:     # numbers outside of the halves, tiny ones, zeros, NaN
        b, r = pool.table[5, 0], 3
        pool.k[b, 0, r, :6] = [1e6, -1e6, 1e-9, -1e-9, 0.0, np.nan]
        pool.k[b, 1, :, 0] = np.nan
        pool.k[b, 1, :, 1] = -0.0
    fresh = np.array([1, 1, 2, 4, page, 10000], np.int32)
    bounds = torch.full((pool.n_pages, n_kv, 2, hd), 7.0, dtype=torch.float16, device=gpu)
    g = OnGpu(pool, gpu, bounds)
    at.pages_bounds(g.p, dev(fresh, gpu), max_new=3)
    torch.cuda.synchronize()
    want = np.full(bounds.shape, 7.0, np.float16)
    for i, n in enumerate(lens):
        for b in range(max(0, n - fresh[i]) // page, ph.blocks(n, page)):
            want[pool.table[i, b]] = ph.key_bounds(pool, i, b)
    got = bounds.cpu().numpy()
    assert np.array_equal(want.astype(np.float32), got.astype(np.float32))
    at.pages_bounds(g.p)
    torch.cuda.synchronize()
    for i, n in enumerate(lens):
        for b in range(ph.blocks(n, page)):
            want[pool.table[i, b]] = ph.key_bounds(pool, i, b)
    assert np.array_equal(want.astype(np.float32), bounds.cpu().numpy().astype(np.float32))


def test_bounds_pass_over_a_bad_page(gpu):
    rng = np.random.default_rng(5)
    pool = ph.Pool(rng, KV_I8, [100], 16, 1, 64)
    pool.table[0, 2], pool.table[0, 3] = pool.n_pages, -1
    bounds = torch.full((pool.n_pages, 1, 2, 64), 7.0, dtype=torch.float16, device=gpu)
    at.pages_bounds(OnGpu(pool, gpu, bounds).p)
    torch.cuda.synchronize()
    made = (bounds != 7.0).flatten(1).any(1).cpu().numpy()
    assert sorted(np.flatnonzero(made)) == sorted(pool.table[0, [0, 1, 4, 5, 6]])


def selected(gpu, pool, h, q, n_sel, first, last, *, window=0, boxes=None, scale=None, **more):
    if boxes is None:
        boxes = np.full((pool.n_pages, pool.n_kv, 2, pool.hd), np.nan, np.float16)
        for i, n in enumerate(pool.lens):
            for b in range(ph.blocks(n, pool.page)):
                boxes[pool.table[i, b]] = ph.key_bounds(pool, i, b)
    g = OnGpu(pool, gpu, dev(boxes, gpu))
    sel = torch.full((len(pool.lens), pool.n_kv, n_sel), -5, dtype=torch.int32, device=gpu)
    with jm.Attention(h, pool.n_kv, pool.hd, 256) as a:
        a.set_window(window)
        if scale is not None:
            a.set_scale(scale)
        a.select(g.p, dev(q, gpu), sel, first=first, last=last, work=work_for(a, g.p, gpu), **more)
    torch.cuda.synchronize()
    return sel.cpu().numpy(), boxes


@pytest.mark.parametrize("h,n_kv,hd", [(8, 2, 64), (32, 8, 128), (16, 2, 256), (7, 1, 72),
                                       (34, 2, 512), (40, 1, 128), (6, 2, 200)])
@pytest.mark.parametrize("n_sel,first,last,window", [(1, 0, 0, 0), (5, 1, 2, 0), (4, 2, 2, 0),
                                                     (9, 0, 1, 500), (64, 1, 1, 0)])
def test_select(gpu, h, n_kv, hd, n_sel, first, last, window):
    page = 16
    rng = np.random.default_rng([h, n_sel])
    lens = [1, 700, 0, 16 * n_sel, 16 * n_sel + 1, 333, 1601]
    pool = ph.Pool(rng, KV_I8, lens, page, n_kv, hd, key_shift=1.0)
    q = rng.standard_normal((len(lens), h, hd)).astype(np.float32)
    q[1, :, 3] = 0.0
    for scale in (None, -0.25):
        got, boxes = selected(gpu, pool, h, q, n_sel, first, last, window=window, scale=scale)
        g = h // n_kv
        for i, n in enumerate(lens):
            mine = boxes[pool.table[i, :ph.blocks(n, page)]]
            for kh in range(n_kv):
                qq = q[i, kh * g:(kh + 1) * g] * (-1 if scale else 1)
                want = ph.choose(qq, mine[:, kh], n, window, page, n_sel, first, last)
                assert np.array_equal(want, got[i, kh]), (i, n, kh, want, got[i, kh])


@pytest.mark.parametrize("nb", [513, 2500, 4097, 8193])
def test_select_ties_and_many_blocks(gpu, nb):
    """Blocks of equal scores (the lower is taken), all of them equal, scores of
    both signs and zeros of both signs, over more blocks than threads, and than
    keys that stay in registers."""
    h, n_kv, hd, page = 2, 1, 64, 16
    rng = np.random.default_rng(6)
    lens = [16 * nb, 16 * nb, 16 * nb - 1]
    pool = ph.Pool(rng, KV_I8, [16] * 3, page, n_kv, hd)
    pool.n_pages = nb
    pool.k = np.zeros((nb, n_kv, page, hd), np.int8)
    pool.v, pool.ks = pool.k, np.zeros((nb, n_kv, page), np.float32)
    pool.vs = pool.ks
    pool.lens = lens
    pool.table = np.stack([rng.permutation(nb) for _ in lens]).astype(np.int32)
    boxes = np.zeros((nb, n_kv, 2, hd), np.float16)
    boxes[:, :, 1, 0] = rng.integers(-3, 4, (nb, n_kv))
    boxes[:, :, 0, 0] = boxes[:, :, 1, 0] - 1
    q = np.zeros((3, h, hd), np.float32)
    q[:, 0, 0], q[:, 1, 0] = 1.0, -0.5
    q[1] = 0.0
    for n_sel, first, last in ((900, 1, 3), (nb - 1, 0, 0), (1, 0, 0), (60, 0, 0), (7, 3, 4)):
        got, _ = selected(gpu, pool, h, q, n_sel, first, last, boxes=boxes)
        for i, n in enumerate(lens):
            want = ph.choose(q[i], boxes[pool.table[i]][:, 0], n, 0, page, n_sel, first, last)
            assert np.array_equal(want, got[i, 0]), (i, n_sel)


def test_select_rows_that_take_part(gpu):
    rng = np.random.default_rng(7)
    pool = ph.Pool(rng, KV_F16, [400, 400, 400], 16, 1, 64)
    q = rng.standard_normal((2, 2, 64)).astype(np.float32)
    got, boxes = selected(gpu, pool, 2, q, 4, 1, 1,
                          rows=torch.tensor([1, 0, 0], dtype=torch.int32, device=gpu),
                          granted=torch.tensor([1, 0, 1], dtype=torch.int32, device=gpu))
    for i, r in ((0, 1), (2, 0)):
        mine = boxes[pool.table[i, :25]]
        assert np.array_equal(got[i, 0], ph.choose(q[r], mine[:, 0], 400, 0, 16, 4, 1, 1))
    assert (got[1] == -5).all()


# ---- refusals that need an instance -------------------------------------------

def test_refusals(gpu):
    rng = np.random.default_rng(8)
    pool = ph.Pool(rng, KV_F16, [40, 20], 16, 2, 64)
    bounds = torch.zeros(pool.n_pages, 2, 2, 64, dtype=torch.float16, device=gpu)
    g = OnGpu(pool, gpu, bounds)
    q, out = torch.zeros(2, 4, 64, device=gpu), torch.zeros(2, 4, 64, device=gpu)
    sel = torch.zeros(2, 2, 3, dtype=torch.int32, device=gpu)

    def code(f, *args, **kw):
        with pytest.raises(jm.AttnError) as e:
            f(*args, **kw)
        return e.value.code
    with jm.Attention(4, 2, 64, 256) as a:
        work = work_for(a, g.p, gpu)
        assert code(a.run_pages, g.p, q, out, work=work[:256]) == jm.ERANGE
        assert code(a.run_pages, g.p, q, out, work=work[16:]) == jm.EINVAL
        assert code(a.run_pages, g.p, q, out, work=work, gate_mode=jm.GATE_ELEM) == jm.EINVAL
        assert code(a.run_pages, g.p, q, out, work=work, gate_mode=3) == jm.EINVAL
        odd = torch.zeros(2 * 4 * 64 + 1, device=gpu)[1:].view(2, 4, 64)
        assert code(a.run_pages, g.p, odd, out, work=work) == jm.EINVAL
        assert code(a.run_pages, g.p, q, odd, work=work) == jm.EINVAL
        assert code(a.select, g.p, q, sel, first=2, last=2, work=work) == jm.EINVAL
        assert code(a.select, OnGpu(pool, gpu).p, q, sel, work=work) == jm.EINVAL
        assert code(a.select, g.p, q, sel, work=work[:0]) in (jm.ERANGE, jm.EINVAL)
        a.set_ring(True)
        assert code(a.run_pages, g.p, q, out, work=work) == jm.ENOTSUP
        assert a.pages_work_bytes(g.p) == 0
        for bad in (lambda: a.run_pages(g.p, q[:1], out[:1], work=work),
                    lambda: a.run_pages(g.p, q, out[:1], work=work),
                    lambda: a.run_pages(g.p, q, out, work=work, rows=sel[0, 0]),
                    lambda: a.run_pages(g.p, q.half(), out, work=work)):
            with pytest.raises(ValueError):
                bad()
        assert a.status() == 0
    with jm.Attention(2, 1, 64, 256) as b:
        assert b.pages_work_bytes(g.p) == 0
    for kv, hd, code_ in ((KV_F32, 264, 0), (KV_I8, 8, 0)):
        wide = ph.Pool(rng, kv, [20], 16, 1, hd)
        with jm.Attention(2, 1, hd, 256) as b:
            assert b.pages_work_bytes(OnGpu(wide, gpu).p) == code_
            w = torch.zeros(1, 2, hd, device=gpu)
            assert code(b.run_pages, OnGpu(wide, gpu).p, w, w.clone(), work=work) == jm.ENOTSUP


# ---- together -----------------------------------------------------------------

class Server:
    """A layer of a program that serves: a pool and its step's buffers."""

    def __init__(self, gpu, kv, n_seqs, max_pages, page, n_pages, h, n_kv, hd, tokens, n_sel=0):
        i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device=gpu)  # noqa: E731
        dt = {KV_I8: torch.int8, KV_I16: torch.int16, KV_F16: torch.float16,
              KV_F32: torch.float32}[kv]
        self.k, self.v = (torch.zeros(n_pages, n_kv, page, hd, dtype=dt, device=gpu)
                          for _ in range(2))
        self.ks, self.vs = (torch.zeros(n_pages, n_kv, page, device=gpu) for _ in range(2))
        self.bounds = torch.zeros(n_pages, n_kv, 2, hd, dtype=torch.float16, device=gpu)
        self.table, self.length = i32(n_seqs, max_pages), i32(n_seqs)
        self.free = torch.arange(n_pages, dtype=torch.int32, device=gpu).flip(0).contiguous()
        self.n_free, self.n_new, self.granted = i32(1).fill_(n_pages), i32(n_seqs), i32(n_seqs)
        self.start, self.taken = i32(n_seqs + 1), i32(n_seqs + 1)
        self.slot, self.pos, self.seq = i32(tokens), i32(tokens), i32(tokens)
        self.p = at.pages(self.k, self.v, self.ks, self.vs, kv_type=kv, table=self.table,
                          length=self.length, free=self.free, n_free=self.n_free,
                          bounds=self.bounds)
        self.cs, self.sn = (dev(x, gpu) for x in ph.rotation(max_pages * page, hd))
        self.kn, self.qn = torch.ones(hd, device=gpu) * 1.1, torch.ones(hd, device=gpu) * 0.9
        self.q = torch.zeros(tokens, h, hd, device=gpu)
        self.kk, self.vv = (torch.zeros(tokens, n_kv, hd, device=gpu) for _ in range(2))
        self.qr, self.out = torch.zeros_like(self.q), torch.zeros_like(self.q)
        self.sel = i32(n_seqs, n_kv, n_sel) if n_sel else None
        self.a = jm.Attention(h, n_kv, hd, 256)
        self.work = work_for(self.a, self.p, gpu)

    def step(self, stream=None):
        hd = self.q.shape[2]
        at.pages_plan(self.p, self.n_new, slot=self.slot, pos=self.pos, seq=self.seq,
                      start=self.start, taken=self.taken, granted=self.granted,
                      length=self.length, n_free=self.n_free, stream=stream)
        at.pages_write(self.p, self.kk, self.vv, slot=self.slot, pos=self.pos, cs=self.cs,
                       sn=self.sn, n_rot=hd, k_norm=self.kn, q=self.q, q_out=self.qr,
                       q_norm=self.qn, stream=stream)
        rows = dict(rows=self.start, granted=self.granted, work=self.work, stream=stream)
        if self.sel is not None:
            at.pages_bounds(self.p, self.granted, max_new=self.q.shape[0], stream=stream)
            self.a.select(self.p, self.qr, self.sel, **rows)
        self.a.run_pages(self.p, self.qr, self.out, sel=self.sel, **rows)


@pytest.mark.parametrize("kv", [KV_I8, KV_I16, KV_F16, KV_F32], ids=NAMES.get)
@pytest.mark.parametrize("n_sel", [0, 3])
def test_serving_steps(gpu, kv, n_sel):
    """Prompts admitted, tokens decoded, sequences released and admitted again
    in a pool too small for all: after each step the cached rows are bit for bit
    those of the contiguous cache, the single tokens' outputs those of
    janas_attn_run_dev over it within the float bar (with few blocks selected:
    of the plain choice and attention)."""
    n_seqs, page, h, n_kv, hd, tokens = 5, 16, 8, 2, 64, 90
    rng = np.random.default_rng([kv, n_sel])
    s = Server(gpu, kv, n_seqs, 12, page, 21, h, n_kv, hd, tokens, n_sel)
    steps = [[30, 0, 17, 0, 1]] + [[1, 25, 1, 0, 1]] + [[1, 1, 1, 1, 0]] * 9 + \
        [[1, -1, 1, 40, 1], [1, 30, 1, 1, -1]] + [[1, 1, 0, 1, 50]] + [[1, 1, 1, 1, 1]] * 20
    dt = s.k.dtype
    cache = [dict(k=torch.zeros(n_kv, 192, hd, dtype=dt, device=gpu),
                  v=torch.zeros(n_kv, 192, hd, dtype=dt, device=gpu),
                  ks=torch.zeros(n_kv, 192, device=gpu), vs=torch.zeros(n_kv, 192, device=gpu))
             for _ in range(n_seqs)]
    lens, refused, singles = [0] * n_seqs, 0, 0
    with jm.Attention(h, n_kv, hd, 192, 1, jm.FLOAT) as ref:
        for n_new in steps:
            for x in (s.q, s.kk, s.vv):
                x.copy_(torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)))
            s.n_new.copy_(torch.tensor(n_new, dtype=torch.int32))
            s.out.fill_(9.0)
            s.step()
            torch.cuda.synchronize()
            granted, t = s.granted.tolist(), 0
            for i, x in enumerate(n_new):
                if x == -1:
                    lens[i] = 0
                    continue
                refused += x > 0 and granted[i] == 0
                if granted[i]:
                    c, sl = cache[i], slice(t, t + x)
                    at.cache_write(at.cache(c["k"], c["v"], c["ks"], c["vs"], kv_type=kv),
                                   s.kk[sl].contiguous(), s.vv[sl].contiguous(),
                                   cs=s.cs[lens[i]:].contiguous(), sn=s.sn[lens[i]:].contiguous(),
                                   n_rot=hd, pos0=lens[i], k_norm=s.kn)
                    lens[i] += x
                    p = torch.arange(lens[i], device=gpu)
                    pg, r = s.table[i].long()[p // page], p % page
                    for name, y in (("k", s.k), ("v", s.v)):
                        assert torch.equal(y[pg, :, r].transpose(0, 1), c[name][:, :lens[i]])
                    if kv in ph.TOP:
                        assert torch.equal(s.ks[pg, :, r].t(), c["ks"][:, :lens[i]])
                    if x == 1:
                        singles += 1
                        if n_sel:
                            check_selected(s, c, kv, i, t, lens[i], page, n_sel)
                        else:
                            o = torch.zeros(1, h, hd, device=gpu)
                            ref.run_dev(kv, [dict(c, q=s.qr[t:t + 1].contiguous(), out=o, cap=192,
                                                  n=1, pos0=lens[i] - 1)])
                            torch.cuda.synchronize()
                            err = float((o[0] - s.out[t]).abs().max())
                            assert within(err, TOL_FLOAT_ABS, f"seq {i} len {lens[i]}")
                    else:
                        assert bool((s.out[sl] == 9.0).all())
                t += x
            assert s.length.tolist() == lens
    s.a.close()
    assert refused and singles > 60


def check_selected(s, c, kv, i, t, n, page, n_sel):
    k, v = (c[x][:, :n].cpu().numpy().astype(np.float64) for x in ("k", "v"))
    if kv in ph.TOP:
        k, v = (x * c[z][:, :n].cpu().numpy().astype(np.float64)[..., None]
                for x, z in ((k, "ks"), (v, "vs")))
    q = s.qr[t].cpu().numpy()
    g, nb = q.shape[0] // k.shape[0], ph.blocks(n, page)
    seen = []
    for kh in range(k.shape[0]):
        k32 = k[kh].astype(np.float32)
        boxes = np.stack([np.stack((ph.outward(k32[b * page:(b + 1) * page].min(0), False),
                                    ph.outward(k32[b * page:(b + 1) * page].max(0), True)))
                          for b in range(nb)])
        want = ph.choose(q[kh * g:(kh + 1) * g], boxes, n, 0, page, n_sel, 1, 1)
        assert np.array_equal(s.sel[i, kh].cpu().numpy(), want)
        seen.append(np.array([p for b in want if b >= 0 for p in range(b * page, (b + 1) * page)
                              if p < n]))
    ref, bar = ph.attend(q, k.transpose(1, 0, 2), v.transpose(1, 0, 2), ph.default_scale(64), seen)
    assert (np.abs(s.out[t].cpu().numpy() - ref).max(1) <= bar).all()


def test_a_captured_step_replays(gpu):
    """A step captured into a graph once and replayed as the sequences grow past
    pages, with another step's eager calls between the replays: each replay's
    tables, rows and outputs those of the same steps made eagerly."""
    args = (gpu, KV_I8, 4, 8, 16, 24, 8, 2, 64, 6, 3)
    s, e, other = Server(*args), Server(*args), Server(*args)
    n_new = torch.tensor([1, 1, 0, 1], dtype=torch.int32, device=gpu)
    for x in (s, e, other):
        x.n_new.copy_(n_new)
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        s.step(st.cuda_stream)      # (once outside the capture)
    torch.cuda.synchronize()
    e.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        s.step(torch.cuda.current_stream().cuda_stream)
    g = torch.Generator(device=gpu).manual_seed(9)
    for i in range(40):
        for x, y in ((s.q, e.q), (s.kk, e.kk), (s.vv, e.vv)):
            x.copy_(torch.randn(x.shape, generator=g, device=gpu))
            y.copy_(x)
        if i == 20:
            for x in (s, e):
                x.n_new.copy_(torch.tensor([1, -1, 1, 1], dtype=torch.int32))
        if i == 21:
            for x in (s, e):
                x.n_new.copy_(n_new)
        torch.cuda.synchronize()
        other.step()
        with torch.cuda.stream(st):
            graph.replay()
        torch.cuda.synchronize()
        e.step()
        torch.cuda.synchronize()
        for name in ("table", "length", "n_free", "slot", "pos", "k", "v", "ks", "vs", "bounds",
                     "sel", "qr", "out"):
            assert torch.equal(getattr(s, name), getattr(e, name)), (i, name)
    assert s.length.tolist()[0] == 41
    for x in (s, e, other):
        x.a.close()


def test_two_calls_at_once(gpu):
    """Calls of one instance on two streams, each with work of its own."""
    h, n_kv, hd, page = 8, 2, 128, 64
    rng = np.random.default_rng(10)
    pools = [ph.Pool(rng, KV_F16, [5000, 300, 2000], page, n_kv, hd) for _ in range(2)]
    q = rng.standard_normal((3, h, hd)).astype(np.float32)
    want = [run_pages(gpu, p, h, q) for p in pools]
    gs = [OnGpu(p, gpu) for p in pools]
    outs = [torch.zeros(3, h, hd, device=gpu) for _ in range(2)]
    qd, streams = dev(q, gpu), [torch.cuda.Stream() for _ in range(2)]
    with jm.Attention(h, n_kv, hd, 256) as a:
        calls = [a.prepare_pages(g.p, qd, o, work=work_for(a, g.p, gpu), stream=st.cuda_stream)
                 for g, o, st in zip(gs, outs, streams)]
        torch.cuda.synchronize()
        for _ in range(20):
            for c in calls:
                c()
        torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert np.array_equal(o.cpu().numpy(), w)


def test_offsets_past_32_bits(gpu):
    """A pool of more than 4 GiB a tensor: rows at its far end."""
    h, n_kv, hd, page = 2, 1, 512, 256
    n_pages = (1 << 32) // (page * hd * 2) + 40
    k = torch.zeros(n_pages, n_kv, page, hd, dtype=torch.float16, device=gpu)
    v = torch.zeros(n_pages, n_kv, page, hd, dtype=torch.float16, device=gpu)
    bounds = torch.zeros(n_pages, n_kv, 2, hd, dtype=torch.float16, device=gpu)
    rng = np.random.default_rng(11)
    far = np.array([n_pages - 1, n_pages - 7, n_pages - 3, 0], np.int32)
    table, length = dev(far[None], gpu), torch.tensor([600], dtype=torch.int32, device=gpu)
    p = at.pages(k, v, kv_type=KV_F16, table=table, length=length, bounds=bounds)
    kk, vv = (rng.standard_normal((600, 1, hd)).astype(np.float32) for _ in range(2))
    t = np.arange(600)
    slot = far[t // page] * page + t % page
    at.pages_write(p, dev(kk, gpu), dev(vv, gpu), slot=dev(slot.astype(np.int32), gpu))
    q = rng.standard_normal((1, h, hd)).astype(np.float32)
    out = torch.zeros(1, h, hd, device=gpu)
    with jm.Attention(h, n_kv, hd, 256) as a:
        a.run_pages(p, dev(q, gpu), out, work=work_for(a, p, gpu))
    at.pages_bounds(p)
    torch.cuda.synchronize()
    k16, v16 = (x.astype(np.float16).astype(np.float64) for x in (kk, vv))
    want, bar = ph.attend(q[0], k16, v16, ph.default_scale(hd), [t])
    assert (np.abs(out[0].cpu().numpy() - want).max(1) <= bar).all()
    assert np.array_equal(bounds[n_pages - 7, 0, 0].cpu().numpy(),
                          k16[256:512, 0].min(0).astype(np.float16))
