"""Part 4's entry points on the CPU: what they refuse, before any device call,
and the plain rules that the GPU tests compare with."""
import ctypes

import numpy as np
import pytest

import janas_amd as jm
import pages_helpers as ph
from janas_amd import attention as at

A = 1 << 20       # an aligned address that is never read


def pool(**over):
    d = dict(k=A, v=A, ks=A, vs=A, bounds=A, n_kv=2, head_dim=64, kv_type=jm.KV_I8, page=16,
             n_pages=8, n_seqs=3, max_pages=4, table=A, len=A, free_pages=A, n_free=A, dev=0)
    d.update(over)
    return at.Pages(**d)


def plan(**over):
    d = dict(n_new=A, len=A, n_free=A, granted=A, start=A, taken=A, slot=A, pos=A, seq=A,
             max_tokens=9)
    d.update(over)
    return at.Plan(**d)


def rows(**over):
    d = dict(k=A, v=A, q=A, q_out=A, k_norm=A, q_norm=A, cs=A, sn=A, slot=A, pos=A, eps=1e-6,
             n_rot=64, n_tab=100, v_norm=0, n=5, n_head=4, k_stride=0, v_stride=0, q_stride=0)
    d.update(over)
    return at.Rows(**d)


TABLES = [(dict(table=None), jm.EINVAL), (dict(len=None), jm.EINVAL), (dict(page=8), jm.EINVAL),
          (dict(page=48), jm.EINVAL), (dict(page=512), jm.EINVAL), (dict(page=0), jm.EINVAL),
          (dict(n_pages=0), jm.EINVAL), (dict(n_seqs=0), jm.EINVAL),
          (dict(n_seqs=65536), jm.EINVAL), (dict(max_pages=0), jm.EINVAL),
          (dict(dev=-1), jm.EINVAL), (dict(n_pages=1 << 27), jm.ERANGE),
          (dict(max_pages=1 << 27), jm.ERANGE)]
POOL = [(dict(k=None), jm.EINVAL), (dict(v=None), jm.EINVAL), (dict(ks=None), jm.EINVAL),
        (dict(vs=None), jm.EINVAL), (dict(n_kv=0), jm.EINVAL), (dict(n_kv=70000), jm.EINVAL),
        (dict(head_dim=0), jm.EINVAL), (dict(head_dim=60), jm.EINVAL),
        (dict(head_dim=520), jm.EINVAL), (dict(kv_type=4), jm.EINVAL),
        (dict(kv_type=-1), jm.EINVAL), (dict(k=A + 8), jm.EINVAL), (dict(vs=A + 4), jm.EINVAL),
        (dict(bounds=A + 2), jm.EINVAL)]


@pytest.mark.parametrize("over,code", TABLES)
def test_plan_refuses_tables(over, code):
    assert at.lib().janas_attn_pages_plan(ctypes.byref(pool(**over)), ctypes.byref(plan()),
                                          None) == code


@pytest.mark.parametrize("over,code", [
    (dict(n_new=None), jm.EINVAL), (dict(len=None), jm.EINVAL), (dict(n_free=None), jm.EINVAL),
    (dict(granted=None), jm.EINVAL), (dict(start=None), jm.EINVAL), (dict(taken=None), jm.EINVAL),
    (dict(slot=None), jm.EINVAL), (dict(pos=None), jm.EINVAL), (dict(seq=None), jm.EINVAL),
    (dict(max_tokens=1 << 31), jm.ERANGE)])
def test_plan_refuses_a_step(over, code):
    f = at.lib().janas_attn_pages_plan
    assert f(ctypes.byref(pool()), ctypes.byref(plan(**over)), None) == code
    assert f(None, ctypes.byref(plan()), None) == jm.EINVAL
    assert f(ctypes.byref(pool()), None, None) == jm.EINVAL
    assert f(ctypes.byref(pool(free_pages=None)), ctypes.byref(plan()), None) == jm.EINVAL
    assert f(ctypes.byref(pool(n_free=None)), ctypes.byref(plan()), None) == jm.EINVAL


@pytest.mark.parametrize("over,code", TABLES + POOL)
def test_write_and_bounds_refuse_a_pool(over, code):
    p = ctypes.byref(pool(**over))
    assert at.lib().janas_attn_pages_write(p, ctypes.byref(rows()), None) == code
    assert at.lib().janas_attn_pages_bounds(p, None, 0, None) == code


@pytest.mark.parametrize("over", [
    dict(k=None), dict(v=None), dict(slot=None), dict(pos=None), dict(cs=None), dict(sn=None),
    dict(n_tab=0), dict(n_rot=63), dict(n_rot=66), dict(q_out=None), dict(n_head=0),
    dict(k_stride=127), dict(v_stride=1), dict(q_stride=255), dict(q_stride=260)])
def test_write_refuses_rows(over):
    # (q_stride 260: queries in place that are not packed)
    f = at.lib().janas_attn_pages_write
    assert f(ctypes.byref(pool()), ctypes.byref(rows(**over)), None) == jm.EINVAL
    assert f(ctypes.byref(pool()), None, None) == jm.EINVAL
    assert f(None, ctypes.byref(rows()), None) == jm.EINVAL


def test_write_of_no_rows_and_too_many():
    f = at.lib().janas_attn_pages_write
    assert f(ctypes.byref(pool()), ctypes.byref(rows(n=0)), None) == jm.OK
    assert f(ctypes.byref(pool()), ctypes.byref(rows(n=1 << 31)), None) == jm.ERANGE
    # (an empty tensor has no address)
    none = at.Rows(n=0, n_rot=64)
    assert f(ctypes.byref(pool()), ctypes.byref(none), None) == jm.OK


def test_bounds_need_their_array():
    assert at.lib().janas_attn_pages_bounds(ctypes.byref(pool(bounds=None)), None, 0,
                                            None) == jm.EINVAL


def test_bounds_refuse_more_workgroups_than_a_launch_takes():
    # 65535 sequences of 257 KV heads: 2^24 workgroups and more
    p = pool(n_seqs=65535, n_kv=257)
    assert at.lib().janas_attn_pages_bounds(ctypes.byref(p), A, 1, None) == jm.ERANGE


def test_run_and_select_need_an_instance():
    L, p, c = at.lib(), ctypes.byref(pool()), at.PagesCall(q=A, out=A, work=A, work_bytes=1 << 30)
    assert L.janas_attn_pages_run(None, p, 0, ctypes.byref(c), None) == jm.EINVAL
    assert L.janas_attn_pages_select(None, p, ctypes.byref(c), 1, 1, A, None) == jm.EINVAL
    assert L.janas_attn_pages_work_bytes(None, p) == 0


def test_python_checks_tensors():
    import torch
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    f32 = lambda *s: torch.zeros(s)  # noqa: E731
    t = dict(table=i32(3, 4), length=i32(3))
    k = torch.zeros(8, 2, 16, 64, dtype=torch.float16)
    p = at.pages(k, k, kv_type=jm.KV_F16, **t)
    assert (p.n_pages, p.n_kv, p.page, p.head_dim, p.n_seqs, p.max_pages) == (8, 2, 16, 64, 3, 4)
    bad = [lambda: at.pages(k, k, kv_type=jm.KV_I8, **t),
           lambda: at.pages(k, k[:7], kv_type=jm.KV_F16, **t),
           lambda: at.pages(k[:, :, ::2], k[:, :, ::2], kv_type=jm.KV_F16, **t),
           lambda: at.pages(k, k, kv_type=jm.KV_F16, table=i32(3, 4).long(), length=i32(3)),
           lambda: at.pages(k, k, kv_type=jm.KV_F16, table=i32(3, 4), length=i32(4)),
           lambda: at.pages(k, k, kv_type=jm.KV_F16, bounds=f32(8, 2, 2, 64), **t),
           lambda: at.pages(k, k, kv_type=jm.KV_F16, free=i32(7), **t),
           lambda: at.prepare_pages_write(p, f32(5, 2, 64), f32(5, 2, 64), slot=i32(4)),
           lambda: at.prepare_pages_write(p, f32(5, 2, 64), f32(4, 2, 64), slot=i32(5)),
           lambda: at.prepare_pages_write(p, f32(1, 2, 64).expand(5, 2, 64), f32(5, 2, 64),
                                          slot=i32(5)),
           lambda: at.prepare_pages_write(p, f32(5, 2, 128)[:, :, ::2], f32(5, 2, 64),
                                          slot=i32(5)),
           lambda: at.prepare_pages_bounds(p, i32(2)),
           lambda: at.prepare_pages_plan(p, i32(3), slot=i32(9), pos=i32(8), seq=i32(9),
                                         start=i32(4), taken=i32(4), granted=i32(3),
                                         length=i32(3), n_free=i32(1)),
           lambda: at.prepare_pages_plan(p, i32(3), slot=i32(9), pos=i32(9), seq=i32(9),
                                         start=i32(3), taken=i32(4), granted=i32(3),
                                         length=i32(3), n_free=i32(1))]
    for f in bad:
        with pytest.raises(ValueError):
            f()


def test_python_refuses_other_devices():
    import torch
    k = torch.zeros(8, 2, 16, 64, dtype=torch.float16)
    x, slot = torch.zeros(5, 2, 64), torch.zeros(5, dtype=torch.int32)
    t = dict(table=torch.zeros(3, 4, dtype=torch.int32), length=torch.zeros(3, dtype=torch.int32))
    p = at.pages(k, k, kv_type=jm.KV_F16, **t)
    with pytest.raises(ValueError, match="host memory"):
        at.pages_write(p, x, x, slot=slot)
    with pytest.raises(ValueError, match="cpu, meta"):
        at.prepare_pages_write(p, x, x, slot=slot.to("meta"))
    with pytest.raises(ValueError, match="cpu, meta"):
        at.prepare_pages_bounds(at.pages(k, k, kv_type=jm.KV_F16, table=t["table"].to("meta"),
                                         length=t["length"]))


def test_python_refuses_strides_past_32_bits():
    """The structures hold them in 32 bits: 2^32 + 128 would be 128."""
    import torch
    far = lambda n: torch.empty_strided((2, n, 64), ((1 << 32) + 64 * n, 64, 1),  # noqa: E731
                                        device="meta")
    near = lambda n: torch.empty(2, n, 64, device="meta")  # noqa: E731
    k = torch.empty(8, 2, 16, 64, dtype=torch.float16, device="meta")
    slot = torch.empty(2, dtype=torch.int32, device="meta")
    t = dict(table=torch.empty(2, 4, dtype=torch.int32, device="meta"),
             length=torch.empty(2, dtype=torch.int32, device="meta"))
    p = at.pages(k, k, kv_type=jm.KV_F16, **t)
    at.prepare_pages_write(p, near(2), near(2), slot=slot, q=near(4))
    for x in (dict(k=far(2)), dict(v=far(2)), dict(q=far(4), q_out=near(4))):
        x = dict(dict(k=near(2), v=near(2), q=near(4)), **x)
        with pytest.raises(ValueError, match="32 bits"):
            at.prepare_pages_write(p, x.pop("k"), x.pop("v"), slot=slot, **x)


def test_plain_plan_keeps_pages_apart():
    """The restatement itself: over random steps every page is in one place -
    the free ones or one table row - and none is lost."""
    rng = np.random.default_rng(3)
    page, n_pages, n_seqs = 16, 40, 6
    table = np.zeros((n_seqs, 9), np.int32)
    s = dict(table=table, free=rng.permutation(n_pages).astype(np.int32),
             n_free=np.array([n_pages]), length=np.zeros(n_seqs, np.int32))
    for _ in range(60):
        n_new = rng.integers(0, 50, n_seqs)
        n_new[rng.random(n_seqs) < 0.2] = ph.NONE
        s = ph.plan(s["table"], s["free"], s["n_free"][0], s["length"], n_new, page, 200)
        held = [s["table"][i, b] for i in range(n_seqs)
                for b in range(ph.blocks(int(s["length"][i]), page))]
        assert sorted(held + list(s["free"][:s["n_free"][0]])) == list(range(n_pages))
        live = s["slot"][s["slot"] >= 0]
        assert len(set(live)) == len(live) == s["granted"].sum()
