"""Which pools the paged calls of an instance take, over a made-up device
(pages_calls.cpp): janas_attn_pages_work_bytes gives 0 for those that
janas_attn_pages_run refuses by the pool's and the instance's sizes alone, and,
with bounds set, for those that janas_attn_pages_select refuses."""
import ctypes
import os
import random
import subprocess

import pytest

import janas_amd as jm
from janas_amd import attention as at
from janas_amd.build import LIB, ROOT

CLANG = "/opt/rocm/llvm/bin/clang++"
A = 1 << 20       # an aligned address that is never read
MOST = (1 << 64) - 1


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    jm.lib()
    so = str(tmp_path_factory.mktemp("pages") / "pages_calls.so")
    libdir = os.path.dirname(LIB)
    subprocess.run([CLANG, "-std=c++17", "-O1", "-shared", "-fPIC", "-D__HIP_PLATFORM_AMD__",
                    "-I/opt/rocm/include", "-I", os.path.join(ROOT, "include"),
                    "-Wno-unused-result", os.path.join(ROOT, "tests", "pages_calls.cpp"), "-o", so,
                    "-Wl,-Bsymbolic", "-L", libdir, "-ljanas_attn", f"-Wl,-rpath,{libdir}",
                    "-Wl,-rpath,/opt/rocm/lib"], check=True)
    L = ctypes.CDLL(so)
    vp, u32 = ctypes.c_void_p, ctypes.c_uint32
    L.made_up.argtypes, L.made_up.restype = [u32, u32, u32, ctypes.c_int], vp
    L.janas_attn_pages_work_bytes.argtypes = [vp, ctypes.POINTER(at.Pages)]
    L.janas_attn_pages_work_bytes.restype = ctypes.c_size_t
    L.janas_attn_pages_run.argtypes = [vp, ctypes.POINTER(at.Pages), ctypes.c_int,
                                       ctypes.POINTER(at.PagesCall), vp]
    L.janas_attn_pages_select.argtypes = [vp, ctypes.POINTER(at.Pages),
                                          ctypes.POINTER(at.PagesCall), u32, u32, vp, vp]
    L.janas_attn_pages_bounds.argtypes = [ctypes.POINTER(at.Pages), vp, u32, vp]
    return L


def pool(**over):
    d = dict(k=A, v=A, ks=A, vs=A, bounds=A, n_kv=2, head_dim=64, kv_type=jm.KV_I8, page=16,
             n_pages=8, n_seqs=3, max_pages=4, table=A, len=A, dev=0)
    d.update(over)
    return at.Pages(**d)


def answers(L, h, p, ring=0, work=MOST):
    """(bytes, run's code, select's code); a refused call launches nothing."""
    a = L.made_up(h, p.n_kv, p.head_dim, ring)
    c = at.PagesCall(q=A, out=A, work=A, work_bytes=work, n_sel=4)
    size, before = L.janas_attn_pages_work_bytes(a, ctypes.byref(p)), L.launched()
    run = L.janas_attn_pages_run(a, ctypes.byref(p), 0, ctypes.byref(c), None)
    assert L.launched() - before == (0 if run else 2)
    sel = L.janas_attn_pages_select(a, ctypes.byref(p), ctypes.byref(c), 1, 1, A, None)
    assert L.launched() - before == (0 if run else 2) + (0 if sel else 1)
    return size, run, sel


@pytest.mark.parametrize("over,run,sel", [
    (dict(), jm.OK, jm.OK),
    # 2^30 units of 16 positions, and one table row fewer: a workgroup may have
    # them all, and a wave's share of them is (units x 3) / 4 and (units x 4) / 4
    # in 32 bits
    (dict(n_seqs=1 << 10, max_pages=1 << 20), jm.ERANGE, jm.OK),
    (dict(n_seqs=(1 << 10) - 1, max_pages=1 << 20), jm.OK, jm.OK),
    (dict(n_seqs=1 << 7, max_pages=1 << 20, page=128), jm.ERANGE, jm.OK),
    # more blocks than a selection takes
    (dict(max_pages=(1 << 20) + 1), jm.OK, jm.ERANGE),
    # more workgroups than a launch takes: the merge's, the selection's
    (dict(n_seqs=65535, n_kv=512, head_dim=64), jm.ERANGE, jm.ERANGE),
    (dict(n_seqs=65535, n_kv=64), jm.OK, jm.OK),
    (dict(n_seqs=65535, n_kv=65), jm.OK, jm.ERANGE)])
@pytest.mark.parametrize("bounds", [A, None])
def test_work_bytes_is_0_where_a_call_is_refused(calls, over, run, sel, bounds):
    p = pool(bounds=bounds, **over)
    size, got, picked = answers(calls, p.n_kv, p)
    assert got == run and picked == (sel if bounds else jm.EINVAL)
    assert (size == 0) == (run != jm.OK or (bounds is not None and sel != jm.OK))
    if size:
        # (of that size, and none smaller)
        assert answers(calls, p.n_kv, p, work=size)[1:] == (got, picked)
        alone = answers(calls, p.n_kv, pool(**dict(over, bounds=None)))[0]
        assert answers(calls, p.n_kv, p, work=alone - 1)[1] == jm.ERANGE


def test_work_bytes_and_the_calls_agree(calls):
    """Pools of all sizes up to the structure's own limits."""
    rng, both = random.Random(3), [0, 0, 0]
    log = lambda lo, hi: int(2 ** rng.uniform(lo, hi))  # noqa: E731
    for _ in range(20000):
        kv = rng.randrange(4)
        hd, page = 8 * log(1, 5.01), 16 << rng.randrange(5)
        p = pool(kv_type=kv, head_dim=hd, page=page, n_kv=log(0, 10), n_seqs=log(0, 15.99),
                 max_pages=log(0, 22), n_pages=log(0, 22), bounds=rng.choice((A, None)))
        size, run, sel = answers(calls, p.n_kv * log(0, 6), p, ring=rng.random() < 0.02)
        refused = run != jm.OK or (p.bounds is not None and sel != jm.OK)
        assert (size == 0) == refused, (size, run, sel, [(x, getattr(p, x)) for x, _ in p._fields_])
        both[0 if not refused else 1 if run else 2] += 1
    assert min(both) > 100, both


@pytest.mark.parametrize("n_seqs,n_kv,hd,code", [
    (65535, 256, 128, jm.OK), (65535, 257, 128, jm.ERANGE), (65535, 128, 136, jm.OK),
    (65535, 129, 136, jm.ERANGE), (65535, 64, 512, jm.OK), (65535, 65, 512, jm.ERANGE),
    (1, 65535, 512, jm.OK)])
def test_bounds_take_what_a_launch_holds(calls, n_seqs, n_kv, hd, code):
    """Below 2^24 workgroups of 256 threads, one for every 128 columns."""
    p, before = pool(n_seqs=n_seqs, n_kv=n_kv, head_dim=hd), calls.launched()
    assert calls.janas_attn_pages_bounds(ctypes.byref(p), A, 1, None) == code
    assert calls.launched() - before == (code == jm.OK)
