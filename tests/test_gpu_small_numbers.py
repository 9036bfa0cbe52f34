"""Query rows and value scales far below one: the planes' power of two stays a
number. Query rows down to subnormal numbers, beside ordinary rows and rows of
zeros; every kernel that takes the query as planes, over every cache type, at
head sizes that fill their tiles and that do not. All scores are then next to 0
and a row is the mean of the values in sight."""
import numpy as np
import pytest
import torch

import janas_amd as jm
import pages_helpers as ph
from attn_helpers import within
from janas_amd import attention as at

pytestmark = pytest.mark.gpu

KV_I8, KV_I16, KV_F16, KV_F32 = jm.KV_I8, jm.KV_I16, jm.KV_F16, jm.KV_F32
NAMES = {KV_I8: "i8", KV_I16: "i16", KV_F16: "f16", KV_F32: "f32"}
# around 2^-114, where 2^14 over the row's largest number leaves the floats,
# below the normal floats, and the smallest of all
SIZES = (2.0 ** -112, 2.0 ** -114, 4e-35, 1e-36, 1e-38, 1e-42, 2.0 ** -149, 0.0)
CASES = [(kv, hd) for kv in NAMES for hd in (64, 72, 128, 256, 384, 512)
         if hd <= 256 or kv != KV_F32]


def queries(rng, n, h, hd):
    """Rows of each size, with zeros among their numbers; the last head's are of
    ordinary size."""
    q = rng.uniform(-1, 1, (n, h, hd))
    q[..., 0] = 1.0
    q[..., 3::5] = 0.0
    size = np.array(SIZES)[np.arange(n * h).reshape(n, h) % len(SIZES)]
    size[:, -1] = 1.0
    return (q * size[..., None]).astype(np.float32)


def check(pool, q, out, what, seen=None):
    for i, n in enumerate(pool.lens):
        for t in range(q.shape[1]):
            sight = np.arange(n if seen is None else seen(n, t))
            want, bar = ph.attend(q[i, t], pool.rows("k", i), pool.rows("v", i),
                                  ph.default_scale(pool.hd), [sight] * pool.n_kv)
            err = np.abs(out[i, t] - want).max(1)
            worst = int(np.argmax(err / bar))
            assert np.isfinite(out[i, t]).all(), (i, t, out[i, t])
            assert within(err[worst], bar[worst], f"{what} len {n} head {worst}"), (err, bar)


@pytest.mark.parametrize("kv,hd", CASES, ids=lambda x: str(x))
def test_pages(gpu, kv, hd):
    h, n_kv, page = 10, 1, 16
    rng = np.random.default_rng([kv, hd])
    pool = ph.Pool(rng, kv, [1, 16, 100, 3000], page, n_kv, hd)
    q = queries(rng, len(pool.lens), h, hd)
    dev = lambda x: None if x is None else torch.from_numpy(x).to(gpu)  # noqa: E731
    k, v, ks, vs = (dev(x) for x in (pool.k, pool.v, pool.ks, pool.vs))
    p = at.pages(k, v, ks, vs, kv_type=kv, table=dev(pool.table),
                 length=dev(np.array(pool.lens, np.int32)))
    out = torch.zeros(q.shape, device=gpu)
    with jm.Attention(h, n_kv, hd, 256) as a:
        work = torch.empty(a.pages_work_bytes(p), dtype=torch.uint8, device=gpu)
        a.run_pages(p, dev(q), out, work=work)
        torch.cuda.synchronize()
    check(pool, q[:, None], out.cpu().numpy()[:, None], f"pages {NAMES[kv]} {hd}")


def run_contiguous(gpu, pool, q, kv, cap=1100):
    """The split kernels (head sizes to 256, and above) over the pool's one
    sequence of 1000 rows, the last of q's tokens at its end."""
    dev = lambda x: torch.from_numpy(x).to(gpu)  # noqa: E731
    rows, p = {}, np.arange(1000)
    for name, x in (("k", pool.k), ("v", pool.v), ("ks", pool.ks), ("vs", pool.vs)):
        if x is None:
            continue
        y = np.zeros((pool.n_kv, cap) + x.shape[3:], x.dtype)
        y[:, :1000] = np.moveaxis(x[pool.table[0, p // 256], :, p % 256], 0, 1)
        rows[name] = dev(y)
    n, h = q.shape[:2]
    out = torch.zeros(q.shape, device=gpu)
    with jm.Attention(h, pool.n_kv, pool.hd, cap, 1, jm.FLOAT) as a:
        a.run_dev(kv, [dict(rows, q=dev(q), out=out, cap=cap, n=n, pos0=1000 - n)], path="split")
        torch.cuda.synchronize()
    return out.cpu().numpy()


# (f32 rows above 128 are refused)
@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("kv,hd", [(kv, hd) for kv, hd in CASES if kv != KV_F32 or hd <= 128],
                         ids=lambda x: str(x))
def test_contiguous(gpu, kv, hd, n):
    h = 10
    rng = np.random.default_rng([kv, hd, n])
    pool = ph.Pool(rng, kv, [1000], 256, 1, hd)
    q = queries(rng, n, h, hd)
    check(pool, q[None], run_contiguous(gpu, pool, q, kv)[None], f"split {NAMES[kv]} {hd}",
          seen=lambda m, t: m - n + t + 1)


@pytest.mark.parametrize("down", [100, 108, 110, 112])
@pytest.mark.parametrize("kv,hd", [(kv, hd) for kv, hd in CASES if kv in ph.TOP],
                         ids=lambda x: str(x))
def test_contiguous_value_scales(gpu, kv, hd, down):
    """Scales of N(0, 1) rows times 2^-down: on both sides of 2^-115 (int8, 2^-5
    of a number; int16 2^-13), all numbers normal floats."""
    down -= 8 if kv == KV_I16 else 0
    rng = np.random.default_rng([kv, hd, down])
    pool = ph.Pool(rng, kv, [1000], 256, 1, hd)
    pool.vs *= np.float32(2.0 ** -down)
    q = rng.standard_normal((1, 10, hd)).astype(np.float32)
    check(pool, q[None], run_contiguous(gpu, pool, q, kv)[None], f"scales {NAMES[kv]} {hd}")
