"""Query rows far below one, down to subnormal numbers, beside ordinary rows and
rows of zeros: the planes' power of two stays a number. Every kernel that takes
the query as planes, over every cache type, at head sizes that fill their tiles
and that do not. All scores are then next to 0 and a row is the mean of the
values in sight."""
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


# (f32 rows above 128 are refused)
@pytest.mark.parametrize("n", [1, 3])
@pytest.mark.parametrize("kv,hd", [(kv, hd) for kv, hd in CASES if kv != KV_F32 or hd <= 128],
                         ids=lambda x: str(x))
def test_contiguous(gpu, kv, hd, n):
    """The split kernels (head sizes to 256, and above)."""
    h, n_kv, cap = 10, 1, 1100
    rng = np.random.default_rng([kv, hd, n])
    pool = ph.Pool(rng, kv, [1000], 256, n_kv, hd)
    pool.table = pool.table[:, :4]
    q = queries(rng, n, h, hd)[None]
    dev = lambda x: None if x is None else torch.from_numpy(x).to(gpu)  # noqa: E731
    rows = {}
    for name, x in (("k", pool.k), ("v", pool.v), ("ks", pool.ks), ("vs", pool.vs)):
        if x is None:
            continue
        y = np.zeros((n_kv, cap) + x.shape[3:], x.dtype)
        p = np.arange(1000)
        y[:, :1000] = np.moveaxis(x[pool.table[0, p // 256], :, p % 256], 0, 1)
        rows[name] = dev(y)
    out = torch.zeros(q.shape[1:], device=gpu)
    with jm.Attention(h, n_kv, hd, cap, 1, jm.FLOAT) as a:
        a.run_dev(kv, [dict(rows, q=dev(q[0]), out=out, cap=cap, n=n, pos0=1000 - n)], path="split")
        torch.cuda.synchronize()
    check(pool, q, out.cpu().numpy()[None], f"split {NAMES[kv]} {hd}",
          seen=lambda m, t: m - n + t + 1)
