"""The plain form of the paged cache's write (perf/operators.py) makes 8- and
16-bit rows by the cache write's rule: one quotient for a row's multiplier, one
for its scale, each rounded once."""
import numpy as np
import pytest
import torch

import pages_helpers as ph
from perf import operators as op


@pytest.mark.parametrize("kv", ["i8", "i16"])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda:0", marks=pytest.mark.gpu)])
def test_quantization_is_one_quotient(kv, device):
    rng = np.random.default_rng(op.KIND[kv])
    x = rng.standard_normal((20000, 128)).astype(np.float32)
    x[7] = 0.0
    x[8], x[9, 1:] = 1.1, 0.0
    want, scale = ph.quantize(x, op.KIND[kv])
    got, z = op._quant(torch.from_numpy(x).to(device), kv)
    assert np.array_equal(got.cpu().numpy(), want)
    assert np.array_equal(z.cpu().numpy(), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("kv", ["i8", "i16"])
@pytest.mark.parametrize("heads", op.HEADS, ids=lambda x: "-".join(map(str, x)))
def test_write_and_its_plain_form(gpu, kv, heads):
    """The framework's call and its plain form leave the same whole numbers and
    scales in the pool, and what the definition says of them is equal too."""
    h, n_kv, hd = heads
    case = op._case("write", h=h, n_kv=n_kv, hd=hd, kv=kv, seqs=9, length=300, new=900, page=32,
                    pad=3)
    res = []
    try:
        for own in (True, False):
            op.own = own
            res.append([x.clone() for x in op.run(op.prepare(case, 5))])
    finally:
        op.own = False
    torch.cuda.synchronize()
    for x, y in zip(res[0][:4], res[1][:4]):      # k, v and their scales
        assert x.dtype == y.dtype and torch.equal(x, y), int((x != y).sum())
    exact = op.exact(case, 5)
    assert exact[0] is None and torch.equal(res[0][1], exact[1])
