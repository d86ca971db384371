"""What the paged attention rounds on the way, and what of it must not show."""
import math

import pytest
import torch

from paged_ref import Batch, compare
from test_paged_gpu import BF16, F16, context

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shape", [dict(nh=4, nkv=2, hd=64), dict(nh=4, nkv=1, hd=128)], ids=["hd64", "hd128"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows", [1, 3, 60])
def test_infinite_values_that_every_row_sees(cuda, rows, shape, dtype):
    """The results are what the formula has: infinite of the value's sign, NaN
    for NaN, other elements as they would be."""
    import ter_amd as T
    seqs = [(rows, rows + 100), (rows, rows + 2500), (rows, rows + 30)]
    b = Batch(seqs, dtype=dtype, seed=9, page=16, **shape)
    want, tol = b.attend()
    for s in range(3):
        for p, d, val in ((3, 0, math.inf), (20, 5, -math.inf), (9, b.hd - 1, math.nan)):
            b.v[b.table[s, p // 16], p % 16, :, d] = val
    cache, batch = b.on_device(T)
    out = context(b).attend(b.q.cuda(), cache, batch).cpu()
    assert (out[..., 0] == math.inf).all() and (out[..., 5] == -math.inf).all() and torch.isnan(out[..., b.hd - 1]).all()
    keep = [d for d in range(b.hd) if d not in (0, 5, b.hd - 1)]
    compare(out[..., keep], want[..., keep], tol[..., keep])


@pytest.mark.parametrize("shape", [dict(nh=4, nkv=2, hd=64), dict(nh=4, nkv=1, hd=128)], ids=["hd64", "hd128"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("rows,shared", [(1, 0), (3, 0), (60, 0), (1, 64), (60, 64)])
@pytest.mark.parametrize("power", [50, 200])
def test_infinite_values_of_vanishing_weight(cuda, power, rows, shared, shape, dtype):
    """A weight of 2^-50 or 2^-200 of the largest is not zero, whatever it is
    rounded to on the way: the result is infinite."""
    import ter_amd as T
    seqs = [(rows, rows + 100), (rows, rows + 2500), (rows, rows + 230)]
    b = Batch(seqs, dtype=dtype, seed=10, page=16, common=shared, **shape)
    b.q = b.q.abs() + 0.5
    q = b.q.double().sum(-1)
    for s in range(3):
        at = (b.table[s, 0], 3)
        b.k[at] = -power * math.log(2) * math.sqrt(b.hd) / float(q.mean())
        b.v[(*at, slice(None), 7)] = math.inf
    low = [float(x) for s in range(3) for x in (b.q.double() @ b.k[b.table[s, 0], 3, 0].double()).aminmax()]
    # scores of that position, e-fold: beyond what fp16 holds beside a largest weight, not beyond binary64
    assert -600 < min(low) / math.sqrt(b.hd) and max(low) / math.sqrt(b.hd) < -24
    cache, batch = b.on_device(T)
    out = context(b).attend(b.q.cuda(), cache, batch, shared=shared).cpu()
    assert (out[..., 7] == math.inf).all()
    keep = [d for d in range(b.hd) if d != 7]
    want, tol = b.attend()
    compare(out[..., keep], want[..., keep], tol[..., keep])
