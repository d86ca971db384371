"""What the paged attention rounds: of few rows (at most 16 of a KV head and
sequence, as single tokens are) nothing between the inputs and the result but in
binary32 and to twice the element type's bits."""
import math

import pytest
import torch

from paged_ref import Batch, compare, half_step, smallest
from test_paged_gpu import BF16, F16, context

pytestmark = pytest.mark.gpu


def expected(b):
    """(result, bound) of the rows: paged_ref.Batch.attend's, but weights are
    held in two elements (half a step of half a step)."""
    u, f32, scale = half_step(b.dtype), 2.0 ** -24, 1 / math.sqrt(b.hd)
    want = torch.full((b.t, b.nh, b.hd), math.nan, dtype=torch.float64)
    tol = want.clone()
    for s, (n, r) in enumerate(zip(b.lens, b.rows)):
        k, v = b.positions(s, b.k), b.positions(s, b.v)
        hidden = torch.arange(n) > torch.arange(n - r, n)[:, None]
        at = slice(int(b.first[s]), int(b.first[s + 1]))
        for h in range(b.nh):
            g, q = h * b.nkv // b.nh, b.q[at, h].double()
            w = torch.softmax((q @ k[:, g].T * scale).masked_fill_(hidden, -math.inf), -1)
            y, mean = w @ v[:, g], w @ v[:, g].abs()
            ds = (q.abs() @ k[:, g].abs().T * scale).amax(-1, keepdim=True) * (b.hd + 8) * f32 + 16 * f32
            rel = 2 * ds + u * u + (n + 64) * f32
            few = n * 2.0 ** -33 * float(v.abs().max()) if b.dtype == F16 else 0.0
            want[at, h] = y
            tol[at, h] = mean * rel + few + (y.abs() + mean * rel) * u + smallest(b.dtype)
    return want, tol


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", [dict(nh=4, nkv=2, hd=64), dict(nh=5, nkv=1, hd=128)], ids=["hd64", "hd128"])
@pytest.mark.parametrize("seqs", [
    [(1, n) for n in (1, 2, 3, 5, 17, 40, 130)], [(3, 3), (2, 20), (3, 300), (1, 700)], [(1, 6000), (3, 2500), (2, 9)],
], ids=["single", "few", "cut"])
def test_few_rows_keep_their_weights(cuda, seqs, shape, dtype):
    import ter_amd as T
    b = Batch(seqs, dtype=dtype, seed=8, page=32, **shape)
    cache, batch = b.on_device(T)
    want, tol = expected(b)
    compare(context(b).attend(b.q.cuda(), cache, batch), want, tol)


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


@pytest.mark.parametrize("shape", [dict(nh=4, nkv=2, hd=64), dict(nh=4, nkv=1, hd=128)], ids=["hd64", "hd128"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 64])
@pytest.mark.parametrize("value", ["1.5", "max", "-max"])
def test_equal_values(cuda, value, shared, shape, dtype):
    """Where all values are one number so is every result, up to the type's
    largest: sums of n terms in binary32 are off by less than half a step."""
    import ter_amd as T
    seqs = [(60, 160), (1, 70), (3, 2500), (100, 900), (1, 3900), (70, 70)]
    b = Batch(seqs, dtype=dtype, seed=11, page=16, common=shared, spread=1.5, **shape)
    x = 1.5 if value == "1.5" else torch.finfo(dtype).max * (-1 if value[0] == "-" else 1)
    b.v = torch.where(torch.isnan(b.v), b.v, torch.full_like(b.v, x))
    assert max(b.lens) * 2.0 ** -23 < half_step(dtype)
    cache, batch = b.on_device(T)
    out = context(b).attend(b.q.cuda(), cache, batch, shared=shared)
    assert (out == x).all(), out[out != x][:4]


@pytest.mark.parametrize("shape", [dict(nh=4, nkv=2, hd=64), dict(nh=4, nkv=1, hd=128)], ids=["hd64", "hd128"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shared", [0, 64])
def test_values_near_the_largest(cuda, shared, shape, dtype):
    """No sum on the way leaves binary32."""
    import ter_amd as T
    seqs = [(60, 160), (1, 70), (3, 2500), (100, 900), (1, 6000)]
    b = Batch(seqs, dtype=dtype, seed=12, page=16, common=shared, **shape)
    top = torch.finfo(dtype).max
    b.v = torch.where(torch.isnan(b.v), b.v, (b.v.float().clamp(-1, 1) * top).to(dtype))
    cache, batch = b.on_device(T)
    out = context(b).attend(b.q.cuda(), cache, batch, shared=shared)
    assert torch.isfinite(out).all()
    want, tol = b.attend()
    compare(out, want, tol)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
def test_many_small_weights(cuda, dtype, hd, rows):
    """2^17 weights of 2^-23 of the largest, subnormal in fp16, are a 64th of
    the sum: in it and in the product with the values alike."""
    import ter_amd as T
    n, page = 1 << 17, 64
    k = torch.zeros(2, page, 1, hd, dtype=dtype, device="cuda")
    k[0, 0] = 1.0  # page 0 is the first one only: one score of hd, zeros behind it
    v = torch.ones_like(k)
    q = torch.ones(rows, 4, hd, dtype=dtype, device="cuda")
    table = torch.ones(1, n // page, dtype=torch.int32, device="cuda")
    table[0, 0] = 0
    cache = T.PagedCache(k, v)
    batch = T.PagedBatch(torch.tensor([0, rows], dtype=torch.int32, device="cuda"),
                         torch.tensor([n], dtype=torch.int32, device="cuda"), table)
    ctx = T.PagedAttention(4, 1, hd, 16, 1e4, dtype=dtype)
    scale = 23 * math.log(2) / hd
    # (sums of equal numbers in binary32, pieces of at most 2^12 of a lane, joined: 2^-11 would be seen)
    assert (ctx.attend(q, cache, batch, scale=scale) == 1.0).all()
    v[0, 0] = 0.0
    m = torch.arange(n - rows, n, dtype=torch.float64) + 1
    small = (m - 1) * 2.0 ** -23
    want = (small / (1 + small))[:, None, None].expand(rows, 4, hd)
    # an exponent of 23 from a rounded scale (2^-24 of it) and exp2, half a
    # step of 2^-15 in subnormals of 2^-24, or of the element type, and of the
    # result; sums of 2^17 terms in lanes and pieces of at most 2^12
    u = half_step(dtype)
    rel = 23 * 2.0 ** -23 + max(2.0 ** -10, u) + 2.0 ** -11 + u
    compare(ctx.attend(q, cache, batch, scale=scale), want, want * rel)
