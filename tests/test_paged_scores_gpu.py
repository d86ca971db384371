"""Paged attention of scores of any size.  Queries and keys are small integers
times powers of two, so that scores are exact in binary32 and a result can be
held to its definition in 64 bits however large they are: a bound that grows
with the score would let everything pass."""
import math

import pytest
import torch

from paged_ref import Batch, compare, half_step, smallest
from test_paged_gpu import BF16, F16, context

pytestmark = pytest.mark.gpu


def exact_batch(seqs, most=3, power=None, sign=None, **kw):
    """A Batch with q and k whole numbers of at most `most`, the key at position
    p of n times 2^power(p, n) and all of one sign against positive queries
    where sign(p, n) is not 0."""
    b = Batch(seqs, **kw)
    g = torch.Generator().manual_seed(kw.get("seed", 0) + 77)
    b.q = torch.randint(-most, most + 1, b.q.shape, generator=g).to(b.dtype)
    if sign:
        b.q = b.q.abs() + 1
    b.k = torch.where(torch.isnan(b.k), b.k, torch.randint(-most, most + 1, b.k.shape, generator=g).to(b.dtype))
    done = set()
    for s, n in enumerate(b.lens):
        for p in range(n if power or sign else 0):
            at = (int(b.table[s, p // b.page]), p % b.page)
            if at in done:
                continue  # a page that sequences share
            done.add(at)
            x = b.k[at].float()
            d = sign(p, n) if sign else 0
            x = d * (x.abs() + 1) if d else x
            b.k[at] = (x * 2.0 ** (power(p, n) if power else 0)).to(b.dtype)
    return b


def expected(b, scale):
    """(result, bound): as the definition has it, in 64 bits."""
    scale = 1 / math.sqrt(b.hd) if scale is None else float(torch.tensor(scale, dtype=torch.float32))
    u = half_step(b.dtype)
    want = torch.full((b.t, b.nh, b.hd), math.nan, dtype=torch.float64)
    tol = want.clone()
    for s, (n, r) in enumerate(zip(b.lens, b.rows)):
        k, v = b.positions(s, b.k), b.positions(s, b.v)
        hidden = torch.arange(n) > torch.arange(n - r, n)[:, None]
        at = slice(int(b.first[s]), int(b.first[s + 1]))
        for h in range(b.nh):
            x = (b.q[at, h].double() @ k[:, h * b.nkv // b.nh].T).masked_fill_(hidden, -math.inf)
            w = torch.softmax((x - x.amax(-1, keepdim=True)) * scale, -1)
            y, mean = w @ v[:, h * b.nkv // b.nh], w @ v[:, h * b.nkv // b.nh].abs()
            # Scores are exact, and so is what the largest is subtracted from
            # where the difference is small.  Weights: an exponent D down to
            # -160 (below that they vanish beside the largest) from a scale and
            # a multiply-add rounded to binary32, 2 * 160 * 2^-24 * ln 2 <
            # 2^-16, as much again for what sums are multiplied by when the
            # maximum moves; then rounded to the element type.  Sums of n
            # terms, joined pieces, the result rounded.
            rel = u + 2.0 ** -15 + (n + 64) * 2.0 ** -24
            few = n * 2.0 ** -33 * float(v.abs().max()) if b.dtype == F16 else 0.0
            want[at, h] = y
            tol[at, h] = mean * rel + few + (y.abs() + mean * rel) * u + smallest(b.dtype)
    return want, tol


def check(b, scale=None, shared=0, what=""):
    import ter_amd as T
    cache, batch = b.on_device(T)
    out = context(b).attend(b.q.cuda(), cache, batch, shared=shared, scale=scale)
    want, tol = expected(b, scale)
    compare(out, want, tol, what)


# one position, few, several tiles, rows enough for the 128-row kernel, cut sequences
SEQS = [(1, 1), (1, 40), (3, 700), (40, 90), (20, 1000), (1, 3000)]
SHAPES = [dict(nh=4, nkv=2, hd=64), dict(nh=3, nkv=1, hd=128)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["hd64", "hd128"])
@pytest.mark.parametrize("scale", [None, 1e3, 1e6, 1e12, 1e30, 1e38])
def test_any_scale(cuda, scale, shape, dtype):
    """Down to all weight on the largest scores, in equal parts where several
    are equal; products of a score and the scale beyond binary32 too."""
    check(exact_batch(SEQS, dtype=dtype, page=32, seed=1, **shape), scale)


@pytest.mark.parametrize("shape", SHAPES, ids=["hd64", "hd128"])
@pytest.mark.parametrize("power", [8, 10, 11, 12, 13])
def test_large_elements(cuda, power, shape):
    """fp16 queries and keys up to the type's largest: scores to 2^36."""
    b = exact_batch(SEQS, power=lambda p, n: power, dtype=F16, page=32, seed=2, **shape)
    b.q = b.q * 2.0 ** power
    assert torch.isfinite(b.q).all()
    check(b)


PATHS = {
    # powers of two of the keys along the sequence, sign of the scores
    "growing": (lambda p, n: 30 * p // n, None),
    "falling": (lambda p, n: 30 - 30 * p // n, None),
    "far below, then near zero": (lambda p, n: 28 if p < n // 2 else 0, lambda p, n: -1 if p < n // 2 else 1),
    "far below throughout": (lambda p, n: 28, lambda p, n: -1),
    "near zero, then far below": (lambda p, n: 0 if p < n // 2 else 28, lambda p, n: 1 if p < n // 2 else -1),
    "in turns": (lambda p, n: 6 * (p // 50 % 5), None),
}


@pytest.mark.parametrize("shared", [0, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=["hd64", "hd128"])
@pytest.mark.parametrize("path", PATHS)
def test_maximum_that_moves(cuda, path, shape, shared):
    """From ordinary scores to large ones and back, within a range of
    positions and between ranges that are joined."""
    power, sign = PATHS[path]
    seqs = [(1, 200), (2, 6000), (45, 700), (1, 129), (16, 2000)]
    check(exact_batch(seqs, power=power, sign=sign, dtype=BF16, page=64, common=128, seed=3, **shape), shared=shared)
