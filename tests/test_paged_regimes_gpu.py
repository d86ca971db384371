"""The paged attention where its work is cut as long calls are: more ranges than
workgroups, ranges of unequal length, ranges of more than 64 key tiles (whose
places in memory are found 64 at a time) and rows joined from hundreds of
ranges.  A sample of rows against the definition in 64 bits; that a case is in
the regime it is for comes from the constants of ter_amd/csrc/paged_plan.h and
paged_attend.hip, repeated here."""
import math

import pytest
import torch

from paged_ref import compare, half_step, smallest
from test_paged_gpu import BF16, F16

pytestmark = pytest.mark.gpu
TILE, LEAD, MIN_PER, TARGET = 64, 3, 2, 96


def plan(seqs, nh, nkv, hd, shared=0):
    """(units of the call, ranges, workgroups at once, tokens of a row tile)."""
    group, tokens = nh // nkv, 1
    while 2 * tokens * group <= 128:
        tokens *= 2
    units, rows = 0, sum(r for r, _ in seqs)
    for r, n in seqs:
        for i in range(0, r, tokens):
            see = n - r + min(r, i + tokens) - shared
            units += nkv * (LEAD + max(1, -(-see // TILE)))
    if shared:
        units += nkv * -(-rows // tokens) * (LEAD + -(-shared // TILE))
    resident = (2 if hd == 128 else 3) * torch.cuda.get_device_properties(0).multi_processor_count
    ranges = -(-units // MIN_PER)
    if ranges > resident:
        ranges = max(resident, min(4 * resident, units // TARGET))
    return units, ranges, resident, tokens


class Long:
    """seqs: (rows, kv_len).  The pages of all sequences are drawn from a small
    cache, so that a long context needs no memory of its own; the first
    `common` positions of all are the same."""

    def __init__(self, seqs, nh, nkv, hd, dtype, page=64, n_pages=700, common=0, seed=0):
        import ter_amd as T
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.seqs, self.nh, self.nkv, self.hd, self.page, self.dtype = seqs, nh, nkv, hd, page, dtype
        self.first = [0]
        for r, _ in seqs:
            self.first.append(self.first[-1] + r)
        width = max(-(-n // page) for _, n in seqs)
        self.table = torch.randint(0, n_pages, (len(seqs), width), generator=g, device="cuda", dtype=torch.int32)
        self.table[:, :common // page] = self.table[:1, :common // page]
        self.k, self.v = (torch.randn(n_pages, page, nkv, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
        self.q = torch.randn(self.first[-1], nh, hd, generator=g, device="cuda").to(dtype)
        self.cache = T.PagedCache(self.k, self.v)
        self.batch = T.PagedBatch(torch.tensor(self.first, dtype=torch.int32, device="cuda"),
                                  torch.tensor([n for _, n in seqs], dtype=torch.int32, device="cuda"), self.table)
        self.ctx = T.PagedAttention(nh, nkv, hd, 16, 1e4, dtype=dtype)

    def row(self, b, i):
        """(result, bound) of row i of sequence b, with the bound of paged_ref.Batch.attend."""
        r, n = self.seqs[b]
        m, u, f32 = n - r + i + 1, half_step(self.dtype), 2.0 ** -24
        p = torch.arange(m, device="cuda")
        page, slot = self.table[b].long()[p // self.page], p % self.page
        group, scale = self.nh // self.nkv, 1 / math.sqrt(self.hd)
        want, tol = [], []
        for h in range(self.nkv):
            k, v = self.k[page, slot, h].double(), self.v[page, slot, h].double()
            q = self.q[self.first[b] + i, h * group:(h + 1) * group].double()
            w = torch.softmax((q @ k.T.contiguous()) * scale, -1)
            mean = w @ v.abs()
            ds = ((q.abs() @ k.abs().T.contiguous()) * scale).amax(-1, keepdim=True) * (self.hd + 8) * f32 + 16 * f32
            rel = 2 * ds + u + (m + 64) * f32
            few = m * 2.0 ** -33 * float(v.abs().max()) if self.dtype == F16 else 0.0
            y = w @ v
            want.append(y)
            tol.append(mean * rel + few + (y.abs() + mean * rel) * u + smallest(self.dtype))
        return torch.cat(want).cpu(), torch.cat(tol).cpu()

    def check(self, rows, shared=0):
        out = self.ctx.attend(self.q, self.cache, self.batch, shared=shared)
        again = self.ctx.attend(self.q, self.cache, self.batch, shared=shared)
        assert torch.equal(out, again), "the same call, the same bits"
        for b, i in rows:
            want, tol = self.row(b, i)
            compare(out[self.first[b] + i], want, tol, f"row {i} of sequence {b}")


def sample(r, n=24):
    """Rows of a sequence: the ends, and others that no step of a power of two finds."""
    return sorted({0, 1, r // 2, r - 2, r - 1} & set(range(r)) | {i * (r - 1) // n for i in range(n)})


HEADS = {64: dict(nh=16, nkv=4, hd=64), 128: dict(nh=12, nkv=3, hd=128)}


@pytest.mark.parametrize("hd,dtype,rows", [(128, BF16, 16001), (64, F16, 12345)])
def test_more_ranges_than_workgroups(cuda, hd, dtype, rows):
    """One long prompt: ranges begin as others end, of more than 64 key tiles
    each, in segments of up to 250."""
    seqs = [(rows, rows)]
    units, ranges, resident, _ = plan(seqs, **HEADS[hd])
    assert ranges > resident and units // ranges > 64 + LEAD and rows // TILE > 2 * 64
    Long(seqs, dtype=dtype, **HEADS[hd]).check([(0, i) for i in sample(rows)])


@pytest.mark.parametrize("hd,dtype,seqs", [
    (128, F16, [(2501, 2501), (900, 1300), (1, 700), (333, 333), (77, 3000)]),
    (64, BF16, [(1, 4000), (2047, 2100), (1500, 1500), (300, 5000), (64, 64)]),
])
def test_ranges_of_unequal_length(cuda, hd, dtype, seqs):
    """Rows that keep the matrix cores busy: longer ranges for the older
    workgroups of a CU."""
    units, ranges, resident, _ = plan(seqs, **HEADS[hd])
    group = HEADS[hd]["nh"] // HEADS[hd]["nkv"]
    assert ranges == resident and units // ranges >= 4 and sum(r for r, _ in seqs) * group > 16 * len(seqs)
    Long(seqs, dtype=dtype, seed=1, **HEADS[hd]).check([(b, i) for b, (r, _) in enumerate(seqs) for i in sample(r, 9)])


@pytest.mark.parametrize("hd,dtype,seqs", [
    (128, F16, [(1, 750001)]),
    (128, BF16, [(1, 450000), (2, 300000), (1, 77)]),
    (64, F16, [(1, 900017)]),
    (64, BF16, [(1, 300001), (1, 250000), (3, 350007), (1, 5)]),
])
def test_ranges_of_many_tiles_of_few_rows(cuda, hd, dtype, seqs):
    """Single tokens over very long contexts: ranges of more than 64 key tiles
    by the kernel for few rows, hundreds of them to a row."""
    units, ranges, resident, _ = plan(seqs, **HEADS[hd])
    assert ranges >= resident and units // ranges > 64 + LEAD
    assert all(r * HEADS[hd]["nh"] // HEADS[hd]["nkv"] <= 16 for r, _ in seqs)
    Long(seqs, dtype=dtype, seed=2, **HEADS[hd]).check([(b, i) for b, (r, _) in enumerate(seqs) for i in range(r)])


@pytest.mark.parametrize("hd,dtype,n,rows,prefix", [(64, F16, 8, 130, 65536), (128, BF16, 40, 20, 65536)])
def test_prefix_of_many_tiles(cuda, hd, dtype, n, rows, prefix):
    """Ranges of more than 64 key tiles on a shared prefix."""
    seqs = [(rows - b % 3, prefix + rows + 17 * b) for b in range(n)]
    units, ranges, resident, _ = plan(seqs, shared=prefix, **HEADS[hd])
    assert ranges >= resident and units // ranges > 64 + LEAD
    x = Long(seqs, dtype=dtype, seed=3, common=prefix, n_pages=1500, **HEADS[hd])
    x.check([(b, i) for b in (0, 1, n // 2, n - 1) for i in (0, rows // 2, rows - 3)], shared=prefix)
