"""The paged-cache operators (PagedAttention.append, .attend, attend(shared=))
against their definitions in 64 bits, on the device.  The cache's unowned
slots hold NaN in every test (paged_ref.Batch)."""
import math

import numpy as np
import pytest
import torch

from paged_ref import Batch, compare, rotated

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16
THETA = 10000.0


def context(b, max_pos=None, neox=True, theta=THETA):
    import ter_amd as T
    return T.PagedAttention(b.nh, b.nkv, b.hd, max_pos or max(b.lens + [1]) + 8, theta, neox=neox, dtype=b.dtype)


def check_attend(b, scale=None, shared=0, what=""):
    import ter_amd as T
    cache, batch = b.on_device(T)
    q = b.q.cuda()
    out = torch.full_like(q, 7.0)
    ctx = context(b)
    got = ctx.attend(q, cache, batch, shared=shared, scale=scale, out=out)
    assert got is out
    want, tol = b.attend(scale)
    n = int(b.first[-1])
    compare(out[:n], want[:n], tol[:n], what)
    assert (out[n:] == 7.0).all(), "rows behind the last sequence"
    return out


SHAPES = [dict(nh=4, nkv=2, hd=64), dict(nh=4, nkv=1, hd=128)]


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["hd64", "hd128"])
@pytest.mark.parametrize("lens", [[1], [15], [16, 17], [63, 64, 65], [127, 128, 129, 1], [1000, 3, 511, 512, 513]],
                         ids=str)
def test_single_tokens(cuda, lens, shape, dtype):
    check_attend(Batch([(1, n) for n in lens], dtype=dtype, seed=len(lens), **shape))


@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=["hd64", "hd128"])
@pytest.mark.parametrize("seqs", [
    [(2, 2)], [(31, 31), (32, 32), (33, 33)], [(64, 64), (65, 65), (1, 1), (127, 127)], [(300, 300)],
    [(1, 700), (40, 900), (5, 5), (129, 200), (64, 128)], [(200, 1200)],
], ids=str)
def test_prompts_and_chunks(cuda, seqs, shape, dtype):
    check_attend(Batch(seqs, dtype=dtype, page=32, seed=len(seqs), **shape))


@pytest.mark.parametrize("nh,nkv", [(3, 3), (3, 1), (10, 2), (12, 1), (16, 1), (17, 1), (32, 1), (128, 1), (66, 2)])
def test_head_groups(cuda, nh, nkv):
    """Groups of 1 to 128 query heads, powers of two and others, single tokens
    and rows together."""
    check_attend(Batch([(1, 130), (7, 90), (20, 20)], nh=nh, nkv=nkv, hd=64, seed=nh))


@pytest.mark.parametrize("page", [16, 48, 64, 112, 256, 4096])
def test_page_sizes(cuda, page):
    check_attend(Batch([(1, 500), (70, 333), (1, page), (3, page + 1)], page=page, seed=page))


@pytest.mark.parametrize("layout", ["hpd", "kv"])
def test_cache_layouts(cuda, layout):
    check_attend(Batch([(1, 333), (40, 100)], page=32, nh=8, nkv=4, layout=layout))


def test_many_sequences(cuda):
    """The most sequences a call takes, lengths of every kind, some empty."""
    rng = np.random.default_rng(5)
    seqs = [(int(rng.choice([0, 1, 1, 1, 2, 9])), int(rng.integers(9, 150))) for _ in range(1024)]
    check_attend(Batch(seqs, nh=2, nkv=1, hd=64))


def test_empty_rows_and_sequences(cuda):
    """Sequences without rows, without positions, rows at positions below zero
    (zeros), rows behind the last sequence (left alone), a call without rows."""
    import ter_amd as T
    b = Batch([(0, 0), (3, 0), (0, 50), (5, 2), (1, 70), (0, 9)], spare_rows=5, dtype=BF16)
    out = check_attend(b)
    assert (out[:3] == 0).all() and (out[3:6] == 0).all()
    cache, batch = b.on_device(T)
    assert context(b).attend(b.q.cuda()[:0], cache, batch).shape == (0, b.nh, b.hd)
    # every sequence empty: nothing is written
    e = Batch([(0, 40), (0, 0)], spare_rows=3)
    check_attend(e)


def test_masked_infinities_and_nan(cuda):
    """Infinities and NaN at positions that a row does not see change nothing;
    at one that it sees they are its result's, as in the formula."""
    import ter_amd as T
    for hd in (64, 128):
        b = Batch([(100, 100), (1, 90), (40, 200)], hd=hd, page=32, seed=3)
        bad = {0: 57, 2: 180}  # sequence: position
        for (s, p), val in zip(bad.items(), (math.nan, math.inf)):
            page = b.table[s, p // 32]
            b.v[page, p % 32, :, 5] = val
            b.v[page, p % 32, 0, hd - 1] = -math.inf
        b.k[b.table[0, 99 // 32], 99 % 32] = math.nan  # the last position of the first sequence
        cache, batch = b.on_device(T)
        out = context(b).attend(b.q.cuda(), cache, batch).cpu()
        clean = Batch([(100, 100), (1, 90), (40, 200)], hd=hd, page=32, seed=3)
        want, tol = clean.attend()
        compare(out[:57], want[:57], tol[:57], "rows before the NaN")
        compare(out[100:101], want[100:101], tol[100:101], "another sequence")
        seen = 101 + 20  # row at position 180
        compare(out[101:seen], want[101:seen], tol[101:seen], "rows before the infinity")
        assert torch.isnan(out[57:99, :, 5]).all() and torch.isinf(out[seen:, :, 5]).all()
        assert (out[57:99, :2, hd - 1] == -math.inf).all() and (out[seen:, :2, hd - 1] == -math.inf).all()
        assert torch.isnan(out[99]).all()
        keep = [d for d in range(hd) if d not in (5, hd - 1)]
        compare(out[57:99][:, :, keep], want[57:99][:, :, keep], tol[57:99][:, :, keep], "other elements")


@pytest.mark.parametrize("shared", [0, 16])
@pytest.mark.parametrize("hd", [64, 128])
def test_masked_nan_of_few_rows(cuda, hd, shared):
    """The same where a sequence has few rows, short ones among long: keys and
    values of every sequence's last position are NaN, which its last row only
    sees."""
    import ter_amd as T
    seqs = [(3, 20), (2, 33), (4, 700), (5, 290), (2, 18), (1, 40), (16, 64)]
    b = Batch(seqs, hd=hd, nh=2, nkv=2, common=16, seed=4)
    want, tol = b.attend()
    for s, n in enumerate(b.lens):
        b.k[b.table[s, (n - 1) // 16], (n - 1) % 16] = math.nan
        b.v[b.table[s, (n - 1) // 16], (n - 1) % 16] = math.nan
    cache, batch = b.on_device(T)
    out = context(b).attend(b.q.cuda(), cache, batch, shared=shared).cpu()
    for s in range(len(seqs)):
        at, end = int(b.first[s]), int(b.first[s + 1]) - 1
        compare(out[at:end], want[at:end], tol[at:end], f"sequence {s}")
        assert torch.isnan(out[end]).all()


@pytest.mark.parametrize("nh,nkv,seqs", [(128, 1, [(1, 5000), (3, 900)]), (17, 1, [(1, 6000), (9, 1500)]),
                                         (6, 2, [(2, 9000), (1, 10), (1, 30)])])
def test_long_sequences_of_few_rows(cuda, nh, nkv, seqs):
    """Cut among many workgroups, groups of every size."""
    check_attend(Batch(seqs, nh=nh, nkv=nkv, page=64, dtype=BF16, seed=nh))


@pytest.mark.parametrize("shared", [0, 32])
def test_row0_that_decreases(cuda, shared):
    """Not allowed, and without a meaning for the rows it confuses; the others
    are right and nothing else is written."""
    import ter_amd as T
    b = Batch([(4, 40), (4, 50), (4, 60), (4, 70)], common=32, spare_rows=6)
    cache, batch = b.on_device(T)
    wild = T.PagedBatch(torch.tensor([0, 4, 12, 7, 16], dtype=torch.int32, device="cuda"), batch.kv_len, batch.pages)
    out = torch.full((b.t, b.nh, b.hd), 7.0, dtype=b.dtype, device="cuda")
    ctx = context(b)
    ctx.attend(b.q.cuda(), cache, wild, shared=shared, out=out)
    want, tol = b.attend()
    compare(out[:4], want[:4], tol[:4])
    assert (out[16:] == 7.0).all()
    k = torch.zeros(b.t, b.nkv, b.hd, dtype=b.dtype, device="cuda")
    ctx.append(None, k, k, cache, wild)
    torch.cuda.synchronize()


@pytest.mark.parametrize("shared", [0, 16])
def test_overlapping_sequences_keep_to_the_workspace(cuda, shared):
    """More row tiles than rows could have: no more ranges than the workspace
    has places for."""
    import ter_amd as T
    from ter_amd import _lib as L
    n = 20
    kd = torch.zeros(4, 16, 1, 64, dtype=F16, device="cuda")
    batch = T.PagedBatch(torch.tensor([0, n] * 10 + [0], dtype=torch.int32, device="cuda"),
                         torch.full((n,), 60, dtype=torch.int32, device="cuda"),
                         torch.arange(4, dtype=torch.int32, device="cuda").repeat(n, 1))
    ctx = T.PagedAttention(128, 1, 64, 64, THETA)
    cache = T.PagedCache(kd, kd)
    q = torch.zeros(n, 128, 64, dtype=F16, device="cuda")
    out = torch.empty_like(q)
    need = L.lib().ter_hip_paged_attend_ws(ctx._h, batch._ref, cache._ref, n, shared)
    ws = torch.full((need + (1 << 24),), 165, dtype=torch.uint8, device="cuda")
    rc = L.lib().ter_hip_paged_attend(ctx._h, batch._ref, cache._ref, n, q.data_ptr(), 128 * 64, out.data_ptr(), 128 * 64,
                                      shared, 0.0, ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert (ws[need:] == 165).all()


def test_overlapping_sequences_beyond_counting(cuda):
    """The same with more work than a call can have: none is done."""
    import ter_amd as T
    n = 1024
    kd = torch.zeros(1, 4096, 1, 64, dtype=F16, device="cuda")
    row0 = torch.tensor([0, n] * 512 + [0], dtype=torch.int32, device="cuda")
    batch = T.PagedBatch(row0, torch.full((1024,), 1 << 20, dtype=torch.int32, device="cuda"),
                         torch.zeros(1024, 256, dtype=torch.int32, device="cuda"))
    out = torch.full((n, 128, 64), 7.0, dtype=F16, device="cuda")
    for shared in (0, 4096):
        T.PagedAttention(128, 1, 64, 16, THETA).attend(torch.zeros_like(out), T.PagedCache(kd, kd), batch, shared=shared,
                                                       out=out)
        assert (out == 7.0).all()


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("hd", [64, 128])
def test_scores_of_minus_infinity(cuda, hd, rows):
    """Keys that no weight can fall on, whole tiles and ranges of them, beside
    scores far below zero: the others' softmax, NaN where there are no others."""
    import ter_amd as T
    n = 3000
    b = Batch([(rows, n), (rows, 130)], hd=hd, nh=4, nkv=1, page=64, dtype=BF16, seed=6)
    b.q = b.q.abs() + 0.5
    b.k = torch.where(torch.isnan(b.k), b.k, -(b.k.abs() * 8 + 4))  # scores: about -10 sqrt(hd)
    # 2,000 positions of the first sequence, all of the second
    for s, (lo, hi) in enumerate(((0, 2000), (0, 130))):
        for p in range(lo, hi):
            b.k[b.table[s, p // 64], p % 64, :, 0] = -math.inf
    cache, batch = b.on_device(T)
    out = context(b).attend(b.q.cuda(), cache, batch).double().cpu()
    assert torch.isnan(out[rows:]).all()
    k, v = b.positions(0, b.k)[2000:, 0], b.positions(0, b.v)[2000:, 0]
    for i in range(rows):
        m = n - rows + i + 1 - 2000
        for h in range(4):
            q = b.q[i, h].double()
            w = torch.softmax((k[:m] @ q) / math.sqrt(hd), 0)
            mean = w @ v[:m].abs()
            ds = float((k[:m].abs() @ q.abs()).max()) / math.sqrt(hd) * (hd + 8) * 2.0 ** -24 + 16 * 2.0 ** -24
            rel = 2 * ds + 2.0 ** -8 + (n + 64) * 2.0 ** -24
            assert ((out[i, h] - w @ v[:m]).abs() <= mean * rel + ((w @ v[:m]).abs() + mean * rel) * 2.0 ** -8).all(), (i, h)


def test_peaked_and_flat_scores(cuda):
    """Scores so far apart that all but one weight vanishes, growing along the
    sequence (the running maximum moves at every step), and all equal."""
    b = Batch([(90, 600), (1, 600)], spread=4.0, page=64)
    check_attend(b)
    for s in (0, 1):
        for p in range(600):
            b.k[b.table[s, p // 64], p % 64] *= p / 300
    check_attend(b)
    b = Batch([(90, 600), (1, 600)], page=64)
    b.k = torch.where(torch.isnan(b.k), b.k, torch.ones_like(b.k))
    check_attend(b)


@pytest.mark.parametrize("scale", [1.0, 0.01, 1e-30])
def test_scale(cuda, scale):
    check_attend(Batch([(40, 100), (1, 300)], seed=2), scale=scale)


def test_large_values(cuda):
    """fp16 products near the type's largest values: scores of 10^6 and more."""
    b = Batch([(20, 50), (1, 130)], spread=100.0)
    check_attend(b)


@pytest.mark.parametrize("common,shared", [(64, 64), (320, 320), (320, 300), (320, 17), (320, 15), (96, 96)])
@pytest.mark.parametrize("rows", ["ones", "some"])
def test_shared_prefix(cuda, common, shared, rows):
    """shared=n: results as without it.  Prefixes that end inside a tile or a
    page, and too short to count (15)."""
    rng = np.random.default_rng(common + shared)
    seqs = [(1 if rows == "ones" else int(rng.integers(1, 30)), common + int(rng.integers(30, 200))) for _ in range(9)]
    for dtype, hd in ((F16, 128), (BF16, 64)):
        check_attend(Batch(seqs, common=common, page=32, dtype=dtype, hd=hd, nh=8, nkv=2, seed=1), shared=shared)


def test_shared_prefix_of_everything(cuda):
    """Rows inside the prefix (they see a part of it), sequences that end with
    it or before it, empty ones, one alone."""
    check_attend(Batch([(40, 128), (128, 128), (1, 100), (0, 64), (2, 0), (1, 128), (3, 140)], common=128, page=64),
                 shared=128)
    check_attend(Batch([(1, 500)], common=496, nh=32, nkv=8), shared=496)
    check_attend(Batch([(150, 300), (140, 290)], common=256, page=64, nh=8, nkv=1), shared=256)


@pytest.mark.parametrize("hd,n,prefix", [(64, 130, 1024), (128, 40, 4096)])
def test_shared_prefix_of_many(cuda, hd, n, prefix):
    """Enough rows for several row tiles on the prefix, which itself is split."""
    rng = np.random.default_rng(n)
    check_attend(Batch([(1, prefix + int(rng.integers(1, 70))) for _ in range(n)], common=prefix, page=64, hd=hd, nh=4,
                       nkv=1, spare_rows=2), shared=prefix)


def test_bad_pages_read_as_zeros(cuda):
    """Ids outside the cache: attend takes zeros there, append writes nothing."""
    import ter_amd as T
    b = Batch([(1, 300), (50, 120)], page=16)
    b.table[0, 3], b.table[0, 7], b.table[1, 2] = -1, b.k.shape[0], 1 << 30
    b.table[1, 5] = -(1 << 31)
    check_attend(b)
    cache, batch = b.on_device(T)
    k = torch.randn(51, b.nkv, b.hd).to(b.dtype)
    before = cache.k.clone()
    context(b).append(None, k.cuda(), k.cuda(), cache, batch)
    changed = (cache.k.view(torch.int16) != before.view(torch.int16)).any(-1).any(-1).cpu()
    want = torch.zeros_like(changed)
    for s, r in ((0, 1), (1, 50)):
        for p in range(b.lens[s] - r, b.lens[s]):
            if 0 <= b.table[s, p // 16] < b.k.shape[0]:
                want[b.table[s, p // 16], p % 16] = True
    assert (changed == want).all()


def test_lengths_past_the_table(cuda):
    """kv_len beyond the table: attend sees what the table holds, append drops
    what has no place; row0 out of range is clamped."""
    import ter_amd as T
    b = Batch([(1, 64), (4, 30)], page=16)
    cache, batch = b.on_device(T)
    ctx = context(b, max_pos=200)
    short = T.PagedBatch(batch.row0, torch.tensor([100, 30], dtype=torch.int32, device="cuda"),
                         batch.pages[:, :4].contiguous())
    out = ctx.attend(b.q.cuda(), cache, short)
    want, tol = b.attend()
    compare(out, want, tol)
    k = torch.ones(5, b.nkv, b.hd, dtype=b.dtype, device="cuda")
    before = cache.k.clone()
    ctx.append(None, k, k, cache, short)
    assert torch.equal(cache.k[b.table[0, :4].tolist()], before[b.table[0, :4].tolist()])
    wild = T.PagedBatch(torch.tensor([-3, 1, 99], dtype=torch.int32, device="cuda"), batch.kv_len, batch.pages)
    out = ctx.attend(b.q.cuda(), cache, wild)
    compare(out[:1], want[:1], tol[:1])
    torch.cuda.synchronize()


def test_offsets_past_32_bits(cuda):
    """Pages more than 4 GiB into the cache, and strides of pages that far."""
    import ter_amd as T
    b = Batch([(1, 200), (33, 100)], page=64, nh=8, nkv=8, hd=128)
    n = (1 << 32) // (64 * 8 * 128 * 2) + 64  # pages in a little over 4 GiB
    kd = torch.empty(n, 64, 8, 128, dtype=b.dtype, device="cuda")
    vd = torch.empty_like(kd)
    move = {i: n - 1 - 3 * i for i in range(b.k.shape[0])}
    for i, j in move.items():
        kd[j], vd[j] = b.k[i].cuda(), b.v[i].cuda()
    assert kd[-1].data_ptr() - kd.data_ptr() > 1 << 32
    table = torch.tensor([[move.get(int(i), -1) for i in row] for row in b.table], dtype=torch.int32, device="cuda")
    _, batch = b.on_device(T)
    far = T.PagedBatch(batch.row0, batch.kv_len, table)
    cache = T.PagedCache(kd, vd)
    out = context(b).attend(b.q.cuda(), cache, far)
    want, tol = b.attend()
    compare(out, want, tol)
    k = torch.randn(34, 8, 128).to(b.dtype).cuda()
    context(b).append(None, k, k, cache, far)
    assert torch.equal(vd[move[int(b.table[0, 199 // 64])], 199 % 64], k[0])
    assert torch.equal(vd[move[int(b.table[1, 1])], 99 % 64], k[33])


@pytest.mark.parametrize("neox", [True, False], ids=["neox", "norm"])
@pytest.mark.parametrize("dtype", [F16, BF16], ids=["f16", "bf16"])
@pytest.mark.parametrize("shape", [dict(nh=4, nkv=2, hd=64), dict(nh=20, nkv=5, hd=128), dict(nh=1, nkv=1, hd=64),
                                   dict(nh=40, nkv=10, hd=128)], ids=str)
def test_append(cuda, shape, dtype, neox):
    """Rotated queries and keys, copied values, everything else untouched."""
    import ter_amd as T
    b = Batch([(1, 1), (3, 40), (0, 20), (70, 70), (2, 1), (1, 700), (0, 0)], dtype=dtype, page=32, spare_rows=2, **shape)
    cache, batch = b.on_device(T)
    g = torch.Generator().manual_seed(9)
    k = torch.randn(b.t, b.nkv, b.hd, generator=g).to(dtype)
    v = torch.randn(b.t, b.nkv, b.hd, generator=g).to(dtype)
    ctx = context(b, neox=neox, theta=500000.0)
    q_out = torch.full_like(b.q, 5.0).cuda()
    assert ctx.append(b.q.cuda(), k.cuda(), v.cuda(), cache, batch, q_out=q_out) is q_out
    pos, seq = [], []
    for s, (r, n) in enumerate(zip(b.rows, b.lens)):
        pos += list(range(n - r, n))
        seq += [s] * r
    keep = [i for i, p in enumerate(pos) if p >= 0]
    at = [pos[i] for i in keep]
    want, tol = rotated(b.q[keep], at, 500000.0, neox, dtype)
    compare(q_out[keep], want, tol, "q")
    kw, kt = rotated(k[keep], at, 500000.0, neox, dtype)
    page = [int(b.table[seq[i], pos[i] // 32]) for i in keep]
    slot = [p % 32 for p in at]
    compare(cache.k[page, slot], kw, kt, "k")
    assert torch.equal(cache.v[page, slot].cpu(), v[keep])
    left = [i for i in range(b.t) if i not in keep]
    assert (q_out[left] == 5.0).all()
    for now, was in ((cache.k.cpu(), b.k.clone()), (cache.v.cpu(), b.v.clone())):
        was[page, slot] = now[page, slot]
        assert torch.equal(now.view(torch.int16), was.view(torch.int16)), "untouched places"


def test_append_far_positions(cuda):
    """Positions up to the largest a context takes: angles beyond binary32."""
    import ter_amd as T
    at = [(1 << 20) - 1, 777_777, 99_999]
    n = (1 << 20) // 65536
    table = torch.full((3, n), -1, dtype=torch.int32)
    for s, p in enumerate(at):
        table[s, p // 65536] = s
    kd = torch.zeros(3, 65536, 1, 64, dtype=BF16, device="cuda")
    cache = T.PagedCache(kd, torch.zeros_like(kd))
    batch = T.PagedBatch(torch.arange(4, dtype=torch.int32, device="cuda"),
                         torch.tensor(at, dtype=torch.int32, device="cuda") + 1, table.cuda())
    ctx = T.PagedAttention(1, 1, 64, 1 << 20, THETA, dtype=BF16)
    x = torch.randn(3, 1, 64).to(BF16)
    out = ctx.append(x.cuda(), x.cuda(), x.cuda(), cache, batch)
    want, tol = rotated(x, at, THETA, True, BF16)
    compare(out, want, tol)
    for s, p in enumerate(at):
        assert torch.equal(kd[s, p % 65536, 0], out[s, 0])
    # a context that ends before them leaves them alone
    near = T.PagedAttention(1, 1, 64, 99_999, THETA, dtype=BF16)
    kd.zero_()
    out = near.append(x.cuda(), x.cuda(), x.cuda(), cache, batch, q_out=torch.full_like(x, 3.0).cuda())
    assert (out == 3.0).all() and not kd.any()


def test_append_in_place_and_from_fused_rows(cuda):
    """q, k and v as parts of one projection's rows, q rotated in place; 2-D rows."""
    import ter_amd as T
    b = Batch([(5, 5), (1, 20)], nh=8, nkv=2, hd=64)
    cache, batch = b.on_device(T)
    rows = torch.randn(6, 12 * 64).to(b.dtype).cuda()
    was = rows.clone()
    q, k, v = rows[:, :512], rows[:, 512:640], rows[:, 640:]
    ctx = context(b)
    ref = ctx.append(was[:, :512].reshape(6, 8, 64), was[:, 512:640].reshape(6, 2, 64), was[:, 640:].reshape(6, 2, 64),
                     *b.on_device(T))
    got = ctx.append(q, k, v, cache, batch, q_out=q)
    assert got is q and torch.equal(q, ref.reshape(6, 512)) and torch.equal(rows[:, 512:], was[:, 512:])
    # attention from and into parts of rows
    full = torch.zeros(6, 3, 8, 64, dtype=b.dtype, device="cuda")
    out = ctx.attend(q, cache, batch, out=full[:, 1])
    assert torch.equal(out, ctx.attend(ref, cache, batch)) and not full[:, 0].any() and not full[:, 2].any()


def test_agrees_with_the_decode_attention(cuda):
    """One sequence, prompt by append + attend, then token by token: the keys
    and outputs of Attention.decode, whose angles are rounded to binary32."""
    import ter_amd as T
    nh, nkv, hd, smax = 20, 5, 128, 128
    g = torch.Generator().manual_seed(4)
    n = 90
    q, k, v = (torch.randn(n, h, hd, generator=g).half().cuda() for h in (nh, nkv, nkv))
    A = T.Attention(nh, nkv, hd, smax, 500000.0, neox=True)
    kc, vc = (torch.zeros(smax, nkv, hd, dtype=F16, device="cuda") for _ in range(2))
    ref = [A.decode(q[i], k[i], v[i], kc, vc, torch.tensor([i], dtype=torch.int32, device="cuda")) for i in range(n)]
    # the decode attention's cache is a paged one whose pages lie in order
    kp, vp = (torch.zeros(smax // 16, 16, nkv, hd, dtype=F16, device="cuda") for _ in range(2))
    cache = T.PagedCache(kp, vp)
    table = torch.arange(smax // 16, dtype=torch.int32, device="cuda")[None]
    ctx = T.PagedAttention(nh, nkv, hd, smax, 500000.0)
    row0, lens = torch.tensor([0, 83], dtype=torch.int32, device="cuda"), torch.tensor([83], dtype=torch.int32, device="cuda")
    batch = T.PagedBatch(row0, lens, table)
    got = list(ctx.attend(ctx.append(q[:83], k[:83], v[:83], cache, batch), cache, batch))
    row0.copy_(torch.tensor([0, 1]))
    for i in range(83, n):
        lens.fill_(i + 1)
        got.append(ctx.attend(ctx.append(q[i:i + 1], k[i:i + 1], v[i:i + 1], cache, batch), cache, batch)[0])
    assert torch.equal(vp.view(smax, nkv, hd), vc)
    # keys: angles off by position * 2^-23, then both rounded
    size = k.float().abs().amax() * 2 * (n * 2.0 ** -23)
    d = (kp.view(smax, nkv, hd).float() - kc.float()).abs()
    assert (d <= kc.float().abs() * 2.0 ** -10 + size + 2.0 ** -24).all()
    # outputs: each weight changes by that times |q||k|; rounded twice
    for i in range(n):
        e = (got[i].float() - ref[i].float()).abs()
        size = q[i].float().norm(dim=-1).max() * k[:i + 1].float().norm(dim=-1).max()
        ds = 2 * (2.0 ** -10 + n * 2.0 ** -22) * float(size) / hd ** 0.5
        assert (e <= (2 * ds + 2.0 ** -9) * v[:i + 1].float().abs().amax()).all(), i


@pytest.mark.parametrize("shared", [0, 64])
def test_streams_and_graphs(cuda, shared):
    """Calls on several streams at once, and two captured graphs of one
    context replayed at the same time while eager calls run; lengths that
    change between replays."""
    import ter_amd as T
    one = Batch([(1, 64 + n) for n in (5, 200, 90)], common=64, seed=1)
    two = Batch([(30, 64 + 60), (1, 64 + 900)], common=64, seed=2)
    ctx = context(two)
    sets = []
    for b in (one, two):
        cache, batch = b.on_device(T)
        q = b.q.cuda()
        sets.append((q, cache, batch, ctx.attend(q, cache, batch, shared=shared)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    for _ in range(5):
        outs = []
        for st, (q, cache, batch, _) in zip(streams, sets):
            with torch.cuda.stream(st):
                outs += [ctx.attend(q, cache, batch, shared=shared) for _ in range(4)]
            outs.append(ctx.attend(q, cache, batch, shared=shared, stream=st.cuda_stream))
        torch.cuda.synchronize()
        for i, o in enumerate(outs):
            assert torch.equal(o, sets[i // 5][3]), "the same call, the same bits"
    graphs = []
    for q, cache, batch, _ in sets:
        out = torch.empty_like(q)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            ctx.attend(q, cache, batch, shared=shared, out=out)
        graphs.append((g, out))
    for rep in range(4):
        for (g, out), st in zip(graphs, streams):
            with torch.cuda.stream(st):
                out.zero_()
                g.replay()
        eager = ctx.attend(sets[0][0], sets[0][1], sets[0][2], shared=shared)
        torch.cuda.synchronize()
        assert torch.equal(eager, sets[0][3])
        for (g, out), s in zip(graphs, sets):
            assert torch.equal(out, s[3]), rep
    # other lengths through the same graph
    cut = Batch([(1, 64 + n) for n in (5, 200, 90)], common=64, seed=1)
    cut.lens = [66, 150, 70]
    sets[0][2].kv_len.copy_(torch.tensor(cut.lens, dtype=torch.int32))
    graphs[0][0].replay()
    want, tol = cut.attend()
    compare(graphs[0][1], want, tol, "replayed with other lengths")


def test_append_and_attend_in_one_graph(cuda):
    """A decode step (append, attend, the length counted up) captured once and
    replayed token by token, against eager steps."""
    import ter_amd as T
    b = Batch([(1, 40), (1, 7), (1, 100)], page=16)
    b.table[:] = np.arange(b.table.size).reshape(b.table.shape)
    n = b.table.size
    ctx = context(b, max_pos=400)
    kd, vd = (torch.randn(n, 16, b.nkv, b.hd).half().cuda() for _ in range(2))
    steps = [[torch.randn(3, h, b.hd).half().cuda() for h in (b.nh, b.nkv, b.nkv)] for _ in range(8)]
    start = torch.tensor([40, 7, 100], dtype=torch.int32, device="cuda") - 9

    def run(graph):
        cache = T.PagedCache(kd.clone(), vd.clone())
        lens = start.clone()
        batch = T.PagedBatch(torch.arange(4, dtype=torch.int32, device="cuda"), lens,
                             torch.from_numpy(b.table).cuda())
        buf = [torch.empty_like(x) for x in steps[0]]
        out = torch.empty_like(buf[0])

        def step():
            lens.add_(1)
            ctx.attend(ctx.append(*buf, cache, batch, q_out=buf[0]), cache, batch, out=out)

        if graph:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                step()
        got = []
        for s in steps:
            for x, y in zip(buf, s):
                x.copy_(y)
            g.replay() if graph else step()
            got.append(out.clone())
        return got, cache.k, cache.v

    e, g = run(False), run(True)
    assert torch.equal(e[1], g[1]) and torch.equal(e[2], g[2])
    for x, y in zip(e[0], g[0]):
        assert torch.equal(x, y)


def test_a_served_layer(cuda):
    """One layer of a Llama-shaped model for a batch of prompts and single
    tokens, as a server runs it: rows normed and quantized, Q/K/V as a GEMM
    list with fp16 outputs, append, attend, O: the framework's own products
    beside the operators, every step checked from what went into it."""
    import ter_amd as T
    from oracle import oracle as O
    H, nh, nkv, hd = 512, 8, 2, 64
    seqs = [(20, 20), (1, 77), (33, 60), (1, 5)]
    b = Batch(seqs, nh=nh, nkv=nkv, hd=hd)
    t = b.t
    g = torch.Generator().manual_seed(3)
    hidden = torch.randn(t, H, generator=g).cuda()
    gamma = (torch.rand(H, generator=g) + 0.5).half().cuda()
    W = {nm: T.PackedTrits.from_v11(O.v11_pack(O.rand_trits(i, H, n, 0.4)), H, n, 0.02)
         for i, (nm, n) in enumerate([("q", nh * hd), ("k", nkv * hd), ("v", nkv * hd), ("o", H)])}
    xq, xs = T.rmsnorm_quant(hidden, gamma, 1e-5)
    rows = {nm: torch.empty(t, n, dtype=F16, device="cuda") for nm, n in (("q", nh * hd), ("k", nkv * hd), ("v", nkv * hd))}
    T.GemmPlan([dict(w=W[nm], x=xq, x_scale_dev=xs, y16=rows[nm]) for nm in "qkv"]).launch()
    before = {nm: x.cpu().view(t, -1, hd) for nm, x in rows.items()}
    cache, batch = b.on_device(T)
    ctx = context(b)
    q = ctx.append(rows["q"], rows["k"], rows["v"], cache, batch, q_out=rows["q"])
    att = ctx.attend(q, cache, batch)
    aq, as_ = T.quant_int8(att.view(t, -1).float())
    y = torch.empty(t, H, dtype=torch.float32, device="cuda")
    T.mm_batched(W["o"], aq, y=y, x_scale_dev=as_)
    pos = [p for r, n in seqs for p in range(n - r, n)]
    for nm, got in (("q", q.view(t, nh, hd)), ("k", None)):
        want, tol = rotated(before[nm], pos, THETA, True, F16)
        if nm == "k":
            seq = [s for s, (r, _) in enumerate(seqs) for _ in range(r)]
            got = cache.k[[int(b.table[s, p // 16]) for s, p in zip(seq, pos)], [p % 16 for p in pos]]
        compare(got, want, tol, nm)
    b.q, b.k, b.v = q.view(t, nh, hd).cpu(), cache.k.cpu(), cache.v.cpu()
    want, tol = b.attend()
    compare(att, want, tol, "attention")
    _, ry = O.gemm_v11(aq.cpu().numpy(), as_.cpu().numpy(), W["o"].to_v11().cpu().numpy(), 0.02, nh * hd, H)
    assert (y.cpu().numpy().view(np.int32) == ry.view(np.int32)).all()


def test_python_refusals(cuda):
    """What the wrapper refuses, before anything is launched."""
    import ter_amd as T
    b = Batch([(1, 20), (2, 30)])
    cache, batch = b.on_device(T)
    ctx = context(b)
    q, k = b.q.cuda(), torch.zeros(3, b.nkv, b.hd, dtype=b.dtype, device="cuda")
    for bad in (q.float(), q.cpu(), q.to(BF16)):
        with pytest.raises(TypeError):
            ctx.attend(bad, cache, batch)
    for bad in (q[:, :2], q[:, :, :32], q.transpose(0, 1), q.view(-1)):
        with pytest.raises(ValueError):
            ctx.attend(bad, cache, batch)
    with pytest.raises(ValueError):
        ctx.attend(q, cache, batch, out=torch.empty_like(q)[:2])
    for scale in (0.0, 1e-50, math.nan):
        with pytest.raises(ValueError):
            ctx.attend(q, cache, batch, scale=scale)
    with pytest.raises(ValueError):
        ctx.append(q, k, k[:2], cache, batch)
    with pytest.raises(ValueError):
        ctx.append(None, k, k, cache, batch, q_out=q)
    for kd, vd in ((cache.k, cache.v[1:]), (cache.k, cache.v.to(BF16)), (cache.k[0], cache.v[0]),
                   (cache.k.transpose(2, 3), cache.v.transpose(2, 3))):
        with pytest.raises(ValueError):
            T.PagedCache(kd, vd)
    with pytest.raises(TypeError):
        T.PagedCache(cache.k.float(), cache.v.float())
    with pytest.raises(ValueError):
        T.PagedBatch(batch.row0[:2], batch.kv_len, batch.pages)
    with pytest.raises(TypeError):
        T.PagedBatch(batch.row0.long(), batch.kv_len, batch.pages)
    other = T.PagedCache(cache.k.to(BF16), cache.v.to(BF16))
    with pytest.raises(ValueError):
        ctx.attend(q, other, batch)
    from ter_amd._lib import TerHipError
    with pytest.raises(TerHipError):
        ctx.attend(q, cache, batch, shared=-1)
    odd = torch.zeros(4, 24, b.nkv, b.hd, dtype=b.dtype, device="cuda")
    with pytest.raises(TerHipError):
        ctx.attend(q, T.PagedCache(odd, odd), batch)
    shifted = torch.zeros(q.numel() + 8, dtype=b.dtype, device="cuda")[4:-4].view_as(q)
    with pytest.raises(TerHipError):
        ctx.attend(shifted, cache, batch)
