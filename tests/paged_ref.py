"""Batches over a paged cache for the tests, and their results in 64 bits from
the definitions, each with a bound on what the kernels' roundings can add up
to (so no test holds a tolerance that was tuned)."""
import math

import numpy as np
import torch


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def smallest(dtype):
    """Half the spacing of the subnormals."""
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2


class Batch:
    """seqs: (rows, kv_len) of each sequence.  Every slot of the cache that no
    sequence owns a position of holds NaN, so whatever reads or keeps a masked
    place shows.  common: the first `common` positions are one run of pages
    for all sequences (a multiple of page).  layout: order of the cache in
    memory ("phd", heads before positions "hpd", k and v interleaved "kv")."""

    def __init__(self, seqs, nh=4, nkv=2, hd=64, page=16, dtype=torch.float16, common=0, layout="phd", seed=0,
                 spare_rows=0, device="cuda", spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.nh, self.nkv, self.hd, self.page, self.dtype, self.device = nh, nkv, hd, page, dtype, device
        self.rows = [r for r, _ in seqs]
        self.lens = [n for _, n in seqs]
        first = np.concatenate([[0], np.cumsum(self.rows)]).astype(np.int32)
        self.first = first
        self.t = int(first[-1]) + spare_rows
        n_common = common // page
        assert common % page == 0
        need = [max(0, -(-n // page)) for n in self.lens]
        width = max(need + [1]) + 1
        n_pages = n_common + sum(max(0, k - n_common) for k in need) + 2
        ids = torch.randperm(n_pages, generator=g).tolist()
        table = np.full((len(seqs), width), -1, np.int32)
        nxt = n_common
        for b, k in enumerate(need):
            own = max(0, k - n_common)
            table[b, :min(k, n_common)] = ids[:min(k, n_common)]
            table[b, n_common:n_common + own] = ids[nxt:nxt + own]
            nxt += own
        self.table = table
        self.k = torch.full((n_pages, page, nkv, hd), math.nan, dtype=dtype)
        self.v = self.k.clone()
        for b, n in enumerate(self.lens):
            for p in range(need[b]):
                m = min(page, n - p * page)
                if p < n_common and not torch.isnan(self.k[table[b, p], m - 1, 0, 0]):
                    continue  # a common page that is filled this far already
                self.k[table[b, p], :m] = (torch.randn(m, nkv, hd, generator=g) * spread).to(dtype)
                self.v[table[b, p], :m] = torch.randn(m, nkv, hd, generator=g).to(dtype)
        self.q = (torch.randn(self.t, nh, hd, generator=g) * spread).to(dtype)
        self.layout = layout

    def pages_of(self, x):
        """A cache tensor of the batch's layout on the device, contents x."""
        if self.layout == "hpd":
            return x.permute(0, 2, 1, 3).contiguous().to(self.device).permute(0, 2, 1, 3)
        return x.to(self.device)

    def on_device(self, T):
        if self.layout == "kv":
            both = torch.stack([self.k, self.v], 1).to(self.device)
            kd, vd = both[:, 0], both[:, 1]
        else:
            kd, vd = self.pages_of(self.k), self.pages_of(self.v)
        cache = T.PagedCache(kd, vd)
        batch = T.PagedBatch(torch.from_numpy(self.first).to(self.device),
                             torch.tensor(self.lens, dtype=torch.int32, device=self.device),
                             torch.from_numpy(self.table).to(self.device))
        return cache, batch

    def positions(self, b, x):
        """Positions 0 .. kv_len - 1 of sequence b of a cache tensor (bad pages: zeros)."""
        out = torch.zeros(max(0, self.lens[b]), self.nkv, self.hd, dtype=torch.float64)
        for p in range(-(-max(0, self.lens[b]) // self.page)):
            m = min(self.page, self.lens[b] - p * self.page)
            i = int(self.table[b, p])
            if 0 <= i < x.shape[0]:
                out[p * self.page:p * self.page + m] = x[i, :m].double()
        return out

    def attend(self, scale=None, offset=0):
        """(result, bound) [t][nh][hd] of the rows; rows of no sequence are NaN in both."""
        u, hd = half_step(self.dtype), self.hd
        scale = 1 / math.sqrt(hd) if scale is None else scale
        want = torch.full((self.t, self.nh, hd), math.nan, dtype=torch.float64)
        tol = want.clone()
        f32 = 2.0 ** -24
        for b in range(len(self.rows)):
            n, r = self.lens[b], self.rows[b]
            k, v = self.positions(b, self.k), self.positions(b, self.v)
            for h in range(self.nh):
                g = h * self.nkv // self.nh
                q = self.q[self.first[b]:self.first[b + 1], h].double()
                lim = torch.arange(n - r, n) + 1
                for i in range(r):
                    at = int(self.first[b]) + i
                    m = int(lim[i])
                    if m <= 0:
                        want[at, h], tol[at, h] = 0.0, 0.0
                        continue
                    s = (k[:m, g] @ q[i]) * scale
                    w = torch.softmax(s, 0)
                    # a masked place takes no part: only visible rows are multiplied
                    want[at, h] = w @ v[:m, g]
                    mean = w @ v[:m, g].abs()
                    # scores: products summed in binary32, and their scaling;
                    # exp and the scaled maximum add a few units of 2^-24 of
                    # the exponent
                    ds = float(((k[:m, g].abs() @ q[i].abs()) * scale).max()) * (hd + 8) * f32 + 16 * f32
                    # weights rounded to the element type, sums of m terms in
                    # binary32, joined pieces, the result rounded
                    rel = 2 * ds + u + (m + 64) * f32
                    few = m * 2.0 ** -33 * float(v[:m, g].abs().max()) if self.dtype == torch.float16 else 0.0
                    tol[at, h] = mean * rel + few + (want[at, h].abs() + mean * rel) * u + smallest(self.dtype)
        return want, tol


def rotated(x, pos, theta, neox, dtype):
    """(result, bound) of the rotation of x [n][heads][hd] to positions pos [n]."""
    x = x.double()
    d = x.shape[-1]
    ang = torch.as_tensor(pos, dtype=torch.float64)[:, None] * float(theta) ** (
        -torch.arange(0, d, 2, dtype=torch.float64) / d)
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    a, z = (slice(0, d // 2), slice(d // 2, d)) if neox else (slice(0, d, 2), slice(1, d, 2))
    y, size = torch.empty_like(x), torch.empty_like(x)
    y[..., a], y[..., z] = x[..., a] * c - x[..., z] * s, x[..., a] * s + x[..., z] * c
    size[..., a] = size[..., z] = x[..., a].abs() + x[..., z].abs()
    # cos and sin, the product and the multiply-add rounded to binary32 (the
    # angle in 64 bits: 2^-53 of at most 2^20), then once to the element type
    e = size * (4 * 2.0 ** -24 + 2.0 ** -32)
    return y, (y.abs() + e) * half_step(dtype) + e + smallest(dtype)


def compare(got, want, tol, what=""):
    """got within tol of want where want is finite, equal where it is not."""
    got = got.double().cpu()
    fine = torch.isfinite(want)
    bad = (fine & ~((got - want).abs() <= tol)) | (~fine & (torch.isnan(got) != torch.isnan(want))) | \
        (~fine & ~torch.isnan(want) & (got != want))
    if bad.any():
        i = tuple(int(v) for v in bad.nonzero()[0])
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} off, first at {i}: got {got[i].item()}, "
                             f"want {want[i].item()}, allowed {tol[i].item()}")
