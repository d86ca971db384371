"""The 8-bit product by its definition, on the CPU: exact integer sums (in
binary64, whose 53 bits hold them), and the binary32 steps around them one by
one, each rounded as the operator defines it.  So results are compared bit for
bit, without a tolerance."""
import torch


def quantized(x):
    """(q int8, x_scale) of rows of any type."""
    x = x.float()
    s = torch.tensor(127.0) / (x.abs().amax(1) + torch.tensor(1e-9))
    q = (x * s[:, None]).round().clamp(-128, 127)
    return q, torch.tensor(1.0) / s


def product(x, xs, w, ws, dtype):
    """x, w: integers [M][K], [N][K] of any type; xs, ws fp32."""
    sums = x.double() @ w.double().t()
    if dtype == torch.int32:
        return sums.to(torch.int32)
    # (sums beyond 2^24 are rounded to binary32 first, as the conversion does)
    return (sums.to(torch.int64).float() * (xs[:, None] * ws)).to(dtype)


def bits(t):
    """The bits of a tensor's values, NaN as one value."""
    if t.dtype == torch.int32:
        return t
    t = torch.where(t.isnan(), torch.full_like(t, float("nan")), t)
    return t.view(torch.int32 if t.dtype == torch.float32 else torch.int16)


def same(a, b):
    assert a.dtype == b.dtype and a.shape == b.shape
    x, y = bits(a.cpu()), bits(b.cpu())
    bad = (x != y).nonzero()
    assert len(bad) == 0, f"{len(bad)} of {x.numel()} differ, first at {bad[0].tolist()}: " \
                          f"{a.cpu()[tuple(bad[0])]} against {b.cpu()[tuple(bad[0])]}"
