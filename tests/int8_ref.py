"""The 8-bit product by its definition, on the CPU: exact integer sums (in
binary64, whose 53 bits hold them), and the binary32 steps around them one by
one, each rounded as the operator defines it.  So results are compared bit for
bit, without a tolerance."""
import torch

# Sizes (rows, channels, K) for which a call on 256 CUs takes each of the tiles.
TILES = {
    "64x64": [(822, 282, 22), (1219, 1393, 69), (2000, 1000, 1500)],
    "96x256": [(3124, 766, 227), (1203, 2773, 654)],
    "128x256": [(2651, 2973, 36), (1296, 5610, 457)],
    "256x128": [(2687, 2524, 125), (1882, 3533, 323)],
    "160x256": [(4199, 2166, 35), (1162, 7279, 81), (1773, 5284, 161)],
    "192x256": [(4291, 7989, 100), (1529, 7368, 371)],
    "224x256": [(1602, 8023, 117), (1944, 6223, 314)],
    "256x256": [(8293, 3748, 51), (4047, 4051, 247)],
}


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
# few tiles of a long K, computed by parts of it
PARTS = [(380, 512, 8192), (65, 33, 9000), (209, 1282, 8192), (128, 2560, 6912), (70, 1003, 4097), (500, 40, 20000)]
