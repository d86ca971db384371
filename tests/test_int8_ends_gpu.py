"""The 8-bit product, its weights and the draws on data whose last value is the
last of its memory (a block that the allocator maps by itself), at every alignment and
by every path."""
import pytest
import torch

import ter_amd as T
from tests.int8_ref import product, quantized, same
from tests.sample_ref import draw

pytestmark = pytest.mark.gpu

FLOATS = (torch.float16, torch.bfloat16, torch.float32)
BLOCK = 32 << 20  # bytes; blocks of 10 MiB and more are a mapping each


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int16).to(torch.int8)


def at_the_end(t, stride=None, off=0):
    """A copy of t [m][n], rows `stride` apart, that ends `off` elements before the
    end of a block."""
    m, n = t.shape
    stride = stride or n
    block = torch.full((BLOCK // t.element_size(),), 1, dtype=t.dtype, device="cuda")
    x = torch.as_strided(block, (m, n), (stride, 1), block.numel() - off - ((m - 1) * stride + n))
    x.copy_(t)
    return x


# few rows by one to four blocks of 16 and in tiles; K of one chunk to past the waves' first units
SHAPES = [(1, 16), (1, 48), (2, 112), (5, 16), (16, 144), (17, 48), (33, 272), (64, 16), (64, 640), (65, 144), (70, 48),
          (130, 1040), (300, 2064)]


@pytest.mark.parametrize("m,k", SHAPES)
@pytest.mark.parametrize("off,gap", [(0, 0), (0, 16), (0, 5), (5, 0), (16, 0)])
@pytest.mark.parametrize("n", [40, 600])
def test_integer_rows(cuda, m, k, n, off, gap):
    """Read in place where rows are aligned, laid out first where they are not."""
    g = gen(m + k + n)
    w, ws = ints(g, n, k), torch.rand(n, generator=g) * 0.01
    W = T.PackedInt8.from_int8(w.cuda(), ws.cuda())
    x, xs = ints(g, m, k), torch.rand(m, generator=g) * 0.01
    xd = at_the_end(x, k + gap, off)
    same(T.mm_int8(W, xd, dtype=torch.int32), product(x, None, w, ws, torch.int32))
    same(T.mm_int8(W, xd, xs.cuda(), dtype=torch.float16), product(x, xs, w, ws, torch.float16))


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("m,k", [(1, 1), (1, 2560), (4, 1000), (5, 16), (9, 2049), (20, 4100), (70, 144), (3, 8200), (2, 17000)])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_rows_quantized_within_the_call(cuda, m, k, off, dt):
    g = gen(m + k)
    w, ws = ints(g, 50, k), torch.rand(50, generator=g) * 0.01
    W = T.PackedInt8.from_int8(w.cuda(), ws.cuda())
    x = torch.randn(m, k, generator=g).to(dt)
    same(T.mm_int8(W, at_the_end(x, off=off)), product(*quantized(x), w, ws, dt))


@pytest.mark.parametrize("n,k", [(1, 1), (33, 100), (40, 256), (7, 2051)])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_weights(cuda, n, k, off):
    g = gen(n + k)
    q, s = ints(g, n, k), torch.rand(n, generator=g)
    scale = at_the_end(s[None], off=off)[0]
    back, sb = T.PackedInt8.from_int8(at_the_end(q, off=off), scale).to_int8()
    assert torch.equal(back.cpu(), q) and torch.equal(sb.cpu(), s)
    for dt in FLOATS:
        w = torch.randn(n, k, generator=g).to(dt)
        back, sb = T.PackedInt8.quantize(at_the_end(w, off=off)).to_int8()
        want, ws = quantized(w)
        assert torch.equal(back.cpu(), want.to(torch.int8)) and torch.equal(sb.cpu(), ws)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("m,v", [(1, 1), (1, 4097), (3, 20001), (2, 70), (300, 1003)])
@pytest.mark.parametrize("off", [0, 1, 8])
def test_draws(cuda, m, v, off, dt):
    g = gen(m + v)
    x, u = torch.randn(m, v, generator=g).to(dt), torch.rand(m, generator=g)
    xd = at_the_end(x, off=off)
    for kw in (dict(), dict(top_k=20, top_p=0.9), dict(temperature=0.0)):
        t = T.sample(xd, u.cuda(), **kw).cpu()
        for r in range(0, m, 1 + m // 8):
            assert t[r] == draw(x[r].double().numpy(), u[r].item(), **kw)[0]
