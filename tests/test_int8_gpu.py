"""The 8-bit product on the GPU against its definition, bit for bit: sizes
around every tile's edge, types, strides, alignments, values at their limits,
streams and graphs."""
import pytest
import torch

import ter_amd as T
from tests.int8_ref import PARTS, TILES, product, quantized, same

pytestmark = pytest.mark.gpu

FLOATS = (torch.float16, torch.bfloat16, torch.float32)


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(g, *shape):
    return torch.randint(-128, 128, shape, generator=g, dtype=torch.int16).to(torch.int8)


def scales(g, n):
    return torch.rand(n, generator=g) * 0.02 + 1e-4


def weights(g, n, k):
    w, ws = ints(g, n, k), scales(g, n)
    return T.PackedInt8.from_int8(w.cuda(), ws.cuda()), w, ws


SIZES = [
    # rows around 16 and 64, channels around 16 and 32, K around 16, 64 and 128
    (1, 1, 1), (1, 16, 64), (1, 17, 128), (2, 31, 65), (15, 33, 127), (16, 32, 128), (17, 64, 129), (3, 5, 257),
    (33, 100, 640), (64, 128, 256), (65, 129, 272), (127, 255, 512), (128, 256, 1024), (129, 257, 1040), (5, 2560, 2560),
    (1, 640, 2560), (7, 512, 2048), (257, 515, 387), (300, 1000, 2048), (1, 4099, 6912), (513, 769, 144), (1000, 31, 80),
    (1, 3, 20000), (19, 70, 9000),
    # few rows by so many channels that tiles take them
    (17, 9601, 128), (33, 10007, 200), (64, 9700, 130),
]


@pytest.mark.parametrize("m,n,k", SIZES)
def test_integer_rows(cuda, m, n, k):
    g = gen(m * 7 + n * 3 + k)
    W, w, ws = weights(g, n, k)
    x, xs = ints(g, m, k), scales(g, m)
    for dt in (torch.int32,) + FLOATS:
        same(T.mm_int8(W, x.cuda(), xs.cuda(), dtype=dt), product(x, xs, w, ws, dt))


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("m,n,k", SIZES)
def test_rows_quantized_within_the_call(cuda, m, n, k, dt):
    g = gen(m * 5 + n + k)
    W, w, ws = weights(g, n, k)
    x = (torch.randn(m, k, generator=g) * torch.rand(m, 1, generator=g) * 3).to(dt)
    q, xs = quantized(x)
    for out in FLOATS if n < 300 else (dt,):
        same(T.mm_int8(W, x.cuda(), dtype=out), product(q, xs, w, ws, out))


@pytest.mark.parametrize("m,n,k", [(1, 2048, 2048), (8, 2560, 2560), (40, 6912, 2560), (200, 2048, 8192), (700, 2560, 640),
                                   (2050, 1030, 1031), (4096, 512, 2048),
                                   # weights of 128 MiB and more pass the caches by
                                   (1, 131103, 1024), (9, 131103, 1024), (30, 131103, 1024), (100, 131103, 1024)])
def test_larger(cuda, m, n, k):
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int16).to(torch.int8)
    x = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int16).to(torch.int8)
    xs, ws = (torch.rand(i, generator=g, device="cuda") * 0.01 + 1e-5 for i in (m, n))
    W = T.PackedInt8.from_int8(w, ws)
    want = x.double() @ w.double().t().contiguous()
    assert torch.equal(T.mm_int8(W, x, dtype=torch.int32), want.to(torch.int32))
    want = want.to(torch.int32).float() * (xs[:, None] * ws)
    for dt in FLOATS:
        same(T.mm_int8(W, x, xs, dtype=dt), want.to(dt))


@pytest.mark.parametrize("m,n,k", [s for sizes in TILES.values() for s in sizes] + PARTS)
def test_every_tile(cuda, m, n, k):
    """Sizes that do not fill the last tiles, in several rounds of the GPU."""
    g = torch.Generator(device="cuda").manual_seed(m + n + k)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int16).to(torch.int8)
    wide = torch.randint(-128, 128, (m, k + 16), generator=g, device="cuda", dtype=torch.int16).to(torch.int8)
    x = wide[:, :k]
    xs, ws = (torch.rand(i, generator=g, device="cuda") * 0.01 + 1e-5 for i in (m, n))
    W = T.PackedInt8.from_int8(w, ws)
    want = (x.double() @ w.double().t().contiguous()).to(torch.int32)
    y = torch.full((m + 1, n + 8), -7, dtype=torch.int32, device="cuda")
    T.mm_int8(W, x, out=y[:m, :n])
    assert torch.equal(y[:m, :n], want)
    assert (y[m:] == -7).all() and (y[:, n:] == -7).all()
    y = torch.full((m + 1, n + 8), -7, dtype=torch.bfloat16, device="cuda")
    T.mm_int8(W, x, xs, out=y[:m, :n])
    assert torch.equal(y[:m, :n], (want.float() * (xs[:, None] * ws)).bfloat16())
    assert (y[m:] == -7).all() and (y[:, n:] == -7).all()


def test_the_largest_sums(cuda):
    """K at its limit with the values that make the largest sum: 128 * 128 *
    131071 is 2^31 - 2^14."""
    k = T._lib.INT8_K_MAX
    w = torch.full((3, k), -128, dtype=torch.int8)
    w[1] = 127
    x = torch.full((2, k), -128, dtype=torch.int8)
    W = T.PackedInt8.from_int8(w.cuda(), torch.ones(3).cuda())
    y = T.mm_int8(W, x.cuda(), dtype=torch.int32).cpu()
    assert y.tolist() == [[128 * 128 * k, -128 * 127 * k, 128 * 128 * k]] * 2


@pytest.mark.parametrize("dt", (torch.int8,) + FLOATS)
@pytest.mark.parametrize("m,n,k,pad,off", [(33, 70, 128, 16, 0), (33, 70, 128, 16, 16), (20, 50, 128, 1, 0),
                                           (20, 50, 128, 8, 3), (70, 40, 100, 28, 0), (3, 64, 37, 5, 1), (1, 64, 256, 7, 7),
                                           (260, 300, 256, 48, 16)])
def test_rows_of_wider_ones(cuda, m, n, k, pad, off, dt):
    """Parts of wider rows at any place, into parts of wider rows: nothing
    beside them is read into the results or written."""
    g = gen(m + n + k + pad + off)
    W, w, ws = weights(g, n, k)
    xs = scales(g, m)
    if dt == torch.int8:
        wide = ints(g, m, k + pad + off)
    else:
        wide = torch.randn(m, k + pad + off, generator=g).to(dt)
        wide[:, :off] = wide[:, off + k:] = float("nan")
    x = wide[:, off:off + k]
    q, s = (x, xs) if dt == torch.int8 else quantized(x)
    args = (xs.cuda(),) if dt == torch.int8 else ()
    for out in FLOATS:
        y = torch.full((m, n + 11), 7.0, dtype=out, device="cuda")
        T.mm_int8(W, wide.cuda()[:, off:off + k], *args, out=y[:, 3:n + 3])
        same(y[:, 3:n + 3].contiguous(), product(q, s, w, ws, out))
        assert (y[:, :3] == 7).all() and (y[:, n + 3:] == 7).all()


def test_rows_at_the_end_of_an_allocation(cuda):
    """Rows whose last value is the last of its memory."""
    g = gen(5)
    W, w, ws = weights(g, 40, 48)
    for off in (0, 5, 16):
        wide = ints(g, 19, 64)
        flat = wide.flatten().cuda()
        x = torch.as_strided(flat, (19, 48), (64, 1), 64 - 48)  # the last 48 of each row
        same(T.mm_int8(W, x, dtype=torch.int32), product(wide[:, 16:], None, w, ws, torch.int32))


@pytest.mark.parametrize("m", [1, 5, 40, 300])
@pytest.mark.parametrize("dt", FLOATS)
def test_infinities_and_nan_stay_in_their_rows(cuda, dt, m):
    g = gen(m)
    W, w, ws = weights(g, 77, 300)
    x = torch.randn(m, 300, generator=g).to(dt)
    q, xs = quantized(x)
    want = product(q, xs, w, ws, torch.float32)
    for i, v in enumerate((float("nan"), float("inf"), -float("inf"))):
        r = (i * 37) % m
        x[r, (i * 111) % 300] = v
        want[r] = float("nan")
    y = T.mm_int8(W, x.cuda(), dtype=torch.float32)
    same(y, want)


def test_rows_of_zeros_and_extremes(cuda):
    g = gen(9)
    W, w, ws = weights(g, 40, 130)
    x = torch.randn(6, 130, generator=g)
    x[0] = 0
    x[1] *= 1e-30  # below the 1e-9 in the scale's denominator
    x[2] *= 1e30
    x[3] = 3.4e38 * x[3].sign()
    x[4] = 0
    x[4, 7] = -2.5
    q, xs = quantized(x)
    for dt in FLOATS:
        same(T.mm_int8(W, x.cuda(), dtype=dt), product(q, xs, w, ws, dt))


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("n,k", [(1, 1), (33, 100), (64, 128), (100, 515), (7, 4000)])
def test_weights_quantized_and_back(cuda, n, k, dt):
    g = gen(n + k)
    w = (torch.randn(n, k + 3, generator=g) * 0.03).to(dt)
    if n > 3:
        w[2] = 0
    W = T.PackedInt8.quantize(w.cuda()[:, 1:k + 1])
    q, s = W.to_int8()
    want, ws = quantized(w[:, 1:k + 1])
    assert torch.equal(q.cpu(), want.to(torch.int8))
    same(s, ws)
    x, xs = ints(g, 3, k), scales(g, 3)
    same(T.mm_int8(W, x.cuda(), xs.cuda()), product(x, xs, want, ws, torch.float32))


def test_pack_and_back(cuda):
    g = gen(3)
    for n, k in ((1, 1), (31, 63), (96, 256), (130, 1000)):
        W, w, ws = weights(g, n, k)
        q, s = W.to_int8()
        assert torch.equal(q.cpu(), w)
        same(s, ws)


def test_no_rows(cuda):
    W, _, _ = weights(gen(1), 20, 30)
    y = T.mm_int8(W, torch.empty(0, 30, dtype=torch.float16, device="cuda"))
    assert y.shape == (0, 20) and y.dtype == torch.float16


def test_weights_filled_on_another_stream(cuda):
    """Their memory is that stream's, not what the current one still writes."""
    g = gen(12)
    q, ws = ints(g, 3000, 2000).cuda(), scales(g, 3000).cuda()
    w = q.float()
    st = torch.cuda.Stream()
    n = T.PackedInt8(2000, 3000).buf.numel()
    torch.cuda.synchronize()
    for fill in (lambda s: T.PackedInt8.from_int8(q, ws, stream=s), lambda s: T.PackedInt8.quantize(w, stream=s)):
        want = [t.cpu() for t in fill(None).to_int8()]
        busy = torch.empty(n, dtype=torch.uint8, device="cuda")
        for _ in range(200):
            busy.fill_(7)
        del busy
        W = fill(st.cuda_stream)
        torch.cuda.synchronize()
        for a, b in zip(W.to_int8(), want):
            assert torch.equal(a.cpu(), b)


def test_another_stream(cuda):
    """Given as a handle: the call's workspace comes from that stream's memory."""
    g = gen(2)
    W, w, ws = weights(g, 300, 700)
    x = torch.randn(50, 700, generator=g)
    q, xs = quantized(x)
    xd = x.cuda()
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    a = T.mm_int8(W, xd, dtype=torch.bfloat16, stream=st.cuda_stream)
    with torch.cuda.stream(st):
        b = T.mm_int8(W, xd, dtype=torch.bfloat16)
    st.synchronize()
    want = product(q, xs, w, ws, torch.bfloat16)
    same(a, want)
    same(b, want)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_captured_and_replayed(cuda, m):
    g = gen(m)
    W, w, ws = weights(g, 515, 1111)
    x = torch.randn(m, 1111, generator=g).half().cuda()
    y = torch.empty(m, 515, dtype=torch.float16, device="cuda")
    T.mm_int8(W, x, out=y)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            T.mm_int8(W, x, out=y)
        graphs.append(gr)
    for i in range(4):
        new = torch.randn(m, 1111, generator=g).half()
        x.copy_(new)
        y.zero_()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        same(y, product(*quantized(new), w, ws, torch.float16))
        T.mm_int8(W, x[:1])  # eager work between


@pytest.mark.parametrize("m,n,k", PARTS[:4])
def test_parts_of_k_in_graphs(cuda, m, n, k):
    """Rows quantized and parts' sums in one workspace: two graphs on two streams
    at once, replayed with new rows, beside eager calls."""
    g = gen(m)
    W, w, ws = weights(g, n, k)
    parts = []
    for dt in (torch.float16, torch.float32):
        x = torch.randn(m, k, generator=g).to(dt).cuda()
        T.mm_int8(W, x, dtype=torch.bfloat16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = T.mm_int8(W, x, dtype=torch.bfloat16)
        parts.append((graph, x, y, torch.cuda.Stream()))
    for _ in range(3):
        want = []
        for _, x, y, _ in parts:
            new = torch.randn(m, k, generator=g).to(x.dtype)
            x.copy_(new)
            y.fill_(7)
            want.append(product(*quantized(new), w, ws, torch.bfloat16))
        torch.cuda.synchronize()
        for graph, _, _, st in parts:
            with torch.cuda.stream(st):
                graph.replay()
        eager = [T.mm_int8(W, x, dtype=torch.bfloat16) for _, x, _, _ in parts]
        torch.cuda.synchronize()
        for (_, _, y, _), e, want_y in zip(parts, eager, want):
            same(y, want_y)
            same(e, want_y)
