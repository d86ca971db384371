"""Sampling on the GPU against its definition: tokens are equal, probabilities
within the rounding of binary32 (2^-24) and of the weights (2^-42, and 2^-45 of
the sum)."""
import numpy as np
import pytest
import torch

import ter_amd as T
from tests.sample_ref import draw

pytestmark = pytest.mark.gpu

FLOATS = (torch.float16, torch.bfloat16, torch.float32)
# one rounding to binary32, and the weights' error in numerator and sum
PROB = 2.0 ** -24 + 2.0 ** -40


def at(v, i):
    return v if np.isscalar(v) else v[i].item()


def check(logits, u, prob=True, **kw):
    m = logits.shape[0]
    p = torch.full((m,), -5.0, device="cuda")
    dev = {k: v.cuda() if isinstance(v, torch.Tensor) else v for k, v in kw.items()}
    t = T.sample(logits.cuda(), u.cuda(), prob_out=p, **dev).cpu()
    assert t.dtype == torch.int32 and t.shape == (m,)
    p = p.cpu()
    x = logits.double().numpy()
    for r in range(m):
        token, want = draw(x[r], u[r].item(), **{k: at(v, r) for k, v in kw.items()})
        assert t[r].item() == token, f"row {r}: token {t[r].item()}, {token} by the definition"
        assert abs(p[r].item() - want) <= PROB * want, f"row {r}: probability {p[r].item()}, {want}"
    return t


def rows(seed, m, v, dt, spread=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(m, v, generator=g) * spread).to(dt), torch.rand(m, generator=g)


SETTINGS = [
    dict(),
    dict(temperature=0.0),
    dict(temperature=0.7, top_k=1),
    dict(temperature=0.8, top_k=50, top_p=0.95),
    dict(top_k=1000),
    dict(top_p=0.9),
    dict(top_p=0.5, min_p=0.02),
    dict(min_p=0.1),
    dict(temperature=0.05, top_k=300, top_p=0.99, min_p=0.001),
    dict(temperature=1.9, top_k=5000, top_p=0.97),
    dict(temperature=3.0, top_p=0.999),
]


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("kw", SETTINGS, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()) or "all")
@pytest.mark.parametrize("m,v", [(1, 1), (3, 2), (2, 63), (4, 1000), (2, 4097), (3, 32003), (2, 128256)])
def test_settings(cuda, m, v, kw, dt):
    check(*rows(m + v, m, v, dt), **kw)


@pytest.mark.parametrize("m", [17, 130, 300])
@pytest.mark.parametrize("dt", FLOATS)
def test_many_rows(cuda, m, dt):
    check(*rows(m, m, 5003, dt), temperature=0.9, top_k=400, top_p=0.93, min_p=0.002)
    check(*rows(m + 1, m, 5003, dt), top_p=0.93)
    check(*rows(m + 2, m, 5003, dt))


@pytest.mark.parametrize("m,v", [(40, 3001), (6, 128256), (270, 900)])
def test_settings_of_each_row(cuda, m, v):
    g = torch.Generator().manual_seed(m)
    i = torch.arange(m)
    kw = dict(temperature=torch.rand(m, generator=g) * 2 * (i % 7 != 3), top_k=(torch.rand(m, generator=g) * 60).int() * (i % 3 != 1),
              top_p=torch.where(i % 4 == 0, torch.rand(m, generator=g), torch.tensor(1.0)),
              min_p=torch.where(i % 5 == 0, torch.rand(m, generator=g) * 0.3, torch.tensor(0.0)))
    kw["top_k"] = kw["top_k"].int()
    check(*rows(m + v, m, v, torch.float16), **kw)


@pytest.mark.parametrize("dt", FLOATS)
def test_settings_out_of_range_on_the_device(cuda, dt):
    """What the host refuses as a number counts as off (or as the limit) in a tensor."""
    nan, inf = float("nan"), float("inf")
    t = [1, -1, nan, inf, 1, 1, 1, 1, 1, 1e-45, 1e38]
    k = [-3, 5, 5, 5, 9999, 5, 5, 5, 5, 5, 0]
    p = [1, .5, .5, .5, 7, nan, 0, -1, .5, .5, 1]
    q = [0, 0, 0, 0, 0, 0, 0, nan, 3, 0, -1]
    u = [.5, .5, .5, .5, .5, 1.5, -1, nan, .5, .5, .9]
    m = len(t)
    x, _ = rows(7, m, 777, dt)
    check(x, torch.tensor(u), temperature=torch.tensor(t, dtype=torch.float32), top_k=torch.tensor(k, dtype=torch.int32),
          top_p=torch.tensor(p, dtype=torch.float32), min_p=torch.tensor(q, dtype=torch.float32))


def spread_u(m):
    return torch.tensor([(2 * i + 1) / (2 * m) for i in range(m)])


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("v", [1, 5, 1000, 4096, 40000])
@pytest.mark.parametrize("value", [0.0, -65504.0, 11.5])
def test_equal_logits(cuda, v, dt, value):
    """Every token alike: the draw goes by the index, cuts by the lowest."""
    m = 8
    x = torch.full((m, v), value).to(dt)
    u = spread_u(m)
    check(x, u)
    check(x, u, top_k=37)
    check(x, u, top_p=0.3)
    check(x, u, top_k=2000, top_p=0.25)
    check(x, u, min_p=1.0)
    check(x, torch.tensor([0.5] * m))  # u times the sum is a running sum: the next one


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("v", [300, 9000, 70000])
def test_ties_at_a_cut(cuda, v, dt):
    """A few distinct values: cuts and draws fall within equal ones."""
    g = torch.Generator().manual_seed(v)
    x = torch.randint(-3, 4, (12, v), generator=g).to(dt)
    x[:, 3] = 0.0
    x[:, 4] = -0.0
    u = spread_u(12)
    check(x, u)
    check(x, u, top_k=v // 9)
    check(x, u, top_p=0.61)
    check(x, u, top_k=v // 3, top_p=0.77, min_p=0.01)
    check(x, u, temperature=0.0)
    check(x, u, temperature=50.0, top_p=0.7)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("v", [50, 20000])
def test_masked_logits(cuda, v, dt):
    """-infinity and NaN are never drawn; rows with one token left, and none."""
    x, u = rows(v, 8, v, dt)
    x[0, ::2] = -float("inf")
    x[1, 1:] = -float("inf")
    x[2, :-1] = float("nan")
    x[3] = -float("inf")
    x[4] = float("nan")
    x[5, : v // 2] = float("nan")
    x[6] = torch.finfo(dt).min  # the type's lowest value is a number
    x[6, 7] = -float("inf")
    x[7, ::3] = torch.finfo(dt).min
    for kw in (dict(), dict(top_k=v // 2 + 3), dict(top_p=0.9), dict(top_k=3, top_p=0.5, min_p=0.1), dict(temperature=0.0)):
        t = check(x, u, **kw)
        assert t[1] == 0 and t[2] == v - 1 and t[3] == -1 and t[4] == -1


@pytest.mark.parametrize("dt", FLOATS)
def test_infinite_logits(cuda, dt):
    x, u = rows(4, 3, 3000, dt)
    x[0, 17] = float("inf")
    x[1, [5, 900, 2999]] = float("inf")
    x[2] = float("inf")
    u = torch.tensor([0.99, 0.5, 0.75])
    assert check(x, u).tolist() == [17, 900, 2250]
    check(x, u, top_k=2, top_p=0.4)
    check(x, u, temperature=0.0)


@pytest.mark.parametrize("dt", FLOATS)
def test_ends_of_u(cuda, dt):
    x, _ = rows(6, 4, 9001, dt)
    u = torch.tensor([0.0, 2.0 ** -30, 1 - 2.0 ** -24, 0.5])
    for kw in (dict(), dict(top_k=100), dict(top_p=0.8)):
        t = check(x, u, **kw)
        assert t[0] == int(x[0].float().argmax())


def test_far_apart_and_close_logits(cuda):
    """Scores of any size; and values a rounding apart, which only binary64
    tells apart in a sum."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(6, 5000, generator=g)
    x[1] *= 1e4
    x[2] = 1e30 * x[2]
    x[3] = 1000.0 + x[3] * 1e-3
    x[4] = 1.0 + torch.arange(5000) * 2.0 ** -23
    x[5] = -3.0e38
    x[5, 40] = 3.0e38
    u = torch.rand(6, generator=g)
    for kw in (dict(), dict(top_k=700), dict(top_p=0.7), dict(top_p=0.7, top_k=2500, min_p=0.2), dict(temperature=1e4)):
        check(x, u, **kw)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("m,v,pad", [(1, 1, 0), (9, 70, 3), (3, 4097, 1), (2, 128256, 0), (300, 9001, 5), (700, 64, 0)])
def test_largest_of_every_row(cuda, m, v, pad, dt):
    """Temperature 0 and top_k 1 on the host, which go a way of their own, as on
    the device: of equal logits the lower index, rows masked or infinite."""
    g = torch.Generator().manual_seed(m + v)
    x = (torch.randn(m, v + pad, generator=g) * 2).round().to(dt)
    x[m // 2, : v // 2] = float("nan")
    x[m // 3, pad:] = -float("inf")
    x[m - 1, v // 3:] = 1e4
    if m > 4:
        x[3, 1::7] = float("inf")
        x[4, pad:] = float("nan")
        x[5] = -0.0
        x[5, ::2] = 0.0
        x[6] = torch.finfo(dt).min
        x[7] = torch.finfo(dt).max
        x[7, v // 2:] = float("inf")
    u = torch.rand(m, generator=g)
    part = x[:, pad:]
    want = check(part[:8], u[:8], temperature=0.0)
    on_device = T.sample(x.cuda()[:, pad:], u.cuda(), temperature=torch.zeros(m, device="cuda")).cpu()
    assert torch.equal(on_device[:8], want)
    for kw in (dict(temperature=0.0), dict(temperature=0.0, top_p=0.5, min_p=0.2, top_k=v), dict(top_k=1),
               dict(top_k=1, temperature=torch.full((m,), 1.5, device="cuda"), top_p=0.1)):
        p = torch.full((m,), -1.0, device="cuda")
        t = T.sample(x.cuda()[:, pad:], u.cuda(), prob_out=p, **kw).cpu()
        assert torch.equal(t, on_device)
        assert torch.equal(p.cpu(), (on_device >= 0).float())


@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("t", [1e-37, 1e-38, 1e-40, 2.0 ** -149])
def test_temperatures_near_zero(cuda, t, m):
    """Those below 2^-120 count as it: logits within a few times that of each
    other, up to thousands of times the temperature given, and ordinary ones."""
    g = torch.Generator().manual_seed(9)
    x = torch.randn(m, 4500, generator=g) * 1e-36
    x[1::2] *= 1e3
    x[1::4] *= 1e33
    x[0, :50] -= 1e-35
    temps = torch.full((m,), t)
    for kw in (dict(), dict(top_k=700, top_p=0.9), dict(top_k=2000, min_p=1e-4)):
        want = check(x, u := torch.rand(m, generator=g), temperature=2.0 ** -120, **kw)
        for temperature in (t, temps.cuda()):
            got = T.sample(x.cuda(), u.cuda(), temperature=temperature, **kw)
            assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("m", [2, 300])
@pytest.mark.parametrize("spread,v", [(1e-4, 3000), (1e-4, 20000), (3e-3, 20000), (0.0, 20000), (1e-5, 70000)])
def test_a_cluster_far_below_the_largest(cuda, spread, v, m):
    """One logit far above, all others within a bin or a part of one: of different
    values, more than lists hold, and of equal ones."""
    g = torch.Generator().manual_seed(v)
    x = -12.0 + torch.randn(m, v, generator=g) * spread
    x[:, 77] = 0.0
    u = spread_u(m)
    for kw in (dict(), dict(top_k=v // 2), dict(top_p=0.9), dict(top_k=900, top_p=0.95), dict(temperature=2.0, min_p=1e-3)):
        if m > 2:
            check(x[::60], u[::60], **kw)
            whole = T.sample(x.cuda(), u.cuda(), **kw)
            assert torch.equal(whole[::60], T.sample(x[::60].cuda(), u[::60].cuda(), **kw))
        else:
            check(x, u, **kw)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("v", [4095, 4096, 4097, 8191, 12289, 20001])
def test_vocabularies_around_a_slice(cuda, v, dt):
    """The largest logit, the cuts and the token at the ends of slices."""
    x, u = rows(v, 7, v, dt)
    for r, i in enumerate((0, v - 1, v // 2, v // 2 - 1, (v + 1) // 2, 4095 % v, 4096 % v)):
        x[r, i] = 9.0
    check(x, u)
    check(x, u, top_k=1)
    check(x, u, top_k=1024)
    check(x, u, top_k=1025, top_p=0.99)
    check(x, torch.full((7,), 0.9999), top_p=0.9)


@pytest.mark.parametrize("dt", FLOATS)
@pytest.mark.parametrize("pad,off", [(1, 0), (5, 3), (8, 8), (13, 1)])
def test_rows_of_wider_ones(cuda, dt, pad, off):
    wide, u = rows(pad, 5, 3000 + pad + off, dt)
    wide[:, :off] = 60000.0
    wide[:, off + 3000:] = 60000.0
    x = wide[:, off:off + 3000]
    got = T.sample(wide.cuda()[:, off:off + 3000], u.cuda(), top_k=20, temperature=0.5)
    assert got.tolist() == [draw(x[r].double().numpy(), u[r].item(), 0.5, 20)[0] for r in range(5)]


def test_the_largest_vocabulary(cuda):
    v = T._lib.SAMPLE_V_MAX
    x, u = rows(3, 2, v, torch.float32)
    check(x, u, top_p=0.95)
    check(x, u)
    check(torch.zeros(1, v, dtype=torch.float16), torch.tensor([0.75]))


def test_offsets_past_2_to_the_32(cuda):
    """Rows of which some lie beyond 2^32 bytes."""
    v, m = 1 << 19, 4200
    big = torch.zeros(m * v, dtype=torch.float16, device="cuda")
    x = big.view(m, v)
    u = torch.rand(m, device="cuda")
    x[4199, 77] = 40.0
    x[4100, v - 1] = 40.0
    t = T.sample(x, u, top_k=1)
    want = torch.zeros(m, dtype=torch.int32)
    want[4199], want[4100] = 77, v - 1
    assert torch.equal(t.cpu(), want)
    p = torch.empty(m, device="cuda")
    t = T.sample(x, u, top_p=0.3, prob_out=p).cpu()
    assert t[4199] == 77 and t[4100] == v - 1
    del big, x


def test_the_same_in_every_batch(cuda):
    """A row's token depends on neither its batch nor the launch."""
    x, u = rows(11, 64, 50257, torch.bfloat16)
    x, u = x.cuda(), u.cuda()
    for kw in (dict(temperature=0.9), dict(top_k=40), dict(top_p=0.95)):
        whole = T.sample(x, u, **kw)
        assert torch.equal(whole, T.sample(x, u, **kw))
        for n in (1, 7, 30):
            assert torch.equal(whole[:n], T.sample(x[:n].contiguous(), u[:n], **kw))


def test_no_rows_and_outputs_of_the_caller(cuda):
    assert T.sample(torch.empty(0, 9, dtype=torch.float16, device="cuda"), torch.empty(0, device="cuda")).shape == (0,)
    x, u = rows(2, 3, 100, torch.float32)
    out = torch.full((5,), -9, dtype=torch.int32, device="cuda")
    T.sample(x.cuda(), u.cuda(), out=out[1:4])
    assert out[0] == -9 and out[4] == -9 and (out[1:4] >= 0).all()


def test_another_stream(cuda):
    x, u = rows(8, 9, 30000, torch.float16)
    xd, ud = x.cuda(), u.cuda()
    want = T.sample(xd, ud, top_p=0.9)
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    a = T.sample(xd, ud, top_p=0.9, stream=st.cuda_stream)
    with torch.cuda.stream(st):
        b = T.sample(xd, ud, top_p=0.9)
    st.synchronize()
    assert torch.equal(a, want) and torch.equal(b, want)


@pytest.mark.parametrize("m", [1, 20, 300])
def test_captured_and_replayed(cuda, m):
    """Two graphs, replayed in turn with eager work between: settings, logits
    and random numbers are read when they run."""
    x, u = rows(m, m, 6007, torch.float16)
    x, u = x.cuda(), u.cuda()
    k = torch.full((m,), 30, dtype=torch.int32, device="cuda")
    t = torch.empty(m, dtype=torch.int32, device="cuda")
    T.sample(x, u, top_k=k, out=t)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            T.sample(x, u, top_k=k, out=t)
        graphs.append(gr)
    for i in range(4):
        nx, nu = rows(100 + m + i, m, 6007, torch.float16)
        x.copy_(nx)
        u.copy_(nu)
        k.fill_(0 if i == 2 else 10 + i)
        t.zero_()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        got = t.cpu()
        T.sample(x[:1], u[:1], top_p=0.5)
        for r in range(min(m, 20)):
            assert got[r] == draw(nx[r].double().numpy(), nu[r].item(), top_k=0 if i == 2 else 10 + i)[0]
