"""CPU checks of sizes that the C-ABI takes in 32 bits: the binding refuses those
past them, where the rest of the number would be a smaller size that is in range."""
import types

import pytest
import torch

import ter_amd as T


class Shape(torch.Tensor):
    """A CUDA tensor of any size, without memory or a device."""

    @staticmethod
    def __new__(cls, shape, dtype):
        return torch.Tensor._make_wrapper_subclass(cls, shape, dtype=dtype, device="cuda:0")

    @classmethod
    def __torch_dispatch__(cls, func, args, *rest):
        raise AssertionError(f"{func} of a tensor without memory")


@pytest.fixture
def reached(monkeypatch):
    """What a call comes to behind its checks, instead of memory and launches."""
    class Reached(Exception):
        pass

    def stop(*args):
        raise Reached

    monkeypatch.setattr(T.fabric, "_empty_on", stop)
    monkeypatch.setattr(T.fabric, "_launch_on", stop)
    return Reached


@pytest.mark.parametrize("dt", (torch.int8, torch.float16, torch.float32))
@pytest.mark.parametrize("m", [1 << 31, (1 << 32) + 5, 1 << 40])
def test_rows_of_a_product(reached, m, dt):
    W = types.SimpleNamespace(K=1, N=1, _dev=0, _ref=None)
    scale = [Shape((m,), torch.float32)] * (dt == torch.int8)
    out = Shape((m, 1), torch.float32)
    for kw in (dict(), dict(out=out)):
        with pytest.raises(ValueError, match="too many"):
            T.mm_int8(W, Shape((m, 1), dt), *scale, **kw)
    # (the checks let the others pass)
    few = [Shape((5,), torch.float32)] * (dt == torch.int8)
    with pytest.raises(reached):
        T.mm_int8(W, Shape((5, 1), dt), *few)


@pytest.mark.parametrize("dt", (torch.bfloat16, torch.float32))
@pytest.mark.parametrize("m,v", [(1 << 31, 1), ((1 << 32) + 5, 1), (1, 1 << 31), (3, (1 << 32) + 1000)])
def test_rows_and_vocabulary_of_a_draw(reached, m, v, dt):
    u, token = Shape((m,), torch.float32), Shape((m,), torch.int32)
    for kw in (dict(), dict(out=token, prob_out=u)):
        with pytest.raises(ValueError, match="too many"):
            T.sample(Shape((m, v), dt), u, **kw)
    with pytest.raises(reached):
        T.sample(Shape((5, 1000), dt), Shape((5,), torch.float32))
