"""CPU checks of the sampling operator's boundary: every refusal comes before
device work.  (Header and binding: test_int8.py.)"""
import ctypes as C

import pytest

from ter_amd import _lib as L

A = 1 << 20  # an address that nothing may follow
NAN, INF = float("nan"), float("inf")


def call(p=None, **kw):
    a = dict(x=A, ty=L.T_F16, st=1000, rows=4, V=1000, u=A, t=A, prob=A, ws=A, nb=1 << 40)
    a.update(kw)
    s = L.SampleParams()
    s.temperature, s.top_p = 1.0, 1.0
    for k, v in (p or {}).items():
        setattr(s, k, v)
    return L.lib().ter_hip_sample(a["x"], a["ty"], a["st"], a["rows"], a["V"], a["u"], C.byref(s) if p != 0 else None,
                                  a["t"], a["prob"], a["ws"], a["nb"], None)


@pytest.mark.parametrize("kw,code", [
    (dict(x=None), L.ERR_NULL), (dict(u=None), L.ERR_NULL), (dict(t=None), L.ERR_NULL),
    (dict(ty=L.T_I8), L.ERR_PAYLOAD), (dict(ty=-1), L.ERR_PAYLOAD), (dict(ty=7), L.ERR_PAYLOAD),
    (dict(st=999), L.ERR_SHAPE), (dict(st=-1000), L.ERR_SHAPE), (dict(st=1 << 40), L.ERR_SHAPE),
    (dict(rows=-1), L.ERR_SHAPE), (dict(rows=(1 << 20) + 1), L.ERR_SHAPE),
    (dict(V=0), L.ERR_SHAPE), (dict(V=(1 << 19) + 1, st=1 << 20), L.ERR_SHAPE),
    (dict(x=A + 1), L.ERR_ALIGN), (dict(x=A + 2, ty=L.T_F32), L.ERR_ALIGN), (dict(u=A + 2), L.ERR_ALIGN),
    (dict(t=A + 1), L.ERR_ALIGN), (dict(prob=A + 3), L.ERR_ALIGN),
])
def test_refusals(kw, code):
    assert call(**kw) == code
    assert L.lib().ter_hip_last_error()


@pytest.mark.parametrize("p,code", [
    (dict(temperature=-0.1), L.ERR_SHAPE), (dict(temperature=NAN), L.ERR_SHAPE), (dict(temperature=INF), L.ERR_SHAPE),
    (dict(top_k=-1), L.ERR_SHAPE),
    (dict(top_p=-0.1), L.ERR_SHAPE), (dict(top_p=1.01), L.ERR_SHAPE), (dict(top_p=NAN), L.ERR_SHAPE),
    (dict(min_p=-0.1), L.ERR_SHAPE), (dict(min_p=1.01), L.ERR_SHAPE), (dict(min_p=NAN), L.ERR_SHAPE),
    (dict(temperature_dev=A + 1), L.ERR_ALIGN), (dict(top_k_dev=A + 2), L.ERR_ALIGN),
    (dict(top_p_dev=A + 1), L.ERR_ALIGN), (dict(min_p_dev=A + 1), L.ERR_ALIGN),
])
def test_refused_settings(p, code):
    assert call(p) == code


def test_no_rows():
    assert call(rows=0, x=None, u=None, t=None, prob=None) == L.OK
    assert call(0) == L.ERR_NULL
    assert L.lib().ter_hip_sample_ws(0, 10) == 0 and L.lib().ter_hip_sample_ws(-1, 10) == 0


def test_python_refusals():
    """Arguments that the binding itself refuses, without a device."""
    import torch

    import ter_amd as T
    x = torch.zeros(2, 5)
    with pytest.raises(TypeError):
        T.sample(x, torch.zeros(2))
    with pytest.raises(TypeError):
        T.PackedInt8.quantize(x)
    with pytest.raises(TypeError):
        T.PackedInt8.from_int8(x, x[0])
    with pytest.raises(ValueError):
        T.PackedInt8(0, 5)
