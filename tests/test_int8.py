"""CPU checks of the 8-bit product's boundary: the header, the binding and the
library agree, and every refusal comes before device work."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

from ter_amd import _lib as L

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
A = 1 << 20  # an address that nothing may follow


@pytest.mark.parametrize("header,signatures,consts", [
    ("ter_hip_int8.h", L.INT8_SIGNATURES,
     {"INT8_K_MAX": L.INT8_K_MAX, "INT8_N_MAX": L.INT8_N_MAX, "INT8_M_MAX": L.INT8_M_MAX, "INT8_Y_MAX": L.INT8_Y_MAX,
      "T_F16": L.T_F16, "T_BF16": L.T_BF16, "T_F32": L.T_F32, "T_I8": L.T_I8, "T_I32": L.T_I32}),
    ("ter_hip_sample.h", L.SAMPLE_SIGNATURES,
     {"SAMPLE_V_MAX": L.SAMPLE_V_MAX, "SAMPLE_ROWS_MAX": L.SAMPLE_ROWS_MAX}),
])
def test_header_binding_and_library_agree(header, signatures, consts, tmp_path):
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", header)).read(), flags=re.S)
    names = set(re.findall(r"^[A-Za-z_][\w\s\*]*?\b(ter_hip_\w+)\s*\(", text, flags=re.M))
    assert names == {n for n, _, _ in signatures}
    for n in names:
        assert hasattr(L.lib(), n)
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not installed")
    src = tmp_path / "t.c"
    checks = "".join(f"    if (TER_HIP_{k} != {v}ll) return 1;\n" for k, v in consts.items())
    sizes = {"ter_hip_int8.h": [("ter_hip_w8_t", L.W8), ("ter_hip_rows_t", L.Rows)],
             "ter_hip_sample.h": [("ter_hip_sample_params_t", L.SampleParams)]}[header]
    checks += "".join(f"    if (sizeof({t}) != {C.sizeof(s)}) return 2;\n" for t, s in sizes)
    src.write_text(f'#include "{header}"\nint main(void) {{\n{checks}    return 0;\n}}\n')
    r = subprocess.run([gcc, "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"),
                        str(src), "-o", str(tmp_path / "t")], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    assert subprocess.run([str(tmp_path / "t")], timeout=60).returncode == 0


def weight(K=100, N=40, **kw):
    w = L.W8()
    assert L.lib().ter_hip_w8_init(C.byref(w), A, 1 << 40, K, N) == L.OK
    for k, v in kw.items():
        setattr(w, k, v)
    return w


@pytest.mark.parametrize("K,N,ok", [(1, 1, True), (0, 5, False), (5, 0, False), (-1, 5, False), (131071, 1, True),
                                    (131072, 1, False), (1, 1 << 23, True), (1, (1 << 23) + 1, False)])
def test_shapes(K, N, ok):
    n = L.lib().ter_hip_w8_bytes(K, N)
    assert (n > 0) == ok
    w = L.W8()
    assert L.lib().ter_hip_w8_init(C.byref(w), A, 1 << 62, K, N) == (L.OK if ok else L.ERR_SHAPE)
    if ok:
        # tiles of whole 32-channel pairs and 128-value units, and the scales
        assert n == -(-N // 32) * -(-K // 128) * 4096 + -(-N // 32) * 32 * 4
        assert L.lib().ter_hip_w8_init(C.byref(w), A, n, K, N) == L.OK
        assert L.lib().ter_hip_w8_init(C.byref(w), A, n - 1, K, N) == L.ERR_SHAPE
        assert L.lib().ter_hip_w8_init(C.byref(w), A + 128, n, K, N) == L.ERR_ALIGN
        assert L.lib().ter_hip_w8_init(C.byref(w), None, n, K, N) == L.ERR_NULL
        assert L.lib().ter_hip_w8_init(None, A, n, K, N) == L.ERR_NULL


def test_weight_refusals():
    lib = L.lib()
    w = weight()
    r = C.byref(w)
    assert lib.ter_hip_w8_pack(None, A, 100, A, None) == L.ERR_NULL
    assert lib.ter_hip_w8_pack(r, None, 100, A, None) == L.ERR_NULL
    assert lib.ter_hip_w8_pack(r, A, 99, A, None) == L.ERR_SHAPE
    assert lib.ter_hip_w8_pack(r, A, 1 << 40, A, None) == L.ERR_SHAPE
    assert lib.ter_hip_w8_pack(r, A, 100, None, None) == L.ERR_NULL
    assert lib.ter_hip_w8_pack(r, A, 100, A + 2, None) == L.ERR_ALIGN
    assert lib.ter_hip_w8_quantize(r, None, L.T_F16, 100, None) == L.ERR_NULL
    assert lib.ter_hip_w8_quantize(r, A, L.T_I8, 100, None) == L.ERR_PAYLOAD
    assert lib.ter_hip_w8_quantize(r, A, -1, 100, None) == L.ERR_PAYLOAD
    assert lib.ter_hip_w8_quantize(r, A + 1, L.T_F16, 100, None) == L.ERR_ALIGN
    assert lib.ter_hip_w8_quantize(r, A + 2, L.T_F32, 100, None) == L.ERR_ALIGN
    assert lib.ter_hip_w8_unpack(r, None, A + 1, None) == L.ERR_ALIGN
    assert lib.ter_hip_w8_unpack(r, None, None, None) == L.OK
    for bad, code in ((weight(K=100, bytes=10), L.ERR_SHAPE), (weight(data=A + 16), L.ERR_ALIGN),
                      (weight(scale=None), L.ERR_NULL)):
        assert lib.ter_hip_w8_unpack(C.byref(bad), A, A, None) == code
    w.K = 0
    assert lib.ter_hip_w8_unpack(C.byref(w), A, A, None) == L.ERR_SHAPE


def rows(**kw):
    r = L.Rows(A, A, 100, L.T_I8, 7)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


@pytest.mark.parametrize("row,y,code", [
    (dict(data=None), {}, L.ERR_NULL),
    (dict(scale=None), {}, L.ERR_NULL),
    (dict(scale=A + 2), {}, L.ERR_ALIGN),
    (dict(stride=99), {}, L.ERR_SHAPE),
    (dict(stride=-100), {}, L.ERR_SHAPE),
    (dict(type=L.T_I32), {}, L.ERR_PAYLOAD),
    (dict(type=-1), {}, L.ERR_PAYLOAD),
    (dict(type=9), {}, L.ERR_PAYLOAD),
    (dict(n=-1), {}, L.ERR_SHAPE),
    (dict(n=(1 << 23) + 1), {}, L.ERR_SHAPE),
    (dict(type=L.T_F16, data=A + 1), {}, L.ERR_ALIGN),
    (dict(type=L.T_F32, data=A + 2), {}, L.ERR_ALIGN),
    ({}, dict(y=None), L.ERR_NULL),
    ({}, dict(y=A + 1), L.ERR_ALIGN),
    ({}, dict(ys=39), L.ERR_SHAPE),
    ({}, dict(yt=L.T_I8), L.ERR_PAYLOAD),
    ({}, dict(yt=5), L.ERR_PAYLOAD),
    ({}, dict(yt=-1), L.ERR_PAYLOAD),
    (dict(type=L.T_F16), dict(yt=L.T_I32), L.ERR_PAYLOAD),
    ({}, dict(ws=None), L.ERR_NULL),
    ({}, dict(ws=A + 8), L.ERR_ALIGN),
    ({}, dict(nb=7 * 132 - 1), L.ERR_SHAPE),
])
def test_product_refusals(row, y, code):
    a = dict(y=A, ys=40, yt=L.T_F16, ws=A, nb=1 << 30)
    a.update(y)
    w, r = weight(), rows(**row)
    assert L.lib().ter_hip_w8_mm(C.byref(w), C.byref(r), a["y"], a["ys"], a["yt"], a["ws"], a["nb"], None) == code
    assert L.lib().ter_hip_last_error()


def test_no_rows_and_workspaces():
    lib = L.lib()
    w = weight()
    assert lib.ter_hip_w8_mm(C.byref(w), C.byref(rows(n=0, data=None)), None, 0, L.T_F16, None, 0, None) == L.OK
    assert lib.ter_hip_w8_mm(C.byref(w), None, A, 40, L.T_F16, A, 1 << 30, None) == L.ERR_NULL
    assert lib.ter_hip_w8_mm(None, C.byref(rows()), A, 40, L.T_F16, A, 1 << 30, None) == L.ERR_NULL

    def ws(w, **kw):
        return lib.ter_hip_w8_mm_ws(C.byref(w), C.byref(rows(**kw)))

    assert ws(w) == 7 * 132  # K = 100: laid out first
    assert ws(w, n=0) == 0 and ws(w, stride=99) == 0
    w = weight(K=112)
    assert ws(w, stride=112) == 0 and ws(w, stride=128) == 0
    assert ws(w, stride=120) == 7 * 132 and ws(w, stride=112, data=A + 8) == 7 * 132
    assert ws(w, stride=113, n=1) == 0
    assert ws(w, stride=112, type=L.T_BF16) == 7 * 132
    # more results than a call takes
    w = weight(K=16, N=1 << 23)
    assert ws(w, stride=16, n=1 << 14) == 0
    r = rows(stride=16, n=1 << 14)
    assert lib.ter_hip_w8_mm(C.byref(w), C.byref(r), A, 1 << 23, L.T_F16, A, 1 << 30, None) == L.ERR_SHAPE
