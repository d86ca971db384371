"""CPU checks of the 8-bit product's boundary: the header, the binding and the
library agree, and every refusal comes before device work."""
import ctypes as C
import os
import re
import shutil
import subprocess
import sys
import textwrap

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


# ---- what a call launches, over the HIP runtime without a device

PRELUDE = """
import ctypes as C, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
fake.fake_log.restype = C.c_char_p
fake.fake_fail.argtypes = [C.c_char_p]
from ter_amd import _lib as L
lib = C.CDLL(L.LIB_PATH)
for name, res, args in L.SIGNATURES + L.INT8_SIGNATURES + L.SAMPLE_SIGNATURES:
    f = getattr(lib, name)
    f.restype, f.argtypes = res, args
A = 1 << 20
def log():
    lines = fake.fake_log().decode().splitlines()
    fake.fake_reset()
    return lines
def mm(M, N, K, xt=L.T_I8, yt=L.T_F16, stride=None):
    w = L.W8()
    assert lib.ter_hip_w8_init(C.byref(w), A, 1 << 60, K, N) == 0, lib.ter_hip_last_error()
    x = L.Rows(A, A, stride or K, xt, M)
    need = lib.ter_hip_w8_mm_ws(C.byref(w), C.byref(x))
    return lib.ter_hip_w8_mm(C.byref(w), C.byref(x), A, N, yt, A if need else None, need, None)
def draw(rows, V, ty=L.T_F16, temperature=1.0, top_k=0, dev=None):
    p = L.SampleParams()
    p.temperature, p.top_p, p.top_k, p.temperature_dev = temperature, 1.0, top_k, dev
    need = lib.ter_hip_sample_ws(rows, V)
    return lib.ter_hip_sample(A, ty, V, rows, V, A, C.byref(p), A, None, A if need else None, need, None)
def kernels():
    # (device, blocks, threads, LDS, name) of the launches
    return [l.split(None, 5)[1:] for l in log() if l.startswith("launch")]
"""


@pytest.fixture(scope="module")
def fake(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not installed")
    so = str(tmp_path_factory.mktemp("fake") / "libfakehip.so")
    subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", "-Wall",
                    os.path.join(ROOT, "tests", "c", "fake_hip.cpp"), "-o", so], check=True)

    def run(body):
        r = subprocess.run([sys.executable, "-c", PRELUDE + textwrap.dedent(body), so], cwd=ROOT, text=True,
                           stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=120)
        assert r.returncode == 0, r.stdout

    return run


def test_launches_of_a_product(fake):
    fake("""
    # one launch where rows are read in place or quantized by the product's kernel, else two
    assert mm(1, 2560, 2560, L.T_F16) == 0
    (k,) = kernels()
    assert "int8_stream_kernel" in k[4], k
    assert mm(4, 2560, 4096, L.T_F32) == 0 and len(kernels()) == 1
    for M, K in ((5, 128), (4, 4100), (1, 16400)):
        assert mm(M, 2560, K, L.T_BF16) == 0
        q, k = kernels()
        assert "rows8" in q[4] and "int8_stream_kernel" in k[4], (q, k)
    assert mm(7, 100, 96) == 0 and len(kernels()) == 1
    assert mm(7, 100, 96, stride=112) == 0 and len(kernels()) == 1
    assert mm(7, 100, 96, stride=100) == 0
    q, k = kernels()
    assert "rows8_copy_kernel" in q[4]
    assert mm(64, 100, 96) == 0 and "int8_stream_kernel" in kernels()[0][4]
    assert mm(65, 100, 96) == 0 and "int8_gemm_kernel" in kernels()[0][4]
    assert mm(0, 100, 96) == 0 and not kernels()
    """)


def test_every_tile_is_some_calls(fake):
    """Each of the eight tiles is taken by the sizes that test_int8_gpu.py runs
    for it; grids and LDS fit the GPU."""
    from tests.int8_ref import TILES
    fake(f"""
    seen = set()
    for tile, sizes in {TILES!r}.items():
        for M, N, K in sizes:
            assert mm(M, N, K, L.T_I8, L.T_I32) == 0, lib.ter_hip_last_error()
            dev, blocks, threads, lds, name = kernels()[-1]
            cfg = name[name.index("GCfg<") + 5:name.index(">")].split(", ")
            mbw, sw, rw, cw = map(int, cfg[:4])
            assert f"{{16 * mbw * rw}}x{{16 * sw * cw}}" == tile, (tile, M, N, K, name)
            tiles = -(-M // (16 * mbw * rw)) * -(-N // (16 * sw * cw))
            assert int(blocks) == min(tiles, 512 if tile == "64x64" else 256) * int(threads) or \\
                int(blocks) == min(tiles, 512 if tile == "64x64" else 256), (blocks, tiles)
            assert int(threads) == 64 * rw * cw and int(lds) <= 160 * 1024
        seen.add(tile)
    assert len(seen) == 8
    """)


def test_parts_of_a_long_k(fake):
    """Few tiles of a long K: by parts that have units each and fit the GPU at
    once, joined by one more launch; their sums in the workspace."""
    from tests.int8_ref import PARTS
    fake(f"""
    for M, N, K in {PARTS!r}:
        assert mm(M, N, K, L.T_I8, L.T_BF16) == 0, lib.ter_hip_last_error()
        *_, p, j = kernels()
        assert "int8_gemm_kernel" in p[4] and "true>" in p[4] and "join" in j[4], (p, j)
        tiles = -(-M // 64) * -(-N // 64)
        parts, rest = divmod(int(p[1]), tiles)
        units = -(-K // 128)
        assert rest == 0 and 2 <= parts <= 8 and int(p[1]) <= 512, p
        assert -(-units // parts) * (parts - 1) < units
        assert int(j[1]) * 256 * 8 >= M * N
        w = L.W8()
        assert lib.ter_hip_w8_init(C.byref(w), A, 1 << 60, K, N) == 0
        x = L.Rows(A, A, K, L.T_I8, M)
        rows = 0 if K % 16 == 0 else -(-M * (units * 128 + 4) // 16) * 16
        assert lib.ter_hip_w8_mm_ws(C.byref(w), C.byref(x)) == rows + parts * M * -(-N // 8) * 32
    assert mm(380, 512, 1024) == 0 and len(kernels()) == 1
    fake.fake_fail(b"int8_join")
    assert mm(380, 512, 8192) == L.ERR_HIP
    """)


def test_rows_of_many_launches(fake):
    """Rows quantized: no launch of 2^32 threads or more."""
    fake("""
    for M, K, launches in ((1 << 21, 8000, 1), ((1 << 21) + 1, 5000, 2), (1 << 23, 16384, 4), (1 << 23, 600, 4),
                           (1 << 23, 16385, 1)):
        assert mm(M, 64, K, L.T_BF16) == 0, lib.ter_hip_last_error()
        k = [x for x in kernels() if "rows8" in x[4]]
        assert len(k) == launches and sum(int(x[1]) for x in k) == M, k
        assert all(int(x[1]) * int(x[2]) < 1 << 32 for x in k), k
    """)


def test_a_failed_launch_is_an_error(fake):
    fake("""
    for part, call in ((b"int8_stream", lambda: mm(3, 100, 96)), (b"int8_gemm", lambda: mm(300, 100, 96)),
                       (b"rows8_quant", lambda: mm(30, 100, 96, L.T_F16)), (b"rows8_copy", lambda: mm(30, 100, 95))):
        fake.fake_fail(part)
        assert call() == L.ERR_HIP, part
        assert lib.ter_hip_last_error()
        fake.fake_fail(b"")
        assert call() == 0
    for part in (b"sample_max", b"sample_bins", b"sample_list", b"sample_finish"):
        fake.fake_fail(part)
        assert draw(2, 50000) == L.ERR_HIP
        fake.fake_fail(b"")
    fake.fake_fail(b"sample_rows")
    assert draw(400, 50000) == L.ERR_HIP
    """)


def test_launches_of_a_draw(fake):
    fake("""
    # a row by slices where rows are few, by one workgroup where they are many or short
    for rows, V, slices in ((1, 128256, 32), (1, 1 << 19, 64), (64, 128256, 8), (256, 128256, 2), (257, 128256, 1),
                            (1, 4096, 1), (1, 4097, 2), (100000, 1000, 1)):
        assert draw(rows, V) == 0, lib.ter_hip_last_error()
        k = kernels()
        need = lib.ter_hip_sample_ws(rows, V)
        if slices == 1:
            assert len(k) == 1 and "sample_rows_kernel" in k[0][4] and int(k[0][1]) == rows and need == 0, k
        else:
            assert [x[4].split("sample_")[1].split("_")[0] for x in k] == ["max", "bins", "list", "finish"], k
            assert [int(x[1]) for x in k] == [rows * slices] * 3 + [rows], k
            assert need % rows == 0 and need > 0
    """)


def test_launches_that_take_the_largest(fake):
    fake("""
    # temperature 0 or top_k 1 on the host: a row's slices and their join; read on the device: the usual way
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_k=1, dev=A)):
        assert draw(2, 128256, **kw) == 0
        a, b = kernels()
        assert "sample_largest_kernel" in a[4] and int(a[1]) == 64 and "largest_join" in b[4] and int(b[1]) == 2, (a, b)
        assert draw(300, 128256, **kw) == 0
        (a,) = kernels()
        assert "sample_largest_kernel" in a[4] and int(a[1]) == 300, a
    assert draw(2, 128256, temperature=0.0, dev=A) == 0 and len(kernels()) == 4
    for part in (b"sample_largest_kernel", b"largest_join"):
        fake.fake_fail(part)
        assert draw(2, 50000, temperature=0.0) == L.ERR_HIP
        fake.fake_fail(b"")
    """)


def test_wait_states_around_the_asm_loads(tmp_path):
    """The loads to LDS of the product in tiles are inline asm: no buffer load
    within five wait states of the lane read that wrote one of its registers."""
    from tests import test_paged_waits as waits
    code = waits.kernels(tmp_path, "int8_gemm_kernel")
    assert len(code) >= 32
    for name, kernel in code.items():
        assert not kernel.faults(), name
