"""CPU checks of the paged-cache operators' boundary: the header, the binding
and the library agree; every refusal comes before device work; what a call
launches (over the HIP runtime without a device of tests/c/fake_hip.cpp)."""
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
FAKE = 1 << 20  # an address that nothing may follow


def test_header_binding_and_library_agree():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "ter_hip_paged.h")).read(), flags=re.S)
    names = set(re.findall(r"^[A-Za-z_][\w\s\*]*?\b(ter_hip_\w+)\s*\(", text, flags=re.M))
    assert names == {n for n, _, _ in L.PAGED_SIGNATURES}
    for n in names:
        assert hasattr(L.lib(), n)
    for macro, value in (("SEQ_MAX", L.PAGED_SEQ_MAX), ("ROWS_MAX", L.PAGED_ROWS_MAX), ("POS_MAX", L.PAGED_POS_MAX)):
        m = re.search(rf"TER_HIP_PAGED_{macro}\s+\(?([\d <]+)\)?", text)
        assert eval(m.group(1)) == value


def test_header_compiles_as_c99(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not installed")
    src = tmp_path / "t.c"
    src.write_text('#include "ter_hip_paged.h"\n'
                   'int main(void) { ter_hip_paged_t* c; return ter_hip_paged_create(&c, 0, 1, 64, 1, 1.f, 0, 0) == '
                   'TER_HIP_ERR_SHAPE ? 0 : 1; }\n')
    lib = os.path.dirname(L.LIB_PATH)
    r = subprocess.run([gcc, "-std=c99", "-Wall", "-Wextra", "-Werror", "-pedantic", "-I", os.path.join(ROOT, "include"),
                        str(src), "-L", lib, "-lter_hip", f"-Wl,-rpath,{lib}", "-o", str(tmp_path / "t")],
                       stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True)
    assert r.returncode == 0, r.stdout
    assert subprocess.run([str(tmp_path / "t")], timeout=60).returncode == 0


@pytest.mark.parametrize("args,code", [
    ((0, 1, 64, 100, 1e4, 0, 0), L.ERR_SHAPE),
    ((4, 3, 64, 100, 1e4, 0, 0), L.ERR_SHAPE),       # heads not a multiple of the KV heads
    ((129, 1, 64, 100, 1e4, 0, 0), L.ERR_SHAPE),     # more than 128 query heads on one KV head
    ((4, 2, 96, 100, 1e4, 0, 0), L.ERR_SHAPE),
    ((4, 2, 64, 0, 1e4, 0, 0), L.ERR_SHAPE),
    ((4, 2, 64, L.PAGED_POS_MAX + 1, 1e4, 0, 0), L.ERR_SHAPE),
    ((4, 2, 64, 100, 0.0, 0, 0), L.ERR_SHAPE),
    ((4, 2, 64, 100, float("nan"), 0, 0), L.ERR_SHAPE),
    ((4, 2, 64, 100, float("inf"), 0, 0), L.ERR_SHAPE),
    ((4, 2, 64, 100, 1e4, 2, 0), L.ERR_PAYLOAD),
    ((4, 2, 64, 100, 1e4, 0, 2), L.ERR_PAYLOAD),
])
def test_create_refusals(args, code):
    h = C.c_void_p(1)
    assert L.lib().ter_hip_paged_create(C.byref(h), *args) == code
    assert not h.value and L.lib().ter_hip_last_error()
    assert L.lib().ter_hip_paged_create(None, 4, 2, 64, 100, 1e4, 0, 0) == L.ERR_NULL


PRELUDE = """
import ctypes as C, sys
fake = C.CDLL(sys.argv[1], mode=C.RTLD_GLOBAL)
fake.fake_log.restype = C.c_char_p
fake.fake_fail.argtypes = [C.c_char_p]
from ter_amd import _lib as L
lib = C.CDLL(L.LIB_PATH)
for name, res, args in L.SIGNATURES + L.PAGED_SIGNATURES:
    f = getattr(lib, name)
    f.restype, f.argtypes = res, args
A = 1 << 20
def log():
    lines = fake.fake_log().decode().splitlines()
    fake.fake_reset()
    return lines
def context(nh=8, nkv=2, hd=64, dtype=0):
    h = C.c_void_p()
    assert lib.ter_hip_paged_create(C.byref(h), nh, nkv, hd, 100, 1e4, 0, dtype) == 0, lib.ter_hip_last_error()
    log()
    return h
def cache(**kw):
    c = L.PagedCache(A, A, 16 * 2 * 64, 2 * 64, 64, 10, 16)
    for k, v in kw.items(): setattr(c, k, v)
    return c
def batch(**kw):
    b = L.PagedBatch(A, A, A, 5, 5, 3)
    for k, v in kw.items(): setattr(b, k, v)
    return b
def append(h, b, c, n=7, q=A, qs=512, k=A, ks=128, v=A, vs=128, o=A, os=512):
    return lib.ter_hip_paged_append(h, C.byref(b) if b else None, C.byref(c) if c else None, n, q, qs, k, ks, v, vs, o,
                                    os, None)
def attend(h, b, c, n=7, q=A, qs=512, o=A, os=512, shared=0, scale=0.0, ws=A, nb=1 << 40):
    return lib.ter_hip_paged_attend(h, C.byref(b) if b else None, C.byref(c) if c else None, n, q, qs, o, os, shared,
                                    scale, ws, nb, None)
h = context()
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


def test_refusals(fake):
    """Each refused before anything is launched."""
    fake("""
    for call in (append, attend):
        for bad, code in (
            (dict(b=None), L.ERR_NULL), (dict(c=None), L.ERR_NULL), (dict(h=None), L.ERR_NULL),
            (dict(n=-1), L.ERR_SHAPE), (dict(n=L.PAGED_ROWS_MAX + 1), L.ERR_SHAPE),
            (dict(b=batch(n_seq=-1)), L.ERR_SHAPE), (dict(b=batch(n_seq=L.PAGED_SEQ_MAX + 1)), L.ERR_SHAPE),
            (dict(b=batch(row0=None)), L.ERR_NULL), (dict(b=batch(kv_len=None)), L.ERR_NULL),
            (dict(b=batch(pages=None)), L.ERR_NULL), (dict(b=batch(row0=A + 2)), L.ERR_ALIGN),
            (dict(b=batch(pages_stride=4)), L.ERR_SHAPE), (dict(b=batch(max_pages=-1)), L.ERR_SHAPE),
            (dict(b=batch(max_pages=70000, pages_stride=70000)), L.ERR_SHAPE),
            (dict(c=cache(k=None)), L.ERR_NULL), (dict(c=cache(v=None)), L.ERR_NULL),
            (dict(c=cache(k=A + 8)), L.ERR_ALIGN), (dict(c=cache(page_size=0)), L.ERR_SHAPE),
            (dict(c=cache(page_size=24)), L.ERR_SHAPE), (dict(c=cache(page_size=1 << 17)), L.ERR_SHAPE),
            (dict(c=cache(n_pages=0)), L.ERR_SHAPE), (dict(c=cache(pos_stride=132)), L.ERR_ALIGN),
            (dict(c=cache(pos_stride=0)), L.ERR_SHAPE), (dict(c=cache(head_stride=-64)), L.ERR_SHAPE),
            (dict(c=cache(page_stride=0)), L.ERR_SHAPE), (dict(c=cache(pos_stride=1 << 27)), L.ERR_SHAPE),
            (dict(q=None), L.ERR_NULL), (dict(q=A + 4), L.ERR_ALIGN), (dict(qs=504), L.ERR_SHAPE),
            (dict(qs=516), L.ERR_ALIGN), (dict(o=None), L.ERR_NULL), (dict(o=A + 2), L.ERR_ALIGN),
            (dict(os=0), L.ERR_SHAPE)):
            a = dict(h=h, b=batch(), c=cache())
            a.update(bad)
            assert call(**a) == code, (call, bad, lib.ter_hip_last_error())
            assert not any(l.startswith("launch") for l in log()), bad
    for bad, code in ((dict(k=None), L.ERR_NULL), (dict(ks=64), L.ERR_SHAPE), (dict(v=A + 8), L.ERR_ALIGN),
                      (dict(q=None, o=A), L.ERR_NULL)):
        assert append(h, batch(), cache(), **bad) == code, bad
    for bad, code in ((dict(shared=-1), L.ERR_SHAPE), (dict(shared=81), L.ERR_SHAPE), (dict(scale=-1.0), L.ERR_SHAPE),
                      (dict(scale=float("nan")), L.ERR_SHAPE), (dict(scale=float("inf")), L.ERR_SHAPE)):
        assert attend(h, batch(), cache(), **bad) == code, bad
    need = lib.ter_hip_paged_attend_ws(h, C.byref(batch()), C.byref(cache()), 7, 0)
    if need:
        assert attend(h, batch(), cache(), nb=need - 1) == L.ERR_SHAPE
        assert attend(h, batch(), cache(), ws=None) == L.ERR_NULL
        assert attend(h, batch(), cache(), ws=A + 8) == L.ERR_ALIGN
    assert not any(l.startswith("launch") for l in log())
    """)


def test_refusals_of_size(fake):
    """More work than units are counted in; a scale that is no number once
    multiplied by log2(e); a workspace for another call."""
    fake("""
    x = context(128, 1, 64)
    c = cache(page_stride=4096 * 64, pos_stride=64, head_stride=64, page_size=4096)
    b = batch(n_seq=1024, max_pages=256, pages_stride=256)
    kw = dict(qs=128 * 64, os=128 * 64)
    assert attend(x, b, c, n=L.PAGED_ROWS_MAX, **kw) == L.ERR_SHAPE and b"too many" in lib.ter_hip_last_error()
    assert not any(l.startswith("launch") for l in log())
    assert attend(x, b, c, n=1024, **kw) == 0
    for scale in (1e39, 2e38, -0.5):
        assert attend(h, batch(), cache(), scale=scale) == L.ERR_SHAPE
    assert attend(h, batch(), cache(), scale=1e38) == 0
    log()
    small = lib.ter_hip_paged_attend_ws(h, C.byref(batch()), C.byref(cache()), 7, 0)
    large = lib.ter_hip_paged_attend_ws(h, C.byref(batch()), C.byref(cache()), 7, 16)
    assert 0 < small < large
    assert attend(h, batch(), cache(), shared=16, nb=small) == L.ERR_SHAPE
    assert attend(h, batch(), cache(), shared=15, nb=small) == 0
    for bad in (dict(n=-1), dict(n=0), dict(n=1 << 20), dict(shared=-1)):
        a = dict(n=7, shared=0)
        a.update(bad)
        assert lib.ter_hip_paged_attend_ws(h, C.byref(batch()), C.byref(cache()), a["n"], a["shared"]) == 0
    """)


def test_launches_and_errors(fake):
    """Nothing to do launches nothing; a failed launch is reported; another
    device than the context's is refused."""
    fake("""
    assert append(h, batch(), cache()) == 0 and len([l for l in log() if l.startswith("launch")]) == 1
    assert append(h, batch(), cache(), q=None, o=None) == 0 and log()
    assert append(h, batch(), cache(), n=0) == 0 and append(h, batch(n_seq=0), cache()) == 0
    assert attend(h, batch(), cache(), n=0) == 0 and attend(h, batch(n_seq=0), cache()) == 0
    assert attend(h, batch(n_seq=0, kv_len=None, pages=None), cache()) == 0
    assert not any(l.startswith("launch") for l in log())
    assert attend(h, batch(max_pages=0, pages=None), cache()) == 0 and log()  # rows that see nothing: zeros
    fake.fake_fail(b"paged_append")
    assert append(h, batch(), cache()) == L.ERR_HIP
    fake.fake_fail(b"paged_attend")
    assert attend(h, batch(), cache()) == L.ERR_HIP
    fake.fake_fail(b"")
    log()
    fake.fake_device(1)
    assert append(h, batch(), cache()) == L.ERR_HIP and attend(h, batch(), cache()) == L.ERR_HIP
    assert b"device" in lib.ter_hip_last_error()
    assert not any(l.startswith("launch") for l in log())
    fake.fake_device(0)
    for nh, nkv, hd, dt in ((8, 2, 128, 0), (8, 2, 64, 1), (8, 2, 128, 1), (128, 1, 64, 0)):
        x = context(nh, nkv, hd, dt)
        c = cache(page_stride=16 * nkv * hd, pos_stride=nkv * hd, head_stride=hd)
        kw = dict(qs=nh * hd, os=nh * hd)
        assert append(x, batch(), c, ks=nkv * hd, vs=nkv * hd, **kw) == 0 and attend(x, batch(), c, **kw) == 0
        lib.ter_hip_paged_destroy(x)
    lib.ter_hip_paged_destroy(None)
    """)


def test_python_refuses_host_tensors():
    import torch
    import ter_amd as T
    x = torch.zeros(2, 16, 2, 64, dtype=torch.float16)
    with pytest.raises(TypeError):
        T.PagedCache(x, x)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(TypeError):
        T.PagedBatch(i, i[:2], torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(TypeError):
        T.PagedAttention(4, 2, 64, 16, 1e4, dtype=torch.float32)


def test_cutting_of_the_work(tmp_path):
    """tests/c/paged_plan.cpp: every unit of work in one range, partial results
    where the joining kernel looks for them, closed forms against counting."""
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not installed")
    exe = str(tmp_path / "paged_plan")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", os.path.join(ROOT, "tests", "c", "paged_plan.cpp"), "-o", exe],
                   check=True)
    r = subprocess.run([exe], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
    assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout
