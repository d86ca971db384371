"""The paged attention's workspace goes by the device of its context, whichever
is current, over a HIP runtime without a device whose two devices differ."""
import os
import shutil
import subprocess
import sys
import textwrap

import pytest

from test_paged import PRELUDE, ROOT

UNLIKE = """
extern "C" {
static int g_broken = 0;
void unlike_break(int b) { g_broken = b; }
int hipDeviceGetAttribute(int* v, int, int device) {
    *v = device == 1 ? 64 : 256;  // the CU count
    return g_broken ? 1 : 0;
}
}
"""


@pytest.fixture(scope="module")
def unlike(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not installed")
    tmp = tmp_path_factory.mktemp("unlike")
    (tmp / "unlike.cpp").write_text(UNLIKE)
    sos = []
    for src in (os.path.join(ROOT, "tests", "c", "fake_hip.cpp"), str(tmp / "unlike.cpp")):
        so = str(tmp / (os.path.basename(src) + ".so"))
        subprocess.run([gxx, "-std=c++17", "-O1", "-shared", "-fPIC", src, "-o", so], check=True)
        sos.append(so)

    def run(body):
        first = "import ctypes, sys\nunlike = ctypes.CDLL(sys.argv[2], mode=ctypes.RTLD_GLOBAL)\n"
        r = subprocess.run([sys.executable, "-c", first + PRELUDE + textwrap.dedent(body), *sos], cwd=ROOT, text=True,
                           stdout=subprocess.PIPE, stderr=subprocess.STDOUT, timeout=120)
        assert r.returncode == 0, r.stdout

    return run


def test_workspace_is_that_of_the_contexts_device(unlike):
    unlike("""
    def need(n=5000):
        return lib.ter_hip_paged_attend_ws(h, C.byref(batch()), C.byref(cache()), n, 0)
    here = need()
    fake.fake_device(1)
    assert need() == here
    fake.fake_device(0)
    assert attend(h, batch(), cache(), n=5000, nb=here) == 0
    fake.fake_device(1)
    other = context()
    assert 0 < lib.ter_hip_paged_attend_ws(other, C.byref(batch()), C.byref(cache()), 5000, 0) < here
    """)


def test_device_that_cannot_be_asked(unlike):
    unlike("""
    unlike.unlike_break(1)
    assert lib.ter_hip_paged_attend_ws(h, C.byref(batch()), C.byref(cache()), 7, 0) == 0
    assert attend(h, batch(), cache()) == L.ERR_HIP and lib.ter_hip_last_error()
    assert not any(l.startswith("launch") for l in log())
    unlike.unlike_break(0)
    assert attend(h, batch(), cache()) == 0 and any(l.startswith("launch") for l in log())
    """)


def test_workspace_holds_the_ranges_that_there_can_be(unlike):
    """Two places for each: not for four times the workgroups that run at a
    time where the tables have no work for them."""
    unlike("""
    def need(n_seq, rows, cap, nh=32, nkv=8, hd=64):
        x = context(nh, nkv, hd)
        c = cache(page_stride=64 * nkv * hd, pos_stride=nkv * hd, head_stride=hd, page_size=64)
        b = batch(n_seq=n_seq, max_pages=cap // 64, pages_stride=cap // 64)
        n = lib.ter_hip_paged_attend_ws(x, C.byref(b), C.byref(c), rows, 0)
        assert attend(x, b, c, n=rows, qs=nh * hd, os=nh * hd, nb=n) == 0
        lib.ter_hip_paged_destroy(x)
        grid = [int(l.split()[2]) for l in log() if "paged_attend" in l and l.startswith("launch")]
        return n, grid[0]
    # 256 CUs, three workgroups of each: 96 single tokens of up to 4096
    # positions are 96 * 8 * (64 + 3) units at most, fewer than 96 a range
    n, grid = need(96, 96, 4096)
    assert grid == 768 and n < 2 * 768 * 128 * (64 + 2) * 4 + (1 << 20)
    # one prompt of 16384: more ranges than workgroups
    n, grid = need(1, 16384, 16384, 20, 5, 128)
    assert grid == 4 * 512
    # little work
    n, grid = need(1, 1, 64)
    assert grid < 64
    """)
