"""CPU checks of where the 8-bit products read their rows.  The hardware checks a
buffer load's vector and immediate offsets against its resource's size, and not
the scalar one: a load whose way into the rows is in the scalar offset
reads past them, which no result shows, since it meets weights of zero."""
import os
import re
import shutil
import subprocess

import pytest

from tests import test_paged_waits as waits

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def walk(tmp_path_factory):
    gxx = shutil.which("g++")
    if gxx is None:
        pytest.skip("g++ not installed")
    exe = str(tmp_path_factory.mktemp("rows") / "int8_rows")
    subprocess.run([gxx, "-std=c++17", "-O2", "-Wall", os.path.join(ROOT, "tests", "c", "int8_rows.cpp"), "-o", exe],
                   check=True)

    def run(kernels):
        r = subprocess.run([exe, kernels], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=120)
        assert r.returncode == 0 and r.stdout.strip() == "ok", r.stdout

    return run


def offsets(kernel):
    """Buffer loads by their scalar offset: (without one, with one)."""
    n = [0, 0]
    for _, op, args in kernel.code:
        if op.startswith("buffer_load"):
            n[re.search(r"s\[\d+:\d+\], (\S+)", args).group(1) != "0"] += 1
    return n


def test_few_rows_are_read_within(walk):
    walk("stream")


def test_loads_of_few_rows_have_no_scalar_offset(tmp_path):
    """In the built code: of a unit's loads those of the row blocks have none, those
    of the strips of weights, which stay within by themselves, have one."""
    found = waits.kernels(tmp_path, "int8_stream_kernel")
    assert len(found) >= 48
    for name, kernel in found.items():
        blocks, strips, _, _, _, rows = map(int, re.findall(r"Li(\d+)E", name)[:6])
        without, with_one = offsets(kernel)
        assert with_one > 0, name
        # (rows of floating types come through LDS)
        assert without * strips == (with_one * blocks if rows == 3 else 0), (name, without, with_one)


def test_tiles_are_read_within(walk):
    walk("tiles")


def test_loads_of_tiles_have_no_scalar_offset(tmp_path):
    """The same of a tile's loads: 8 rows each, or half a strip of weights."""
    found = waits.kernels(tmp_path, "int8_gemm_kernel")
    assert len(found) >= 32
    for name, kernel in found.items():
        mbw, sw, rw, cw = map(int, re.findall(r"Li(\d+)E", name)[:4])
        without, with_one = offsets(kernel)
        # (weights twice: past the caches and through them; rows that the waves do not share evenly: one run more)
        waves = rw * cw
        runs, strips = 2 * mbw * rw, 2 * sw * cw
        assert with_one * waves % (2 * strips) == 0, (name, with_one)
        times = with_one * waves // (2 * strips)
        assert times > 0 and without == times * -(-runs // waves), (name, without, with_one)
