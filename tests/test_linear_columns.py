"""The output head's tile widths, compiled for the host."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
MOST = 0x7fffffff - 1024  # rows of a call


@pytest.fixture(scope="module")
def columns(tmp_path_factory):
    from born_b200 import build
    if shutil.which("g++") is None:
        pytest.skip("no host compiler")
    where = tmp_path_factory.mktemp("columns")
    src, out = where / "columns.cc", where / "columns.so"
    src.write_text('#include "%s"\nextern "C" void columns(int rows, int most, int* out) { born::linear_columns(rows, most, out[0], out[1]); }\n'
                   % os.path.join(ROOT, "born_b200", "csrc", "linear_launch.cuh"))
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.realpath(build.nvcc_path()))), "include")
    subprocess.check_call(["g++", "-std=c++17", "-fwrapv", "-fPIC", "-shared", "-I", include, "-o", str(out), str(src)])
    lib = C.CDLL(str(out))

    def call(rows, most):
        r = (C.c_int * 2)()
        lib.columns(rows, most, r)
        return r[0], r[1]
    return call


@pytest.mark.parametrize("most", [64, 128, 256])
def test_tiles_hold_the_rows(columns, most):
    """Equal tiles of at most `most` columns, none of them empty, up to the most rows that a call takes."""
    for rows in [1, 2, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 256, 257, 300, 511, 512, 513, 1000, 65536, 10 ** 9,
                 2_110_000_000, 2_114_000_000, 2_139_000_000, 2_140_000_000, MOST - 1, MOST]:
        cols, tiles = columns(rows, most)
        assert 16 <= cols <= most and cols % (16 if rows <= 16 else 32) == 0, rows
        assert (tiles - 1) * cols < rows <= tiles * cols, rows
        assert tiles <= (rows + most - 1) // most, rows
