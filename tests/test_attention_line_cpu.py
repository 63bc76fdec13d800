"""The line of key tiles that the CTAs of the attention over the paged cache share: where an offset on it lies, with lengths past 32 bits. The function
of the source, compiled for the host."""
import ctypes
import os
import re
import subprocess

import pytest

from conftest import ROOT

SOURCE = open(os.path.join(ROOT, "sglang_b200", "csrc", "tree_attention.cu")).read()


@pytest.fixture(scope="module")
def line_place(tmp_path_factory):
    m = re.search(r"struct LinePlace \{.*?\n\};\n.*?\n\}\n", SOURCE, re.S)
    assert m, "no line_place in the source"
    at = tmp_path_factory.mktemp("line")
    (at / "place.cpp").write_text("#include <cstdint>\n#define __host__\n#define __device__\n" + m.group(0) + """
extern "C" void place(int64_t offset, int row_tiles, int units, int* out) {
  const LinePlace p = line_place(offset, row_tiles, units);
  out[0] = p.h, out[1] = p.qt, out[2] = p.at;
}
""")
    subprocess.run(["g++", "-std=c++17", "-O2", "-shared", "-fPIC", "-o", str(at / "place.so"), str(at / "place.cpp")], check=True)
    lib = ctypes.CDLL(str(at / "place.so"))
    lib.place.argtypes = [ctypes.c_int64, ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]

    def call(offset, row_tiles, units):
        out = (ctypes.c_int * 3)()
        lib.place(offset, row_tiles, units, out)
        return tuple(out)

    return call


@pytest.mark.parametrize("row_tiles, units", [(1, 1), (1, 8), (5, 11), (1 << 18, 8199), (1 << 26, 1 << 24), (3, (1 << 24) + 7), (46341, 46341)])
def test_place_on_the_line(line_place, row_tiles, units):
    for h in (0, 1, 7):
        for qt in {0, 1 % row_tiles, row_tiles // 2, row_tiles - 1}:
            for at in {0, 1 % units, units // 2, units - 1}:
                assert line_place((h * row_tiles + qt) * units + at, row_tiles, units) == (h, qt, at)


def test_the_walk_begins_there():
    assert SOURCE.count("line_place(offset, s.row_tiles, s.units(kExtraTiles<NT>))") == 1
