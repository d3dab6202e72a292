"""CPU check of what an eviction keeps in its scratch (csrc/ti_evict.h, which the entry point uses, compiled here for the host):
the parts lie one behind the other, each as large as the kernels index it, and what the header promises fits."""
import ctypes as C
import os
import re
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
SRC = r"""
#include "ti_evict.h"
extern "C" int scratch(int n, int kept, int nKv, long* out) {
    const TiEvictScratch s(n, kept, nKv);
    out[0] = s.room; out[1] = s.words; out[2] = s.count; out[3] = s.moves; out[4] = s.keys; out[5] = s.total;
    return s.fits();
}
extern "C" long words() { return TI_EVICT_WORDS; }
"""


@pytest.fixture(scope="module")
def scratch(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("evict")
    (d / "s.cc").write_text(SRC)
    subprocess.check_call([cxx, "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                           "-I", os.path.join(ROOT, "tabinfer_amd", "csrc"), str(d / "s.cc"), "-o", str(d / "s.so")])
    lib = C.CDLL(str(d / "s.so"))
    lib.words.restype = C.c_long

    def layout(n, kept, nKv):
        out = (C.c_long * 6)()
        return (bool(lib.scratch(n, kept, nKv, out)),) + tuple(out)
    layout.words = lib.words()
    return layout


@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 2048, 2049, 100_000, 2 ** 31 - 1])
@pytest.mark.parametrize("nKv", [1, 3, 64])
def test_parts_lie_behind_each_other(scratch, n, nKv):
    for kept in sorted({1, max(1, n // 3), max(1, n // 2), max(1, n - 1), n}):
        fits, room, words, count, moves, keys, total = scratch(n, kept, nKv)
        assert room == min(kept, n - kept) and 64 * words >= kept > 64 * (words - 1)
        assert count >= 2 * nKv * words and count % 2 == 0
        assert moves >= count + nKv and keys >= moves + 2 * nKv * room
        assert total >= keys + (nKv * n if n > 2048 else 0)
        assert fits == (total <= scratch.words)


def promised():
    text = open(os.path.join(ROOT, "include", "ti.h")).read()
    return int(re.search(r"n \* nKv <= (\d+)\.", text).group(1))


def test_what_the_header_promises_fits(scratch):
    for nKv in range(1, 65):
        n = promised() // nKv
        for kept in (1, n // 4, n // 2 - 1, n // 2, n // 2 + 1, n - n // 4, n - 1, n):
            assert scratch(n, kept, nKv)[0], (nKv, kept)
