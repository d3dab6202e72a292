"""CPU check of a paged sequence's last position (csrc/ti_span.h, compiled here for the host with its undefined arithmetic
trapped): every length is defined, those up to 0 are no keys, and the span of no keys is empty."""
import ctypes as C
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
IMAX = 2 ** 31 - 1
SRC = r"""
#include "ti_span.h"
extern "C" int last_pos(int len, long most) { return ti_last_pos(len, most); }
extern "C" int count(int p, int window, int sinks) { return ti_span(p, window, sinks).count(); }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("lengths")
    (d / "s.cc").write_text(SRC)
    subprocess.check_call([cxx, "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                           "-I", os.path.join(ROOT, "tabinfer_amd", "csrc"), str(d / "s.cc"), "-o", str(d / "s.so")])
    lib = C.CDLL(str(d / "s.so"))
    lib.last_pos.argtypes = [C.c_int, C.c_long]
    return lib


@pytest.mark.parametrize("most", [1, 7, 4096, IMAX - 255])
def test_every_length_has_a_last_position(host, most):
    for n in (-2 ** 31, -2 ** 31 + 1, -IMAX // 2, -1, 0, 1, 2, 6, 7, 8, 4095, 4096, IMAX - 256, IMAX - 1, IMAX):
        assert host.last_pos(n, most) == min(max(n, 0), most) - 1, n


def test_no_keys_are_an_empty_span(host):
    for window in (-2 ** 31, -1, 0, 1, IMAX):
        for sinks in (0, 1, IMAX):
            assert host.count(host.last_pos(-2 ** 31, 64), window, sinks) == 0
