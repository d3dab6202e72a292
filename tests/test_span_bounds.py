"""CPU checks of the operators over a part of the KV cache: every bad argument is refused before anything is launched,
and the visible keys and page look-ups (csrc/ti_span.h, compiled here for the host) against a brute-force count."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

from tabinfer_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 0x10000                                          # an address that a refused call does not touch
IMAX = 2 ** 31 - 1

# name -> (arguments that are fine, [(index, value) or several, ...] that are not)
ATTN_W = [P, P, P, P, P, P + 64, 1, 0, 4, 2, 64, 8, 0]
ATTN_P = [P, P, P, P, P, P, P, P + 64, 2, 4, 2, 64, 16, 10, 5, -1, 0]
MASS = [P, P, P, P, P, P + 64, P, 1, 0, 4, 2, 64]
WRITE = [P, P, P, P, P, P, P, P, P, 4, 2, 2, 64, 16, 10, 5]
EVICT = [P, P, P, P, P, P, P, P, 100, 10, 50, 2, 8, 200, 2, 64]
REFUSED = {
    "ti_attn_window_q8": (ATTN_W, [{i: None} for i in range(6)] + [{5: P}, {1: P + 8}, {3: P + 4}, {6: 0}, {6: -1}, {7: -1}, {6: 2, 7: IMAX - 1}, {8: 0},
                                   {9: 0}, {9: 3}, {8: -4}, {9: -2}, {8: 128, 9: 64}, {10: 0}, {10: 48}, {10: 160}, {10: -32}, {12: -1}, {6: 2 ** 22}]),
    "ti_attn_paged_q8": (ATTN_P, [{i: None} for i in range(8)] + [{7: P}, {1: P + 8}, {3: P + 4}, {8: 0}, {8: 2049}, {9: 3}, {9: 65, 10: 65}, {10: 0}, {11: 40},
                                  {12: 0}, {12: 12}, {12: -16}, {13: 0}, {13: -1}, {14: 0}, {14: 2 ** 27 + 1}, {16: -1}]),
    "ti_attn_mass_q8": (MASS, [{i: None} for i in range(7)] + [{5: P}, {1: P + 8}, {7: 0}, {7: 1025}, {8: -1}, {7: 2, 8: IMAX - 1}, {9: 3}, {10: 0}, {11: 31},
                               {11: 256}, {8: 2 ** 23}]),
    "ti_kv_write_paged_q8": (WRITE, [{i: None} for i in (0, 1, 2, 3, 4, 5, 8)] + [{0: P + 4}, {1: P + 8}, {2: P + 4}, {4: P + 8}, {9: 0}, {10: 0}, {11: 0},
                                     {12: 0}, {12: 33}, {12: 160}, {13: 0}, {13: 24}, {14: 0}, {13: 2 ** 20, 15: 2 ** 11}, {6: None, 13: 2 ** 20, 14: 2 ** 11}, {15: 0}, {7: None}, {9: 2 ** 30}]),
    "ti_kv_read_paged_q8": (WRITE, [{i: None} for i in (0, 1, 2, 3, 6, 7, 8)] + [{0: P + 4}, {2: P + 8}, {7: P + 4}, {8: P + 8}, {9: 0}, {10: 0}, {11: 0}, {12: 0},
                                    {12: 33}, {13: 3}, {14: -2}, {15: -1}, {5: None}]),
    "ti_kv_evict_q8": (EVICT, [{i: None} for i in range(8)] + [{0: P + 4}, {2: P + 8}, {8: 0}, {9: -1}, {9: 101}, {10: 0}, {11: -1}, {12: -1}, {11: 45}, {13: 89},
                               {14: 0}, {14: 65}, {15: 0}, {15: 48}, {15: 160}, {11: IMAX, 12: IMAX}]),
}


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_bad_arguments_are_refused(name):
    good, bad = REFUSED[name]
    fn = getattr(abi.lib(), name)
    assert len(good) + 1 == len(abi.SIGS[name])
    ctx = C.addressof(C.create_string_buffer(1 << 16))          # never looked into by a refused call
    assert fn(None, *good) == abi.TI_ERR_INVALID and b"null context" in abi.lib().ti_last_error()
    for change in bad:
        args = list(good)
        for i, v in change.items():
            args[i] = v
        assert fn(ctx, *args) == abi.TI_ERR_INVALID, change
        assert name.encode() in abi.lib().ti_last_error(), change


SRC = r"""
#include "ti_span.h"
extern "C" int span(int p, int window, int sinks, int* first, int* low, int* end) {
    const TiSpan s = ti_span(p, window, sinks);
    *first = s.first; *low = s.low; *end = s.end;
    return s.count();
}
extern "C" long page_row(const int32_t* table, int page, int pages, int width, int seq, int pos) {
    return TiPages{table, ti_log2(page), pages, width}.row(seq, pos);
}
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("span")
    (d / "s.cc").write_text(SRC)
    subprocess.check_call([cxx, "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                           "-I", os.path.join(ROOT, "tabinfer_amd", "csrc"), str(d / "s.cc"), "-o", str(d / "s.so")])
    lib = C.CDLL(str(d / "s.so"))
    lib.page_row.restype = C.c_long
    return lib


def test_spans_against_brute_force(host):
    f, l, e = C.c_int(), C.c_int(), C.c_int()
    for p in (0, 1, 2, 5, 30, 31):
        for window in (-5, -1, 0, 1, 2, 5, 31, 32, 100, IMAX):
            for sinks in (0, 1, 3, 30, 31, 200, IMAX):
                n = host.span(p, window, sinks, C.byref(f), C.byref(l), C.byref(e))
                seen = [j for j in range(p + 1) if window < 0 or j > p - window or j < sinks]
                got = list(range(f.value)) + list(range(l.value, e.value))
                assert got == seen and n == len(seen), (p, window, sinks)
    host.span(IMAX - 1, 7, 3, C.byref(f), C.byref(l), C.byref(e))
    assert (f.value, l.value, e.value) == (3, IMAX - 7, IMAX)


def test_page_rows_against_brute_force(host):
    rng = np.random.default_rng(0)
    for page in (1, 2, 16, 4096):
        pages, width, B = 7, 5, 3
        table = rng.choice(np.array([-2 ** 31, -1, 0, 3, 6, 7, IMAX], np.int32), (B, width))
        t = table.ctypes.data_as(C.c_void_p)
        for seq in range(B):
            for pos in (-2 ** 31, -1, 0, 1, page - 1, page, 2 * page + 1, width * page - 1, width * page, IMAX):
                want = -1
                if 0 <= pos < width * page and 0 <= table[seq, pos // page] < pages:
                    want = int(table[seq, pos // page]) * page + pos % page
                assert host.page_row(t, page, pages, width, seq, pos) == want
        for pos in (-1, 0, pages * page - 1, pages * page, IMAX):
            assert host.page_row(None, page, pages, 0, 0, pos) == (pos if 0 <= pos < pages * page else -1)
    big = np.array([2 ** 20], np.int32)               # a pool of more than 2^31 positions: the row number is 64-bit
    assert host.page_row(big.ctypes.data_as(C.c_void_p), 4096, 2 ** 21, 1, 0, 5) == 2 ** 32 + 5


@pytest.mark.parametrize("name,heads", [("ti_kv_write_paged_q8", 11), ("ti_kv_read_paged_q8", 11)])
def test_paged_rows_of_too_many_heads_are_refused(name, heads):
    ctx = C.addressof(C.create_string_buffer(1 << 16))
    for n in (65, 2 ** 27, IMAX):                       # 2^27 heads of 64: their product passes 32 bits
        args = list(WRITE)
        args[9], args[heads] = 1, n
        assert getattr(abi.lib(), name)(ctx, *args) == abi.TI_ERR_INVALID, n
        assert name.encode() in abi.lib().ti_last_error(), n


def test_blocks_loaded_into_a_waves_lds_are_fenced():
    """k_token_attn.hip: a wave's block is waited for and fenced before it is read, its reads are waited for and fenced
    before the next block's loads overwrite it."""
    src = open(os.path.join(ROOT, "tabinfer_amd", "csrc", "k_token_attn.hip")).read()
    i = src.index("for (; i < c1; i += a.BW) {")
    read, nxt = src.index("W.k[", i), src.index("load(i + a.BW, page);", i)
    assert "s_waitcnt(0x0F70)" in src[i:read] and "ti_wave_lds_fence();" in src[i:read]
    last = src.rindex("W.v[", i, nxt)
    assert "s_waitcnt(0xC07F)" in src[last:nxt] and "ti_wave_lds_fence();" in src[last:nxt]


def test_an_eviction_beyond_the_scratch_is_refused():
    """What the header promises fits (n * nKv up to 16 million, half of the slots moved) is half of a call that does not."""
    ctx = C.addressof(C.create_string_buffer(1 << 16))
    for n, nKv in ((4_200_000, 8), (525_000, 64), (33_600_000, 1)):
        args = [P] * 8 + [n, 0, n // 2, 2, 8, n, nKv, 64]
        assert abi.lib().ti_kv_evict_q8(ctx, *args) == abi.TI_ERR_INVALID
        assert b"exceed the scratch" in abi.lib().ti_last_error()
    for n, nKv in ((16_000_000, 1), (2_000_000, 8), (250_000, 64)):
        keep = n // 2
        words = 2 * nKv * ((keep + 63) // 64) + nKv + 2 * nKv * keep + nKv * n
        assert words <= 512 * 512 * 128
