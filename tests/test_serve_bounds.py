"""CPU checks of the operators around a served batch's step: every bad argument is refused before anything is launched; groups of sequences
(csrc/ti_span.h, compiled here for the host) against a plain search, whatever the numbers on the device are; and the adapters' bound sees a lost
piece of an activation."""
import ctypes as C
import os
import shutil
import subprocess

import numpy as np
import pytest

import serve_ref as ref
from tabinfer_amd import abi

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P, Q, R = 0x10000, 0x100000000, 0x200000000           # addresses that a refused call does not touch
IMAX = 2 ** 31 - 1
NAN, INF = float("nan"), float("inf")

# name -> (arguments that are fine, [(index, value) or several, ...] that are not)
PREP = [P, P, P, P, P, Q, P, P, P, P, P, P, P, P, 4, 2, 4, 2, 64, 16, 10, 5, 0, 0, 1e6, 1e-6]
SHARED = [P, P, P, P, P, P, P, P, P, P + 64, 4, 2, 4, 2, 64, 16, 10, 5]
LORA = [P, P, P, P, P, Q, 3, 64, 40, 8, 2, 0, 0, 1]
LP = [P, P, P, P, P, P, P, 3, 100, 0, 5]
REFUSED = {
    "ti_attn_prep_paged_q8": (PREP, [{i: None} for i in (0, 1, 2, 5, 6, 7, 8, 9, 12)] + [{0: P + 4}, {1: P + 8}, {2: P + 4}, {3: P + 2}, {4: P + 4}, {5: Q + 8}, {6: P + 4}, {8: P + 8},
                              {5: P + 16}, {5: P, 22: 512}, {1: Q}, {2: Q + 2032}, {14: 0}, {14: -1}, {15: 0}, {16: -1}, {16: 65}, {17: 0}, {17: 65}, {18: 0}, {18: 48}, {18: 160}, {19: 0}, {19: 12}, {20: 0},
                              {21: 0}, {11: None, 14: 5, 15: 4}, {22: 255}, {22: 252}, {22: -4}, {23: 130}, {23: 124}, {24: 0.5}, {24: 0.0}, {24: -1.0}, {24: NAN}, {24: INF},
                              {14: 2 ** 24, 15: 2 ** 24}, {19: 2 ** 20, 21: 2 ** 11}]),
    "ti_attn_shared_q8": (SHARED, [{i: None} for i in range(10)] + [{9: P}, {1: P + 8}, {3: P + 4}, {10: 0}, {10: 2049}, {11: 0}, {11: -1}, {11: 5}, {12: 3}, {12: 65, 13: 65}, {13: 0},
                          {14: 40}, {14: 160}, {15: 0}, {15: 12}, {16: 0}, {17: 0}, {17: 2 ** 27 + 1}, {10: 2048, 11: 2048, 12: 64, 13: 64}, {10: 2048, 11: 1, 12: 64, 13: 8}]),
    "ti_lora_add": (LORA, [{i: None} for i in range(6)] + [{0: P + 4}, {2: P + 8}, {3: P + 2}, {5: P}, {5: P + 64}, {6: 0}, {6: -1}, {7: 0}, {7: 40}, {8: 0}, {9: 0}, {9: 129}, {10: 0},
                    {11: 60}, {11: 66}, {11: -64}, {12: 39}, {13: 2}, {13: -1}, {6: 2 ** 18 + 1, 5: Q * 64}]),
    "ti_logprobs": (LP, [{i: None} for i in (0, 1, 2, 5, 6)] + [{7: 0}, {7: -1}, {7: 2 ** 17 + 1}, {8: 0}, {8: -5}, {8: IMAX}, {9: 99}, {9: -1}, {10: -1}, {10: 65}, {8: 4, 10: 5}]),
}


@pytest.mark.parametrize("name", sorted(REFUSED))
def test_bad_arguments_are_refused(name):
    good, bad = REFUSED[name]
    fn = getattr(abi.lib(), name)
    assert len(good) + 1 == len(abi.SIGS[name])
    ctx = C.addressof(C.create_string_buffer(1 << 16))
    assert fn(None, *good) == abi.TI_ERR_INVALID and b"null context" in abi.lib().ti_last_error()
    for change in bad:
        args = list(good)
        for i, v in change.items():
            args[i] = v
        assert fn(ctx, *args) == abi.TI_ERR_INVALID, change
        assert name.encode() in abi.lib().ti_last_error(), change


SRC = r"""
#include "ti_span.h"
extern "C" int group_of(const int32_t* starts, const int32_t* shared, int P, int B, int b) { return ti_group_of(starts, shared, P, B, b).g; }
extern "C" int base(const int32_t* starts, const int32_t* shared, int P, int B, int b) { return ti_group_of(starts, shared, P, B, b).shared; }
extern "C" int first(const int32_t* starts, int B, int g) { return ti_group_members(starts, B, g).first; }
extern "C" int count(const int32_t* starts, int B, int g) { return ti_group_members(starts, B, g).count; }
extern "C" int parts(long total, int nb, int tiles, int wgs, int many, int BW) { return ti_group_parts(total, nb, tiles, wgs, many, BW); }
extern "C" int number(int first, int g, int tile, int G, int rows) { return ti_group_tile(first, g, tile, G, rows); }
"""


@pytest.fixture(scope="module")
def host(tmp_path_factory):
    cxx = shutil.which("g++")
    if cxx is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("groups")
    (d / "s.cc").write_text(SRC)
    subprocess.check_call([cxx, "-std=c++17", "-shared", "-fPIC", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                           "-I", os.path.join(ROOT, "tabinfer_amd", "csrc"), str(d / "s.cc"), "-o", str(d / "s.so")])
    return C.CDLL(str(d / "s.so"))


def test_groups_against_a_plain_search(host):
    rng = np.random.default_rng(1)
    ptr = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    for _ in range(300):
        B, P = int(rng.integers(1, 40)), int(rng.integers(1, 12))
        starts = np.sort(rng.integers(0, B + 1, P + 1)).astype(np.int32)
        shared = rng.choice(np.array([0, -3, 1, 50, IMAX], np.int32), P)
        G, rows = int(rng.choice([1, 2, 5, 16, 64])), 16
        numbers = []
        for g in range(P):
            n = int(starts[g + 1] - starts[g])
            assert host.count(ptr(starts), B, g) == (n if n > 1 else 0)
            if n > 1:
                assert host.first(ptr(starts), B, g) == starts[g]
                numbers += [host.number(int(starts[g]), g, t, G, rows) for t in range((n * G + rows - 1) // rows)]
        # one number for each tile, rising, below what the scratch is laid out for
        assert all(a < b for a, b in zip(numbers, numbers[1:])) and all(0 <= v < host.number(B, P, 0, G, rows) for v in numbers)
        for b in range(B):
            of = [g for g in range(P) if starts[g] <= b < starts[g + 1] and starts[g + 1] - starts[g] > 1 and shared[g] > 0]
            assert host.group_of(ptr(starts), ptr(shared), P, B, b) == (of[0] if of else -1)
            assert host.base(ptr(starts), ptr(shared), P, B, b) == (shared[of[0]] if of else 0)


def test_groups_of_any_numbers_stay_inside(host):
    """starts that fall, lie below zero or behind the last sequence: members, groups and tiles are still of the batch."""
    rng = np.random.default_rng(2)
    ptr = lambda a: a.ctypes.data_as(C.c_void_p)  # noqa: E731
    for _ in range(300):
        B, P, G = int(rng.integers(1, 40)), int(rng.integers(1, 12)), int(rng.choice([1, 3, 16]))
        starts = rng.choice(np.array([-2 ** 31, -1, 0, 1, 2, 5, 20, 39, 40, IMAX], np.int32), P + 1)
        shared = rng.choice(np.array([-1, 1, IMAX], np.int32), P)
        for g in range(P):
            f, n = host.first(ptr(starts), B, g), host.count(ptr(starts), B, g)
            assert 0 <= f <= B and 0 <= n <= B - f
            if n:
                assert 0 <= host.number(f, g, (n * G + 15) // 16 - 1, G, 16) <= host.number(B, P, 0, G, 16)
        for b in range(B):
            g = host.group_of(ptr(starts), ptr(shared), P, B, b)
            assert -1 <= g < P
            if g >= 0:
                f, n = host.first(ptr(starts), B, g), host.count(ptr(starts), B, g)
                assert f <= b < f + n


@pytest.mark.parametrize("K", [64, 512, 2048])
def test_the_adapters_bound_sees_a_lost_piece(K):
    """An activation cut to one f16, or to two bf16 in place of three, is outside the 2-norm that the tests allow."""
    rng = np.random.default_rng(K)
    r, N = 8, 64
    x, y = rng.standard_normal((1, K)), np.zeros((1, N))
    a, b = rng.standard_normal((1, r, K)) * K ** -0.5, 0.05 * rng.standard_normal((1, N, r))
    want, norm, _ = ref.lora(x, y, [0], a, b, np.ones(1))

    def cut(v, bits):
        m, e = np.frexp(v)
        return np.ldexp(np.trunc(np.ldexp(m, bits)), e - bits)
    for bits in (11, 16):
        got, _, _ = ref.lora(cut(x, bits), y, [0], a, b, np.ones(1))
        assert np.linalg.norm(got - want) > norm, bits
    got, _, _ = ref.lora(x.astype(np.float32).astype(np.float64), y, [0], a, b, np.ones(1))
    assert np.linalg.norm(got - want) < norm


def test_runs_of_groups_fit_their_slots(host):
    """Every tile has a run, none more than blocks; all of them have no more than the slots that a call keeps: many, and one a tile."""
    rng = np.random.default_rng(6)
    host.parts.argtypes = [C.c_long] + [C.c_int] * 5
    most = 0.0
    for _ in range(20000):
        units = int(rng.integers(1, 12))
        nb, tiles = np.rint(2.0 ** rng.uniform(0, 22 if rng.random() < 0.1 else 9, units)).astype(int), np.rint(2.0 ** rng.uniform(0, rng.integers(1, 6), units)).astype(int)
        many = int(np.rint(2.0 ** rng.uniform(0, 10)))
        wgs, BW = (many + 1) // 2, 4
        if rng.random() < 0.2:                             # sequences' own keys: always one tile
            wgs, tiles, BW = many, np.ones_like(tiles), int(rng.choice([1, 2, 4]))
        total = int((nb * tiles).sum())
        n = [host.parts(total, int(b), int(t), wgs, many, BW) for b, t in zip(nb, tiles)]
        assert all(1 <= p <= b for p, b in zip(n, nb))
        runs = sum(p * int(t) for p, t in zip(n, tiles))
        assert runs <= many + tiles.sum()
        most = max(most, runs / (many + tiles.sum()))
    assert most > 0.9
