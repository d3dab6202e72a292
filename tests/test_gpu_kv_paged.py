"""Rows of K and V into and out of an int8 KV cache in pages: codes and scales bit for bit those of the contiguous
kvQuantWrite (models/qwen3.js:2180-2216), places that do not exist left alone, and the pages and their attention run
together as a server runs them."""
import numpy as np
import pytest

import span_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
FILL = 0xA5A5A5A5


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def new_pool(ctx, rows, nKv, hd):
    bufs = [ctx.alloc(rows * nKv * hd), ctx.alloc(rows * nKv * hd // 8), ctx.alloc(rows * nKv * hd), ctx.alloc(rows * nKv * hd // 8)]
    for b in bufs:
        ctx.fill_u32(b, FILL, b.nbytes // 4)
    return bufs


def pool_rows(ctx, bufs, rows, nKv, hd):
    """Codes and scales as words: [rows][...]."""
    return [ctx.download(b, np.uint32, b.nbytes // 4).reshape(rows, -1) for b in bufs]


@pytest.mark.parametrize("T,B,nKv,hd,page,pages,width", [(1, 1, 1, 32, 1, 1, 1), (5, 5, 2, 64, 16, 12, 3), (70, 3, 8, 128, 16, 40, 9),
                                                         (33, 2, 5, 96, 4, 30, 12), (300, 1, 1, 32, 128, 4, 3), (64, 64, 8, 128, 64, 100, 2)])
def test_write_and_read_pages(ctx, orc, T, B, nKv, hd, page, pages, width):
    rng = np.random.default_rng(T + hd)
    rows = pages * page
    table = rng.integers(-1, pages + 2, (B, width)).astype(np.int32)
    owner = {}                                          # each place once
    seq, pos = rng.integers(-1, B + 1, T).astype(np.int32), rng.integers(-2, width * page + 3, T).astype(np.int32)
    place = np.full(T, -1, np.int64)
    for t in range(T):
        if 0 <= seq[t] < B and 0 <= pos[t] < width * page:
            p = int(table[seq[t], pos[t] // page])
            if 0 <= p < pages:
                r = p * page + int(pos[t]) % page
                if r in owner:
                    pos[t] = -1
                else:
                    owner[r], place[t] = t, r
    kr, v = ((rng.standard_normal((T, nKv, hd)) * 10.0 ** rng.uniform(-3, 3, (T, nKv, 1))).astype(np.float32) for _ in range(2))
    kr[0, 0, :32] = 0.0                                 # a group of zeros
    cache = new_pool(ctx, rows, nKv, hd)
    dev = [ctx.upload(a) for a in (kr, v, table, seq, pos)]
    outs = [ctx.upload(np.full((T, nKv, hd), np.nan, np.float32)) for _ in range(2)]
    ctx.call("ti_kv_write_paged_q8", dev[0], dev[1], *cache, *dev[2:], T, B, nKv, hd, page, pages, width)
    ctx.call("ti_kv_read_paged_q8", *cache, *dev[2:], *outs, T, B, nKv, hd, page, pages, width)
    got = pool_rows(ctx, cache, rows, nKv, hd)
    back = [ctx.download(o, np.float32, T * nKv * hd).reshape(T, nKv, hd) for o in outs]
    for i, x in enumerate((kr, v)):
        codes, scales = orc.kv_quant(x.ravel())
        codes, scales = codes.reshape(T, -1), scales.reshape(T, -1)
        untouched = np.ones(rows, bool)
        for t in range(T):
            if place[t] >= 0:
                assert np.array_equal(got[2 * i][place[t]], codes[t])
                assert np.array_equal(got[2 * i + 1][place[t]].view(np.float32), scales[t])
                untouched[place[t]] = False
        assert np.all(got[2 * i][untouched] == FILL) and np.all(got[2 * i + 1][untouched] == FILL)
        # code * (scale / 127): two roundings
        want = ref.values(codes.view(np.int8).reshape(T, nKv, hd), scales.reshape(T, nKv, hd // 32)) * (place >= 0)[:, None, None]
        assert np.all(np.abs(back[i] - want) <= 2 * ref.U * np.abs(want) + 2.0 ** -149)
    for b in cache + dev + outs:
        b.free()


def test_no_table_is_the_contiguous_cache(ctx, orc):
    """table NULL: the rows of ti_kv_write_q8, at positions in any order; out of the cache: not written, read as zeros."""
    rng = np.random.default_rng(1)
    T, nKv, hd, cap = 9, 2, 64, 16
    pos = np.array([3, 0, 15, 16, -1, 7, 8, 2 ** 31 - 1, 4], np.int32)
    kr, v = (rng.standard_normal((T, nKv, hd)).astype(np.float32) for _ in range(2))
    a, b = new_pool(ctx, cap, nKv, hd), new_pool(ctx, cap, nKv, hd)
    dk, dv, dp = ctx.upload(kr), ctx.upload(v), ctx.upload(pos)
    outs = [ctx.upload(np.full((T, nKv, hd), np.nan, np.float32)) for _ in range(2)]
    ctx.call("ti_kv_write_paged_q8", dk, dv, *a, None, None, dp, T, 1, nKv, hd, 1, cap, 0)
    ctx.call("ti_kv_read_paged_q8", *a, None, None, dp, *outs, T, 1, nKv, hd, 8, 2, 0)
    row = nKv * hd * 4
    for t in range(T):
        if 0 <= pos[t] < cap:
            ctx.call("ti_kv_write_q8", dk.at(t * row), dv.at(t * row), *b, 1, nKv, hd, int(pos[t]))
    ga, gb = pool_rows(ctx, a, cap, nKv, hd), pool_rows(ctx, b, cap, nKv, hd)
    assert all(np.array_equal(x, y) for x, y in zip(ga, gb))
    back = ctx.download(outs[0], np.float32, T * nKv * hd).reshape(T, -1)
    inside = (pos >= 0) & (pos < cap)
    assert np.all(back[~inside] == 0) and np.all(np.abs(back[inside]).max(1) > 0)
    for x in a + b + outs + [dk, dv, dp]:
        x.free()


def test_a_server_of_pages(ctx):
    """Three conversations of different ages under a window: prompts written in one call, then tokens; each sequence's
    pages outside the window go back to the pool and come up again in another's table."""
    rng = np.random.default_rng(21)
    page, pages, B, nHq, nKv, hd, window, sinks, width = 8, 24, 3, 16, 8, 128, 20, 3, 16
    cache = new_pool(ctx, pages * page, nKv, hd)
    free, table = list(rng.permutation(pages)), np.full((B, width), -1, np.int32)
    hist = [np.zeros((0, 2, nKv, hd), np.float32) for _ in range(B)]
    dt = ctx.upload(table)

    def append(counts):
        seq = np.concatenate([np.full(n, b, np.int32) for b, n in enumerate(counts)])
        pos = np.concatenate([len(hist[b]) + np.arange(n) for b, n in enumerate(counts)]).astype(np.int32)
        rows = rng.standard_normal((len(seq), 2, nKv, hd)).astype(np.float32)
        for b, n in enumerate(counts):
            hist[b] = np.concatenate([hist[b], rows[seq == b]])
            for k in range(width):                       # pages taken and given back
                lo, hi = k * page, (k + 1) * page
                alive = lo < len(hist[b]) and (hi > len(hist[b]) - max(window, n + window - 1) or lo < sinks)
                if alive and table[b, k] < 0:
                    table[b, k] = free.pop()
                if not alive and table[b, k] >= 0:
                    free.insert(0, table[b, k])
                    table[b, k] = -1
        ctx.write(dt, table)
        bufs = [ctx.upload(np.ascontiguousarray(rows[:, i])) for i in range(2)] + [ctx.upload(seq), ctx.upload(pos)]
        ctx.call("ti_kv_write_paged_q8", bufs[0], bufs[1], *cache, dt, bufs[2], bufs[3], len(seq), B, nKv, hd, page, pages, width)
        ctx.sync()
        for x in bufs:
            x.free()

    append([40, 1, 13])
    for step in range(30):
        append([1, 1, 1])
        q = rng.standard_normal((B, nHq, hd)).astype(np.float32)
        lens = np.array([len(h) for h in hist], np.int32)
        dq, dl, do = ctx.upload(q), ctx.upload(lens), ctx.upload(np.full(q.size, np.nan, np.float32))
        ctx.call("ti_attn_paged_q8", dq, *cache, dt, dl, do, B, nHq, nKv, hd, page, pages, width, window, sinks)
        got = ctx.download(do, np.float32, q.size).reshape(q.shape)
        for x in (dq, dl, do):
            x.free()
        for b in range(B):
            x = hist[b].astype(np.float64).reshape(len(hist[b]), 2, nKv, hd // 32, 32)
            s = np.maximum(np.abs(x).max(-1, keepdims=True), 1e-12)
            e = (x.astype(np.float32) / s.astype(np.float32)).astype(np.float64)
            kv = (np.floor(0.5 + 127 * e) * s / 127).reshape(hist[b].shape)
            seen = ref.visible([len(hist[b]) - 1], np.arange(len(hist[b])), window, sinks)
            want, tol, _, _ = ref.attend(q[b:b + 1], kv[:, 0], kv[:, 1], seen)
            assert np.all(np.abs(got[b] - want[0]) <= tol[0]), (step, b)
    for x in cache + [dt]:
        x.free()
