"""Rows of Q, K and V of any sequences: norm, rotation, and K and V into pages (attnPrepQ8, models/qwen3.js:2297-2308, for many rows), against
64 bits (tests/serve_ref.py derives the tolerances), the format's codes, and ti_attn_prep_q8."""
import numpy as np
import pytest

import serve_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
FILL, GUARD = 0xA5A5A5A5, np.float32(-7.25)
THETA, EPS = 1e6, 1e-6


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
    """K codes, K scales, V codes, V scales as [rows][nKv][..]."""
    kinds = ((np.int8, hd), (np.float32, hd // 32)) * 2
    return [ctx.download(b, t, rows * nKv * n).reshape(rows, nKv, n) for b, (t, n) in zip(bufs, kinds)]


def places(rng, T, B, width, page, pages):
    """A table with holes, rows' sequences and positions with bad ones among them, and the rows of the pool: -1 for none, none twice."""
    table = rng.choice(np.concatenate([rng.permutation(pages)[:B * width], np.full(max(1, B * width // 8), -1), [pages, 2 ** 31 - 1]]), (B, width)).astype(np.int32)
    seq, pos = rng.integers(-1, B + 1, T).astype(np.int32), rng.integers(-2, width * page + 3, T).astype(np.int32)
    row, taken = np.full(T, -1, np.int64), set()
    for t in range(T):
        if 0 <= seq[t] < B and 0 <= pos[t] < width * page and 0 <= table[seq[t], pos[t] // page] < pages:
            at = int(table[seq[t], pos[t] // page]) * page + int(pos[t]) % page
            if at in taken:
                pos[t] = -1
            else:
                taken.add(at)
                row[t] = at
    return table, seq, pos, row


def check_cache(got, row, k32, v):
    """The rows written are the codes of k32 and v, the others were left alone. A K code may be the neighbour's where its quotient
    is next to the border: an angle's last bit may turn a cosine's rounding, 8 U of a quotient times 127 < 1e-4."""
    untouched = np.ones(len(got[0]), bool)
    untouched[row[row >= 0]] = False
    for codes, scales in (got[:2], got[2:]):
        assert np.all(codes[untouched].view(np.uint8) == 0xA5) and np.all(scales[untouched].view(np.uint32) == FILL)
    live = row >= 0
    for x, codes, scales, exact in ((k32, got[0], got[1], False), (v, got[2], got[3], True)):
        want, top, far = ref.codes(x[live])
        off = codes[row[live]].astype(int) - want
        if exact:
            assert np.array_equal(scales[row[live]], top) and not off.any()
        else:
            assert np.all(np.abs(scales[row[live]] - top) <= 4 * ref.U * top)
            assert np.all((off == 0) | ((np.abs(off) == 1) & (far < 1e-4)))
            assert np.count_nonzero(off) <= 1e-3 * off.size


# T, B, nHq, nKv, hd, page, pages, width
SHAPES = [(1, 1, 16, 8, 128, 16, 3, 2), (1, 1, 1, 1, 32, 1, 2, 1), (7, 3, 32, 8, 64, 16, 20, 4), (50, 50, 16, 8, 128, 4, 130, 2), (33, 2, 6, 2, 96, 8, 30, 12),
          (300, 1, 20, 5, 32, 64, 9, 6), (129, 4, 5, 5, 96, 32, 40, 9), (64, 7, 64, 1, 64, 1, 900, 100), (20, 2, 0, 8, 128, 16, 9, 3), (17, 2, 40, 8, 128, 2, 70, 20)]


@pytest.mark.parametrize("merged", [False, True])
@pytest.mark.parametrize("T,B,nHq,nKv,hd,page,pages,width", SHAPES)
def test_rows(ctx, T, B, nHq, nKv, hd, page, pages, width, merged):
    rng = np.random.default_rng(T + hd + merged)
    table, seq, pos, row = places(rng, T, B, width, page, pages)
    nq, nkv, extra = nHq * hd, nKv * hd, 12 if merged else 0
    qkv = (rng.standard_normal((T, nq + 2 * nkv + extra)) * 10.0 ** rng.uniform(-2, 2, (T, 1))).astype(np.float32)
    q, k, v = qkv[:, :nq].reshape(T, nHq, hd), qkv[:, nq:nq + nkv].reshape(T, nKv, hd), qkv[:, nq + nkv:nq + 2 * nkv].reshape(T, nKv, hd)
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2))
    rot = rng.integers(-50, 40000, T).astype(np.int32) if merged else None
    cache = new_pool(ctx, pages * page, nKv, hd)
    bufs = [ctx.upload(a) for a in (qw, kw, table, seq, pos)]
    drot = ctx.upload(rot) if merged else None
    out = ctx.upload(np.concatenate([np.full(T * nq, np.nan, np.float32), np.full(64, GUARD)]).astype(np.float32))
    if merged:
        x = ctx.upload(qkv)
        src, ld = (x.at(0) if nHq else None, x.at(4 * nq), x.at(4 * (nq + nkv))), qkv.shape[1]
        own = [x]
    else:
        own = [ctx.upload(np.ascontiguousarray(a)) for a in (q, k, v)]
        src, ld = (own[0] if nHq else None, own[1], own[2]), 0
    ctx.call("ti_attn_prep_paged_q8", *src, bufs[0], bufs[1], out if nHq else None, *cache, bufs[2], bufs[3], bufs[4], drot, T, B, nHq, nKv, hd, page, pages,
             width, ld, ld, THETA, EPS)
    got = ctx.download(out, np.float32, T * nq + 64)
    assert np.all(got[T * nq:] == GUARD)
    at = pos if rot is None else rot
    want, tol = ref.turn(q, qw, at, THETA, EPS)
    assert np.all(np.abs(got[:T * nq].reshape(q.shape) - want) <= tol)
    check_cache(pool_rows(ctx, cache, pages * page, nKv, hd), row, ref.turn32(k, kw, at, THETA, EPS), v)
    for b in own + bufs + cache + [out] + ([drot] if drot else []):
        b.free()


@pytest.mark.parametrize("nHq,nKv,hd", [(16, 8, 128), (32, 8, 64), (4, 4, 32)])
def test_as_the_single_token_call(ctx, nHq, nKv, hd):
    """Codes, scales and queries of ti_attn_prep_q8, bit for bit, on a contiguous cache (no table), queries in place."""
    rng = np.random.default_rng(hd)
    T, cap = 6, 900
    pos = np.array([0, 1, 2, 57, 300, 899], np.int32)
    q, k, v = (rng.standard_normal((T, n, hd)).astype(np.float32) for n in (nHq, nKv, nKv))
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2))
    dq, dk, dv, dqw, dkw, dp = [ctx.upload(a) for a in (q, k, v, qw, kw, pos)]
    a, b, qr = new_pool(ctx, cap, nKv, hd), new_pool(ctx, cap, nKv, hd), ctx.zeros(q.nbytes)
    for t in range(T):
        ctx.call("ti_attn_prep_q8", dq.at(t * q[0].nbytes), dk.at(t * k[0].nbytes), dv.at(t * v[0].nbytes), dqw, dkw, qr.at(t * q[0].nbytes), *a, nHq, nKv, hd,
                 int(pos[t]), THETA, EPS)
    ctx.call("ti_attn_prep_paged_q8", dq, dk, dv, dqw, dkw, dq, *b, None, None, dp, None, T, 1, nHq, nKv, hd, 1, cap, 0, 0, 0, THETA, EPS)
    assert np.array_equal(ctx.download(qr, np.uint32, q.size), ctx.download(dq, np.uint32, q.size))
    for x, y in zip(a, b):
        assert np.array_equal(ctx.download(x, np.uint32, x.nbytes // 4), ctx.download(y, np.uint32, y.nbytes // 4))
    for x in a + b + [dq, dk, dv, dqw, dkw, dp, qr]:
        x.free()


@pytest.mark.parametrize("hd", [32, 64, 96, 128])
def test_far_positions_and_no_norms(ctx, hd):
    """Rotations up to the end of 32 bits and below zero, without norm weights: angles of 64 bits, off by 2^-52 of themselves."""
    rng = np.random.default_rng(hd)
    rot = np.array([0, 1, -1, 12345, 10 ** 6, -10 ** 6, 2 ** 27, 2 ** 31 - 1, -2 ** 31, 77777777], np.int32)
    T, nHq, nKv = len(rot), 4, 2
    q, k, v = (rng.standard_normal((T, n, hd)).astype(np.float32) for n in (nHq, nKv, nKv))
    bufs = [ctx.upload(a) for a in (q, k, v, np.arange(T, dtype=np.int32), rot)]
    cache, out = new_pool(ctx, T, nKv, hd), ctx.zeros(q.nbytes)
    back = [ctx.zeros(k.nbytes) for _ in range(2)]
    ctx.call("ti_attn_prep_paged_q8", *bufs[:3], None, None, out, *cache, None, None, bufs[3], bufs[4], T, 1, nHq, nKv, hd, 1, T, 0, 0, 0, 1e4, EPS)
    ctx.call("ti_kv_read_paged_q8", *cache, None, None, bufs[3], *back, T, 1, nKv, hd, 1, T, 0)
    slack = 2.0 ** -52 * np.abs(rot.astype(np.float64))[:, None, None]            # of an angle, and so of a cosine
    want, tol = ref.turn(q, None, rot, 1e4, EPS)
    half = np.abs(q[..., :hd // 2]) + np.abs(q[..., hd // 2:])
    assert np.all(np.abs(ctx.download(out, np.float32, q.size).reshape(q.shape) - want) <= tol + slack * np.concatenate([half, half], -1))
    want, tol = ref.turn(k, None, rot, 1e4, EPS)
    got = ctx.download(back[0], np.float32, k.size).reshape(k.shape)
    step = np.abs(want.reshape(T, nKv, hd // 32, 32)).max(-1, keepdims=True).repeat(32, -1).reshape(k.shape) / 127
    assert np.all(np.abs(got - want) <= 0.5001 * step + 2e-6)
    for b in bufs + cache + back + [out]:
        b.free()


def test_zeros_and_values_that_are_not_finite(ctx):
    """A row of zeros, with and without a norm, is one of zeros; one head's NaN or infinity stays with its head."""
    T, nHq, nKv, hd = 3, 2, 2, 64
    rng = np.random.default_rng(3)
    q, k, v = (rng.standard_normal((T, n, hd)).astype(np.float32) for n in (nHq, nKv, nKv))
    q[0, 0], k[0, 0], v[0, 0] = 0, 0, 0
    q[1, 1, 5], k[1, 1, 6], v[1, 1, 7] = np.nan, np.inf, np.nan
    w = np.ones(hd, np.float16)
    pos = np.arange(T, dtype=np.int32)
    bufs = [ctx.upload(a) for a in (q, k, v, w, pos)]
    cache, out = new_pool(ctx, T, nKv, hd), ctx.zeros(q.nbytes)
    ctx.call("ti_attn_prep_paged_q8", *bufs[:3], bufs[3], bufs[3], out, *cache, None, None, bufs[4], None, T, 1, nHq, nKv, hd, 1, T, 0, 0, 0, THETA, EPS)
    got = ctx.download(out, np.float32, q.size).reshape(q.shape)
    fine = np.ones((T, nHq), bool)
    fine[1, 1] = False
    want, tol = ref.turn(np.nan_to_num(q), w, pos, THETA, EPS)
    assert np.all(np.abs(got - want)[fine] <= tol[fine]) and not got[0, 0].any() and np.isnan(got[1, 1]).any()
    kc, ks, vc, vs = pool_rows(ctx, cache, T, nKv, hd)
    assert not kc[0, 0].any() and np.all(ks[0, 0] == np.float32(1e-12)) and not vc[0, 0].any()
    want, top, _ = ref.codes(v)
    assert np.array_equal(vc[fine], want[fine]) and np.array_equal(vs[fine], top[fine])
    for b in bufs + cache + [out]:
        b.free()


def test_captured_rows_follow_their_positions(ctx):
    """One captured call replayed with other rows, places and rotations between, and the program's own calls."""
    rng = np.random.default_rng(5)
    T, B, nHq, nKv, hd, page, pages, width = 9, 3, 16, 8, 128, 4, 40, 12
    w = (1 + 0.2 * rng.standard_normal(hd)).astype(np.float16)
    dq, dk, dv = ctx.zeros(T * nHq * hd * 4), ctx.zeros(T * nKv * hd * 4), ctx.zeros(T * nKv * hd * 4)
    dw, dt, ds, dp, dr = ctx.upload(w), ctx.zeros(B * width * 4), ctx.zeros(T * 4), ctx.zeros(T * 4), ctx.zeros(T * 4)
    out, cache, twin = ctx.zeros(T * nHq * hd * 4), new_pool(ctx, pages * page, nKv, hd), new_pool(ctx, pages * page, nKv, hd)
    call = lambda c: ctx.call("ti_attn_prep_paged_q8", dq, dk, dv, dw, dw, out, *c, dt, ds, dp, dr, T, B, nHq, nKv, hd, page, pages, width, 0, 0, THETA, EPS)  # noqa: E731
    ctx.graph_begin()
    call(cache)
    g = ctx.graph_end()
    for _ in range(4):
        table, seq, pos, row = places(rng, T, B, width, page, pages)
        rot = rng.integers(0, 9000, T).astype(np.int32)
        q, k, v = (rng.standard_normal((T, n, hd)).astype(np.float32) for n in (nHq, nKv, nKv))
        for d, a in ((dq, q), (dk, k), (dv, v), (dt, table), (ds, seq), (dp, pos), (dr, rot)):
            ctx.write(d, a)
        for b in cache + twin:
            ctx.fill_u32(b, FILL, b.nbytes // 4)
        ctx.graph_launch(g)
        got = ctx.download(out, np.float32, q.size).reshape(q.shape)
        call(twin)
        assert np.array_equal(got.ravel(), ctx.download(out, np.float32, q.size))
        want, tol = ref.turn(q, w, rot, THETA, EPS)
        assert np.all(np.abs(got - want) <= tol)
        rows = pool_rows(ctx, cache, pages * page, nKv, hd)
        check_cache(rows, row, ref.turn32(k, w, rot, THETA, EPS), v)
        assert all(np.array_equal(x.view(np.uint8), y.view(np.uint8)) for x, y in zip(rows, pool_rows(ctx, twin, pages * page, nKv, hd)))
    ctx.graph_destroy(g)
    for b in [dq, dk, dv, dw, dt, ds, dp, dr, out] + cache + twin:
        b.free()
