"""Attention over a part of the int8 KV cache: under a sliding window with sinks, over pages, and with the keys' weights
added up, against softmax attention in 64 bits (tests/span_ref.py derives the tolerances)."""
import numpy as np
import pytest

import span_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
GUARD = np.float32(-7.25)


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


class Bufs:
    """Uploads that are freed together."""

    def __init__(self, ctx):
        self.ctx, self.all = ctx, []

    def up(self, a):
        self.all.append(self.ctx.upload(a))
        return self.all[-1]

    def out(self, n):
        """n floats of NaN and a guard behind them."""
        return self.up(np.concatenate([np.full(n, np.nan, np.float32), np.full(64, GUARD, np.float32)]))

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        for b in self.all:
            b.free()


def get(ctx, b, n, shape):
    a = ctx.download(b, np.float32, n + 64)
    assert np.all(a[n:] == GUARD)
    return a[:n].reshape(shape)


def queries(rng, T, nHq, hd):
    return (rng.standard_normal((T, nHq, hd)) * rng.choice([0.3, 2.0], (T, nHq, 1))).astype(np.float32)


# T, pos0, nHq, nKv, hd, window, sinks
WINDOWS = [
    (1, 0, 1, 1, 32, -1, 0), (1, 0, 2, 2, 64, 1, 0), (1, 31, 4, 2, 128, 32, 0), (1, 32, 4, 2, 128, 32, 1), (1, 300, 40, 8, 96, 17, 3),
    (1, 4095, 16, 8, 128, 1024, 4), (1, 2500, 16, 1, 32, 2000, 64), (1, 900, 20, 1, 128, 500, 7), (1, 700, 64, 2, 64, 4096, 5),
    (1, 6000, 16, 8, 128, -1, 0), (1, 9, 2, 1, 64, 0, 4), (1, 20000, 8, 8, 128, 15000, 100),
    (2, 0, 16, 8, 128, 1, 1), (3, 1000, 32, 2, 64, 100, 100), (5, 70, 6, 2, 96, 33, 2), (7, 0, 4, 4, 32, 3, 1), (8, 4000, 16, 8, 128, 512, 4),
    (16, 15, 1, 1, 128, 16, 0), (17, 100, 3, 3, 64, -1, 9), (33, 0, 2, 2, 128, 8, 0), (40, 10, 4, 2, 64, 0, 3), (65, 130, 5, 5, 64, 1, 0),
    (64, 3000, 16, 8, 128, 2048, 0), (100, 50, 6, 2, 96, 31, 40), (130, 17, 8, 4, 32, 200, 16), (257, 0, 4, 2, 128, 64, 4),
    (300, 5, 20, 1, 32, 77, 1), (513, 1000, 4, 1, 128, 300, 65), (1025, 0, 2, 1, 64, 1000, 130), (700, 64, 4, 4, 96, -1, 0),
]


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("T,pos0,nHq,nKv,hd,window,sinks", WINDOWS)
def test_window_attention(ctx, T, pos0, nHq, nKv, hd, window, sinks, wide):
    rng = np.random.default_rng(T + 3 * pos0 + hd)
    S = pos0 + T
    q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd, wide)
    with Bufs(ctx) as b:
        o = b.out(q.size)
        ctx.call("ti_attn_window_q8", *[b.up(a) for a in (q, kc, ks, vc, vs)], o, T, pos0, nHq, nKv, hd, window, sinks)
        got = get(ctx, o, q.size, q.shape)
    seen = ref.visible(pos0 + np.arange(T), np.arange(S), window, sinks)
    want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), seen)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("T,pos0,hd", [(1, 200, 128), (1, 77, 32), (6, 100, 64), (70, 333, 128), (150, 40, 96)])
def test_window_of_nothing_gives_zeros(ctx, T, pos0, hd):
    rng = np.random.default_rng(T)
    q, (kc, ks, vc, vs) = queries(rng, T, 4, hd), ref.cache(rng, pos0 + T, 2, hd)
    with Bufs(ctx) as b:
        o = b.out(q.size)
        ctx.call("ti_attn_window_q8", *[b.up(a) for a in (q, kc, ks, vc, vs)], o, T, pos0, 4, 2, hd, 0, 0)
        assert np.all(get(ctx, o, q.size, q.shape) == 0.0)


# scales of keys that a query does not see are NaN or infinite: behind the window, between sinks and window, in the
# future of all queries but the last
@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("T,pos0,nHq,nKv,hd,window,sinks", [(1, 500, 16, 8, 128, 100, 5), (1, 90, 20, 1, 64, 31, 0), (4, 300, 4, 2, 128, 64, 33),
                                                            (70, 200, 4, 2, 128, 40, 3), (40, 100, 4, 2, 96, 50, 0), (300, 7, 2, 1, 64, 99, 1)])
def test_masked_keys_do_not_count(ctx, T, pos0, nHq, nKv, hd, window, sinks, bad):
    rng = np.random.default_rng(T + hd)
    S = pos0 + T
    q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
    seen = ref.visible(pos0 + np.arange(T), np.arange(S), window, sinks)
    never = ~seen.any(0)
    assert never.any() or T > 1
    kb, vb = ks.copy(), vs.copy()
    kb[never], vb[never] = bad, bad
    if T > 1:                                      # the last key: only the last query sees it
        kb[-1], vb[-1] = bad, bad
    with Bufs(ctx) as b:
        o = b.out(q.size)
        ctx.call("ti_attn_window_q8", *[b.up(a) for a in (q, kc, kb, vc, vb)], o, T, pos0, nHq, nKv, hd, window, sinks)
        got = get(ctx, o, q.size, q.shape)
    want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), seen)
    n = T if T == 1 else T - 1
    assert np.all(np.abs(got - want)[:n] <= tol[:n])
    if T > 1:
        assert np.all(np.isnan(got[-1]))


# query elements far above the f16 range and far below it, a V scale next to f32's largest
@pytest.mark.parametrize("T", [1, 5, 90])
def test_query_and_scale_ranges(ctx, T):
    rng = np.random.default_rng(T)
    pos0, nHq, nKv, hd = 150, 4, 2, 128
    S = pos0 + T
    q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
    q[:, 0] *= np.float32(1e7)
    q[:, 1] *= np.float32(1e-7)
    q[:, 2] *= np.float32(1e30)
    ks[:, 0] *= np.float32(1e-7)
    ks[:, 1] *= np.float32(1e-30)
    vs[:, 1] = np.float32(1e36)
    with Bufs(ctx) as b:
        o = b.out(q.size)
        ctx.call("ti_attn_window_q8", *[b.up(a) for a in (q, kc, ks, vc, vs)], o, T, pos0, nHq, nKv, hd, 100, 3)
        got = get(ctx, o, q.size, q.shape)
    seen = ref.visible(pos0 + np.arange(T), np.arange(S), 100, 3)
    want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), seen)
    assert np.all(np.abs(got - want) <= tol)


def test_window_covers_causal_attention(ctx):
    """Without a window, and with one that reaches every key, the causal attention's outputs within both tolerances."""
    rng = np.random.default_rng(4)
    for T, pos0, nHq, nKv, hd in [(1, 1000, 16, 8, 128), (40, 500, 16, 8, 128)]:
        S = pos0 + T
        q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
        _, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), ref.visible(pos0 + np.arange(T), np.arange(S), -1, 0))
        with Bufs(ctx) as b:
            dev = [b.up(a) for a in (q, kc, ks, vc, vs)]
            outs = [b.out(q.size) for _ in range(4)]
            ctx.call("ti_attn_causal_q8", *dev, outs[0], T, pos0, nHq, nKv, hd)
            for o, (w, s) in zip(outs[1:], [(-1, 0), (S, 0), (2 ** 31 - 1, 2 ** 31 - 1)]):
                ctx.call("ti_attn_window_q8", *dev, o, T, pos0, nHq, nKv, hd, w, s)
            got = [get(ctx, o, q.size, q.shape) for o in outs]
        assert np.all(np.abs(got[1] - got[0]) <= 2 * tol)
        assert np.array_equal(got[1], got[2]) and np.array_equal(got[1], got[3])


def test_unaligned_queries_and_outputs(ctx):
    rng = np.random.default_rng(11)
    for T, pos0 in [(1, 60), (3, 100), (50, 20)]:
        nHq, nKv, hd = 4, 2, 64
        S = pos0 + T
        q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
        with Bufs(ctx) as b:
            dq, do = b.up(np.concatenate([[np.float32(0)], q.ravel()])), b.out(q.size + 1)
            ctx.call("ti_attn_window_q8", dq.at(4), *[b.up(a) for a in (kc, ks, vc, vs)], do.at(4), T, pos0, nHq, nKv, hd, 30, 2)
            got = get(ctx, do, q.size + 1, -1)
        want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), ref.visible(pos0 + np.arange(T), np.arange(S), 30, 2))
        assert np.isnan(got[0]) and np.all(np.abs(got[1:].reshape(q.shape) - want) <= tol)


@pytest.mark.parametrize("T", [1, 20])
def test_window_far_into_a_cache_of_more_than_4_gib(ctx, T):
    """Rows past 2^32 bytes: only those that the queries see hold anything."""
    rng = np.random.default_rng(T)
    nHq, nKv, hd, pos0, window, sinks = 2, 1, 128, 34_000_000, 90, 3
    S = pos0 + T
    rows = np.concatenate([np.arange(sinks), np.arange(pos0 + 1 - window, S)])
    q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, len(rows), nKv, hd)
    with Bufs(ctx) as b:
        big = [ctx.alloc(S * hd), ctx.alloc(S * hd // 8), ctx.alloc(S * hd), ctx.alloc(S * hd // 8)]
        b.all += big
        for d, a in zip(big, (kc, ks, vc, vs)):
            row = a[0].nbytes
            ctx.write(d, a[:sinks])
            ctx.write(d, a[sinks:], int(rows[sinks]) * row)
        o = b.out(q.size)
        ctx.call("ti_attn_window_q8", b.up(q), *big, o, T, pos0, nHq, nKv, hd, window, sinks)
        got = get(ctx, o, q.size, q.shape)
    seen = ref.visible(pos0 + np.arange(T), rows, window, sinks)
    want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), seen)
    assert np.all(np.abs(got - want) <= tol)


# ---- pages ----------------------------------------------------------------------------------------
def pool(rng, lens, page, spare=3):
    """A table of pages in random order and the pool's size; entries past a sequence's end are out of the pool."""
    width = max(1, max((max(n, 0) + page - 1) // page for n in lens))
    need = [(max(n, 0) + page - 1) // page for n in lens]
    pages = sum(need) + spare
    ids = rng.permutation(pages).astype(np.int32)
    table = rng.choice(np.array([-1, pages, 2 ** 31 - 1, -2 ** 31], np.int32), (len(lens), width))
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    return table, pages, width


def paged_ref(q, kc, ks, vc, vs, table, pages, page, lens, window, sinks):
    """(out, tolerance) of each sequence's token."""
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    for b, n in enumerate(lens):
        n = min(n, table.shape[1] * page)
        if n <= 0:
            continue
        j = np.arange(n)
        ids = table[b, j // page].astype(np.int64)
        ok = (ids >= 0) & (ids < pages)
        rows = np.where(ok, ids, 0) * page + j % page
        seen = ref.visible([n - 1], j, window, sinks) & ok[None]
        o, t, _, _ = ref.attend(q[b:b + 1], ref.values(kc[rows], ks[rows]), ref.values(vc[rows], vs[rows]), seen)
        want[b], tol[b] = o[0], t[0]
    return want, tol


def run_paged(ctx, q, kc, ks, vc, vs, table, pages, page, lens, nKv, window, sinks):
    B, nHq, hd = q.shape
    with Bufs(ctx) as b:
        o = b.out(q.size)
        ctx.call("ti_attn_paged_q8", *[b.up(a) for a in (q, kc, ks, vc, vs, table, np.asarray(lens, np.int32))], o, B, nHq, nKv, hd, page,
                 pages, table.shape[1], window, sinks)
        return get(ctx, o, q.size, q.shape)


PAGED = [
    ([1], 1, 1, 1, 32, -1, 0), ([0], 16, 2, 1, 64, -1, 0), ([33], 16, 4, 2, 128, -1, 0), ([5, 0, 31, 32, 33, -4], 8, 4, 4, 96, -1, 0),
    ([1000, 1, 517], 16, 16, 8, 128, -1, 0), ([700, 64, 65, 63], 64, 32, 8, 64, 50, 3), ([90, 200], 1, 6, 2, 96, 40, 7),
    ([300, 45, 299], 2, 20, 1, 128, 100, 9), ([4000], 256, 16, 8, 128, -1, 0), ([5000, 20], 16, 16, 1, 32, 0, 40), ([77], 4096, 40, 8, 128, 30, 0),
    (list(range(1, 260, 3)), 32, 2, 1, 64, -1, 0), ([20000] + [3] * 20, 128, 8, 8, 128, -1, 0), ([129] * 40, 8, 5, 5, 32, 64, 64),
    ([1] * 300, 16, 1, 1, 32, -1, 0), ([3000, 2900], 4, 64, 2, 64, 1111, 4),
]


@pytest.mark.parametrize("lens,page,nHq,nKv,hd,window,sinks", PAGED)
def test_paged_attention(ctx, lens, page, nHq, nKv, hd, window, sinks):
    rng = np.random.default_rng(len(lens) + lens[0] + page)
    table, pages, width = pool(rng, lens, page)
    q, (kc, ks, vc, vs) = queries(rng, len(lens), nHq, hd), ref.cache(rng, pages * page, nKv, hd, wide=True)
    want, tol = paged_ref(q, kc, ks, vc, vs, table, pages, page, lens, window, sinks)
    got = run_paged(ctx, q, kc, ks, vc, vs, table, pages, page, lens, nKv, window, sinks)
    assert np.all(np.abs(got - want) <= tol)


@pytest.mark.parametrize("page", [1, 4, 32, 128])
def test_bad_pages_are_not_there(ctx, page):
    """Ids outside the pool in visible places, NaN in every row that no sequence sees, lengths past the table."""
    rng = np.random.default_rng(page)
    lens, nHq, nKv, hd, window, sinks = [400, 130, 128, 9000], 4, 2, 128, 200, 5
    table, pages, width = pool(rng, [400, 130, 128, 512], page)
    hit = rng.random(table.shape) < 0.3
    table[hit] = rng.choice(np.array([-1, pages, 2 ** 31 - 1, -2 ** 31], np.int32), int(hit.sum()))
    table[2] = -1                                       # a sequence of which nothing is there
    q, (kc, ks, vc, vs) = queries(rng, 4, nHq, hd), ref.cache(rng, pages * page, nKv, hd)
    used = np.zeros(pages * page, bool)
    for b, n in enumerate(lens):
        n = min(n, width * page)
        j = np.arange(n)
        j = j[ref.visible([n - 1], j, window, sinks)[0]]
        ids = table[b, j // page].astype(np.int64)
        ok = (ids >= 0) & (ids < pages)
        used[ids[ok] * page + j[ok] % page] = True
    ks[~used], vs[~used] = np.nan, np.inf
    want, tol = paged_ref(q, kc, ks, vc, vs, table, pages, page, lens, window, sinks)
    got = run_paged(ctx, q, kc, ks, vc, vs, table, pages, page, lens, nKv, window, sinks)
    assert np.all(np.abs(got - want) <= tol) and np.all(got[2] == 0.0)


def test_shared_pages_and_rows_of_one_sequence(ctx):
    """Two sequences with a common prefix of pages, and three tokens of one sequence as rows with its table."""
    rng = np.random.default_rng(8)
    page, nHq, nKv, hd = 16, 16, 8, 128
    table = np.array([[3, 1, 7, 2], [3, 1, 0, -1], [3, 1, 7, 2], [3, 1, 7, 2]], np.int32)
    lens = [64, 40, 63, 62]
    q, (kc, ks, vc, vs) = queries(rng, 4, nHq, hd), ref.cache(rng, 8 * page, nKv, hd)
    want, tol = paged_ref(q, kc, ks, vc, vs, table, 8, page, lens, -1, 0)
    got = run_paged(ctx, q, kc, ks, vc, vs, table, 8, page, lens, nKv, -1, 0)
    assert np.all(np.abs(got - want) <= tol)


def test_pages_past_4_gib(ctx):
    rng = np.random.default_rng(9)
    page, pages, nHq, nKv, hd = 16, 2_200_000, 2, 1, 128
    ids = np.array([0, pages - 1, 2_100_000, 5], np.int32)
    q, (kc, ks, vc, vs) = queries(rng, 1, nHq, hd), ref.cache(rng, 4 * page, nKv, hd)
    n = pages * page
    with Bufs(ctx) as b:
        big = [ctx.alloc(n * hd), ctx.alloc(n * hd // 8), ctx.alloc(n * hd), ctx.alloc(n * hd // 8)]
        b.all += big
        for d, a in zip(big, (kc, ks, vc, vs)):
            for i, p in enumerate(ids):
                ctx.write(d, a[i * page:(i + 1) * page], int(p) * page * a[0].nbytes)
        o = b.out(q.size)
        ctx.call("ti_attn_paged_q8", b.up(q), *big, b.up(ids), b.up(np.array([60], np.int32)), o, 1, nHq, nKv, hd, page, pages, 4, -1, 0)
        got = get(ctx, o, q.size, q.shape)
    j = np.arange(64)
    want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), (j < 60)[None])
    assert np.all(np.abs(got - want) <= tol)


def test_captured_paged_step_follows_lengths_and_table(ctx):
    """One captured call replayed with other lengths, pages and queries between, and the program's own work."""
    rng = np.random.default_rng(10)
    page, nHq, nKv, hd, B, width, pages = 8, 16, 8, 128, 3, 40, 130
    kc, ks, vc, vs = ref.cache(rng, pages * page, nKv, hd)
    with Bufs(ctx) as b:
        dev = [b.up(a) for a in (kc, ks, vc, vs)]
        dq, dt, dl = b.up(np.zeros((B, nHq, hd), np.float32)), b.up(np.zeros((B, width), np.int32)), b.up(np.zeros(B, np.int32))
        o, o2 = b.out(B * nHq * hd), b.out(B * nHq * hd)
        args = (B, nHq, nKv, hd, page, pages, width, -1, 0)
        ctx.graph_begin()
        ctx.call("ti_attn_paged_q8", dq, *dev, dt, dl, o, *args)
        g = ctx.graph_end()
        for lens in ([320, 1, 77], [0, 5, 300], [64, 64, 64], [318, 319, 320]):
            table = np.stack([rng.permutation(pages)[:width] for _ in range(B)]).astype(np.int32)
            q = queries(rng, B, nHq, hd)
            for d, a in ((dq, q), (dt, table), (dl, np.array(lens, np.int32))):
                ctx.write(d, a)
            ctx.graph_launch(g)
            ctx.call("ti_attn_paged_q8", dq, *dev, dt, dl, o2, *args)
            got, again = get(ctx, o, q.size, q.shape), get(ctx, o2, q.size, q.shape)
            want, tol = paged_ref(q, kc, ks, vc, vs, table, pages, page, lens, -1, 0)
            assert np.all(np.abs(got - want) <= tol) and np.array_equal(got, again)
        ctx.graph_destroy(g)


# ---- accumulated weights ----------------------------------------------------------------------------
MASS = [(1, 0, 1, 1, 32), (1, 31, 4, 2, 128), (1, 1000, 16, 8, 128), (1, 4321, 40, 8, 96), (1, 900, 20, 1, 64), (1, 9000, 8, 8, 128),
        (2, 0, 4, 4, 64), (3, 500, 16, 1, 32), (16, 100, 1, 1, 128), (17, 33, 6, 2, 96), (64, 0, 4, 2, 128), (100, 700, 16, 8, 128),
        (204, 1, 20, 1, 32), (256, 300, 16, 4, 64), (64, 2000, 64, 2, 128)]


@pytest.mark.parametrize("T,pos0,nHq,nKv,hd", MASS)
def test_mass(ctx, T, pos0, nHq, nKv, hd):
    rng = np.random.default_rng(T + pos0 + hd)
    S, G = pos0 + T, nHq // nKv
    q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
    mass = rng.uniform(0, 5, (S, nKv)).astype(np.float32)
    mass[pos0:] = np.nan                               # set by the call
    with Bufs(ctx) as b:
        o, dm = b.out(q.size), b.up(np.concatenate([mass.ravel(), np.full(64, GUARD)]).astype(np.float32))
        ctx.call("ti_attn_mass_q8", *[b.up(a) for a in (q, kc, ks, vc, vs)], o, dm, T, pos0, nHq, nKv, hd)
        got, gm = get(ctx, o, q.size, q.shape), get(ctx, dm, mass.size, mass.shape)
    seen = ref.visible(pos0 + np.arange(T), np.arange(S), -1, 0)
    want, tol, w, rel = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), seen)
    assert np.all(np.abs(got - want) <= tol)
    w = w.reshape(T, nKv, G, S)
    old = np.where(np.arange(S)[:, None] < pos0, mass, 0.0)
    add = w.sum((0, 2)).T
    # each weight by its relative error, the sum of T G of them by T G roundings, one more onto the old value
    mtol = (w * rel.reshape(T, nKv, G, 1)).sum((0, 2)).T + (T * G + 1) * ref.U * add + 2 * ref.U * np.abs(old + add)
    assert np.all(np.abs(gm - (old + add)) <= mtol)
    assert np.allclose((gm - old)[:, :].sum(0), T * G, rtol=1e-4)


def test_mass_repeats_bit_for_bit(ctx):
    rng = np.random.default_rng(2)
    for T, pos0, nHq, nKv, hd in [(1, 3000, 16, 8, 128), (90, 500, 16, 8, 128)]:
        S = pos0 + T
        q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
        with Bufs(ctx) as b:
            dev = [b.up(a) for a in (q, kc, ks, vc, vs)]
            res = []
            for _ in range(3):
                o, dm = b.out(q.size), b.out(S * nKv)
                ctx.fill_u32(dm, 0, S * nKv)
                ctx.call("ti_attn_mass_q8", *dev, o, dm, T, pos0, nHq, nKv, hd)
                res.append((get(ctx, o, q.size, -1), get(ctx, dm, S * nKv, -1)))
        assert all(np.array_equal(res[0][i], r[i]) for r in res[1:] for i in range(2))
