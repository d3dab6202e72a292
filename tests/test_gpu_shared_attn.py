"""Attention of one token of each of B sequences in groups that share their first positions, against softmax attention in 64 bits
(tests/span_ref.py derives the tolerances)."""
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


def group_of(b, starts, shared):
    for g in range(len(shared)):
        if starts[g] <= b < starts[g + 1]:
            return g if starts[g + 1] - starts[g] > 1 and shared[g] > 0 else -1
    return -1


def make(rng, starts, shared, lens, page, width=None):
    """A table whose shared places are a group's first sequence's; the others' entries there, and all behind a sequence's end, are bad ids."""
    B = len(lens)
    width = width or max(1, max([(max(n, 0) + page - 1) // page for n in lens] + [(max(s, 0) + page - 1) // page for s in shared]))
    owner = np.zeros((B, width), bool)
    for b in range(B):
        g = group_of(b, starts, shared)
        base = shared[g] if g >= 0 else 0
        for k in range(width):
            first = k * page
            owner[b, k] = first < lens[b] and first + page > base
            if g >= 0 and b == starts[g] and first < base:
                owner[b, k] = True
    pages = int(owner.sum()) + 3
    table = rng.choice(np.array([-1, pages, 2 ** 31 - 1, -2 ** 31], np.int32), (B, width))
    table[owner] = rng.permutation(pages)[:owner.sum()]
    return table, pages, width


def expected(q, kc, ks, vc, vs, table, pages, page, starts, shared, lens):
    want, tol = np.zeros(q.shape), np.zeros(q.shape)
    used = np.zeros(len(kc), bool)
    for b, n in enumerate(lens):
        n = min(n, table.shape[1] * page)
        if n <= 0:
            continue
        j = np.arange(n)
        g = group_of(b, starts, shared)
        row = np.where(j < (shared[g] if g >= 0 else 0), starts[g] if g >= 0 else b, b)
        ids = table[row, j // page].astype(np.int64)
        ok = (ids >= 0) & (ids < pages)
        rows = np.where(ok, ids, 0) * page + j % page
        used[rows[ok]] = True
        o, t, _, _ = ref.attend(q[b:b + 1], ref.values(kc[rows], ks[rows]), ref.values(vc[rows], vs[rows]), ok[None])
        want[b], tol[b] = o[0], t[0]
    return want, tol, used


def run(ctx, q, kc, ks, vc, vs, table, pages, page, starts, shared, lens):
    (B, nHq, hd), nKv = q.shape, kc.shape[1]
    bufs = [ctx.upload(a) for a in (q, kc, ks, vc, vs, table, np.asarray(lens, np.int32), np.asarray(starts, np.int32), np.asarray(shared, np.int32))]
    out = ctx.upload(np.concatenate([np.full(q.size, np.nan), np.full(64, GUARD)]).astype(np.float32))
    ctx.call("ti_attn_shared_q8", *bufs, out, B, len(shared), nHq, nKv, hd, page, pages, table.shape[1])
    got = ctx.download(out, np.float32, q.size + 64)
    for b in bufs + [out]:
        b.free()
    assert np.all(got[q.size:] == GUARD)
    return got[:q.size].reshape(q.shape)


def check(ctx, rng, starts, shared, lens, page, nHq, nKv, hd, wide=True):
    table, pages, _ = make(rng, starts, shared, lens, page)
    q = (rng.standard_normal((len(lens), nHq, hd)) * rng.choice([0.3, 2.0], (len(lens), nHq, 1))).astype(np.float32)
    kc, ks, vc, vs = ref.cache(rng, pages * page, nKv, hd, wide=wide)
    want, tol, used = expected(q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
    ks[~used], vs[~used] = np.nan, np.inf                # what nobody sees does not matter
    got = run(ctx, q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
    assert np.all(np.abs(got - want) <= tol)
    return got


# starts, shared, lens, page, nHq, nKv, hd
CASES = [
    ([0, 2], [5], [6, 9], 4, 1, 1, 32), ([0, 2], [32], [33, 64], 16, 4, 2, 128), ([0, 3], [1], [2, 3, 4], 1, 6, 2, 96),
    ([0, 4], [1000], [1077, 1001, 1033, 1600], 16, 16, 8, 128),
    # groups that begin late, end early, are empty, hold one sequence, share nothing
    ([1, 3, 3, 4, 7], [40, 9, 30, 64], [50, 41, 90, 31, 65, 64, 200, 33], 8, 32, 8, 64), ([0, 2, 4], [0, 70], [3, 5, 71, 80], 16, 4, 4, 64),
    ([3, 3], [9], [5, 6, 7, 8], 2, 8, 8, 128), ([0, 1, 2, 3], [5, 6, 7], [9, 9, 9], 4, 2, 1, 128),
    # sequences as long as what is shared, shorter, and of nothing
    ([0, 5], [100], [100, 60, 0, -3, 101], 32, 16, 8, 128), ([0, 3], [31], [0, 0, 0], 16, 4, 2, 64), ([0, 2], [64], [32, 33], 32, 5, 5, 32),
    # row tiles: many query heads a KV head, many sequences
    ([0, 3], [77], [90, 80, 200], 16, 64, 1, 128), ([0, 2], [300], [301, 333], 64, 40, 8, 96), ([0, 40], [500], [501 + 3 * i for i in range(40)], 64, 16, 8, 128),
    ([0, 33, 66], [250, 31], [260 + i for i in range(66)], 2, 16, 1, 32), ([0, 17], [90], [91] * 17, 128, 6, 3, 64),
    # many small groups, many sequences of none
    (list(range(0, 301, 2)), [10 + i % 60 for i in range(150)], [80 + i % 7 for i in range(300)], 16, 4, 2, 64), ([100, 102], [33], [40] * 300, 8, 2, 2, 32),
    # long
    ([0, 6], [20000], [20001 + 700 * i for i in range(6)], 128, 8, 8, 64),
]


@pytest.mark.parametrize("starts,shared,lens,page,nHq,nKv,hd", CASES)
def test_groups(ctx, starts, shared, lens, page, nHq, nKv, hd):
    rng = np.random.default_rng(len(lens) + page + hd)
    got = check(ctx, rng, starts, shared, lens, page, nHq, nKv, hd)
    for b, n in enumerate(lens):
        if n <= 0:
            assert not got[b].any()


@pytest.mark.parametrize("starts,shared,lens,page,nHq,nKv,hd", [
    ([0, 96], [2080], [2081 + i % 50 for i in range(96)], 32, 32, 16, 32), ([0, 12, 24], [8200, 5000], [8201 + 7 * i for i in range(12)] + [5001] * 12, 64, 64, 16, 64)])
def test_runs_long_enough_for_two_workgroups_a_cu(ctx, starts, shared, lens, page, nHq, nKv, hd):
    rng = np.random.default_rng(hd)
    check(ctx, rng, starts, shared, lens, page, nHq, nKv, hd)


@pytest.mark.parametrize("page", [1, 16, 64])
def test_bad_pages_are_not_there(ctx, page):
    """Ids outside the pool in shared places and a sequence's own; lengths and shared lengths past the table."""
    rng = np.random.default_rng(page)
    starts, shared, lens, nHq, nKv, hd = [0, 3, 6], [200, 5000], [300, 210, 250, 4000, 100, 9999], 16, 8, 128
    table, pages, width = make(rng, starts, [200, 320], [300, 210, 250, 320, 100, 320], page, 320 // page)
    hit = rng.random(table.shape) < 0.3
    table[hit] = rng.choice(np.array([-1, pages, 2 ** 31 - 1, -2 ** 31], np.int32), int(hit.sum()))
    q = rng.standard_normal((6, nHq, hd)).astype(np.float32)
    kc, ks, vc, vs = ref.cache(rng, pages * page, nKv, hd)
    want, tol, used = expected(q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
    ks[~used], vs[~used] = np.nan, np.inf
    got = run(ctx, q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
    assert np.all(np.abs(got - want) <= tol)


def test_not_finite_rows_and_keys_stay_their_own(ctx):
    """A NaN query is its row's; a shared key of NaN is its group's; an own one its sequence's."""
    rng = np.random.default_rng(7)
    starts, shared, lens, page, nHq, nKv, hd = [0, 4, 8], [100, 70], [120, 110, 105, 130, 90, 80, 75, 71], 16, 16, 8, 128
    table, pages, _ = make(rng, starts, shared, lens, page)
    q = rng.standard_normal((8, nHq, hd)).astype(np.float32)
    kc, ks, vc, vs = ref.cache(rng, pages * page, nKv, hd)
    want, tol, _ = expected(q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
    q[2, 5] = np.nan
    ks[table[4, 10 // page] * page + 10 % page] = np.nan          # shared by the second group
    ks[table[1, 105 // page] * page + 105 % page] = np.nan        # of sequence 1
    got = run(ctx, q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
    fine = np.ones((8, nHq), bool)
    fine[2, 5], fine[1], fine[4:] = False, False, False
    assert np.all(np.abs(got - want)[fine] <= tol[fine]) and np.isnan(got[~fine]).all()


def test_as_the_ungrouped_call_and_bit_for_bit_again(ctx):
    """With tables that hold the shared pages in every row: within both tolerances of ti_attn_paged_q8; repeated, the same bits."""
    rng = np.random.default_rng(9)
    starts, shared, lens, page, nHq, nKv, hd = [0, 12], [2000], [2001 + 50 * i for i in range(12)], 16, 16, 8, 128
    table, pages, width = make(rng, starts, shared, lens, page)
    table[:, :2000 // page] = table[0, :2000 // page]
    q = rng.standard_normal((12, nHq, hd)).astype(np.float32)
    kc, ks, vc, vs = ref.cache(rng, pages * page, nKv, hd)
    _, tol, _ = expected(q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
    got = [run(ctx, q, kc, ks, vc, vs, table, pages, page, starts, shared, lens) for _ in range(3)]
    assert np.array_equal(got[0], got[1]) and np.array_equal(got[0], got[2])
    bufs = [ctx.upload(a) for a in (q, kc, ks, vc, vs, table, np.asarray(lens, np.int32))] + [ctx.zeros(q.nbytes)]
    ctx.call("ti_attn_paged_q8", *bufs, 12, nHq, nKv, hd, page, pages, width, -1, 0)
    other = ctx.download(bufs[-1], np.float32, q.size).reshape(q.shape)
    for b in bufs:
        b.free()
    assert np.all(np.abs(got[0] - other) <= 2 * tol)


def test_captured_step_follows_groups_and_lengths(ctx):
    """One captured call replayed with other groups, lengths, tables and queries between, and the program's own calls; a second
    captured call on the same context's scratch between its replays."""
    rng = np.random.default_rng(10)
    page, nHq, nKv, hd, B, P, width, pages = 8, 16, 8, 128, 6, 2, 40, 260
    kc, ks, vc, vs = ref.cache(rng, pages * page, nKv, hd)
    dev = [ctx.upload(a) for a in (kc, ks, vc, vs)]
    dq, dt, dl, dst, dsh = ctx.zeros(B * nHq * hd * 4), ctx.zeros(B * width * 4), ctx.zeros(B * 4), ctx.zeros((P + 1) * 4), ctx.zeros(P * 4)
    o, o2 = ctx.zeros(B * nHq * hd * 4), ctx.zeros(B * nHq * hd * 4)
    graphs = []
    for out in (o, o2):
        ctx.graph_begin()
        ctx.call("ti_attn_shared_q8", dq, *dev, dt, dl, dst, dsh, out, B, P, nHq, nKv, hd, page, pages, width)
        graphs.append(ctx.graph_end())
    for starts, shared, lens in [([0, 3, 6], [100, 64], [120, 101, 320, 65, 70, 90]), ([1, 6, 6], [200, 9], [5, 201, 300, 220, 0, 210]),
                                 ([0, 2, 4], [0, 33], [10, 20, 34, 33, 300, 1]), ([0, 6, 6], [310, 0], [311, 312, 313, 320, 318, 311])]:
        table = np.stack([rng.permutation(pages)[:width] for _ in range(B)]).astype(np.int32)
        q = rng.standard_normal((B, nHq, hd)).astype(np.float32)
        for d, a in ((dq, q), (dt, table), (dl, np.array(lens, np.int32)), (dst, np.array(starts, np.int32)), (dsh, np.array(shared, np.int32))):
            ctx.write(d, a)
        for g in graphs:
            ctx.graph_launch(g)
        got, again = ctx.download(o, np.float32, q.size), ctx.download(o2, np.float32, q.size)
        ctx.call("ti_attn_shared_q8", dq, *dev, dt, dl, dst, dsh, o2, B, P, nHq, nKv, hd, page, pages, width)
        want, tol, _ = expected(q, kc, ks, vc, vs, table, pages, page, starts, shared, lens)
        assert np.all(np.abs(got.reshape(q.shape) - want) <= tol)
        assert np.array_equal(got, again) and np.array_equal(got, ctx.download(o2, np.float32, q.size))
    for g in graphs:
        ctx.graph_destroy(g)
    for b in dev + [dq, dt, dl, dst, dsh, o, o2]:
        b.free()
