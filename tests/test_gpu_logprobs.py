"""Log probabilities of given tokens, entropy, rank and the likeliest tokens of rows of logits, against 64 bits (tests/serve_ref.py derives the
tolerances)."""
import numpy as np
import pytest

import serve_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
GUARD = np.float32(-7.25)
LOW = np.float32(-3.402823466e38)


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def run(ctx, x, ids, top, ld=0, offset=0):
    """x: rows as they lie in memory; offset: floats before the first row."""
    T, N = len(ids), x.shape[1] if not ld else None
    return _run(ctx, x, ids, top, T, N, ld, offset)


def _run(ctx, x, ids, top, T, N, ld, offset):
    dx, di = ctx.upload(np.concatenate([np.zeros(offset, np.float32), x.ravel()])), ctx.upload(np.asarray(ids, np.int32))
    outs = [ctx.upload(np.full(n + 16, GUARD, np.float32)) for n in (T, T, T, T * top, T * top)]
    ctx.call("ti_logprobs", dx.at(4 * offset), di, outs[0], outs[1], outs[2], outs[3] if top else None, outs[4] if top else None, T, N, ld, top)
    r = {}
    for name, o, n, dt in zip(("lp", "ent", "rank", "top_ids", "top_lp"), outs, (T, T, T, T * top, T * top), (np.float32, np.float32, np.int32, np.int32, np.float32)):
        v = ctx.download(o, np.float32, n + 16)
        assert np.all(v[n:] == GUARD)
        r[name] = v[:n].view(dt).reshape((T, top) if name.startswith("top") else T)
    for b in [dx, di] + outs:
        b.free()
    return r


def check(got, x, ids, top):
    want, tol = ref.logprobs(x, ids, top)
    assert np.array_equal(got["rank"], want["rank"]) and np.array_equal(got["top_ids"], want["top_ids"])
    for k in ("lp", "ent", "top_lp"):
        g, w = got[k], want[k]
        assert np.array_equal(np.isnan(g), np.isnan(w)), k
        inf = np.isinf(w)
        assert np.array_equal(g[inf], w[inf].astype(np.float32)), k
        fine = np.isfinite(w)
        assert np.all(np.abs(g - np.where(fine, w, 0))[fine] <= tol[k][fine]), k


SHAPES = [(1, 1, 1), (1, 1, 0), (3, 2, 2), (1, 50, 5), (7, 63, 64 - 1), (2, 1000, 64), (5, 1024, 20), (4, 1025, 1), (1, 4096, 20), (9, 4097, 33), (1, 151936, 5), (3, 151936, 64),
          (60, 20000, 20), (1500, 300, 3), (300, 9001, 10), (2, 600000, 20), (70, 151936, 0)]


@pytest.mark.parametrize("T,N,top", SHAPES)
def test_rows(ctx, T, N, top):
    rng = np.random.default_rng(T + N + top)
    x = (2.5 * rng.standard_normal((T, N)) + 3 * rng.standard_normal((T, 1))).astype(np.float32)
    for t in range(T):
        x[t, rng.integers(0, N, 4)] += np.float32(8)
    ids = np.where(rng.random(T) < 0.5, x.argmax(1), rng.integers(0, N, T))
    check(run(ctx, x, ids, top), x, ids, top)


@pytest.mark.parametrize("top", [1, 20, 64])
def test_ties_go_to_the_lower_index(ctx, top):
    """Rows of few different values, of one value, of zeros of both signs, and ties across lanes, waves and parts."""
    rng = np.random.default_rng(top)
    N = 40000
    x = rng.integers(-2, 3, (8, N)).astype(np.float32)
    x[1] = 1.5
    x[2] = np.where(rng.random(N) < 0.5, np.float32(0.0), np.float32(-0.0))
    x[3] = -7
    x[3, rng.permutation(N)[:top // 2]] = 2
    x[4] = LOW
    x[5] = np.sort(rng.standard_normal(N)).astype(np.float32)           # every chunk better than the one before
    x[6] = x[5][::-1]
    x[7] = 0
    x[7, ::1024] = 1                                                    # one lane's
    ids = np.array([0, N - 1, 5, 7, 11, N - 1, 0, 1024])
    check(run(ctx, x, ids, top), x, ids, top)


@pytest.mark.parametrize("top", [1, 20, 64])
def test_masked_and_not_finite(ctx, top):
    """-inf and the type's lowest value as masks, rows of nothing else, NaN, +inf; too few candidates; ids that are none."""
    rng = np.random.default_rng(5)
    N = 9000
    x = rng.standard_normal((12, N)).astype(np.float32)
    x[0, rng.random(N) < 0.99] = -np.inf
    x[1] = -np.inf
    x[1, 4321] = -2                                                     # one token left
    x[2] = -np.inf                                                      # none
    x[3, rng.random(N) < 0.9] = LOW
    x[4] = LOW
    x[5, 77] = np.nan
    x[6, 88] = np.inf
    x[7] = np.nan
    x[8, :] = np.nan
    x[8, [5, 900]] = [1, 2]
    x[9, 0] = np.nan
    x[9, 1:] = -np.inf
    x[10] = -np.inf
    x[10, ::3] = LOW
    x[11] = 3.0e38
    ids = np.array([int(np.flatnonzero(np.isinf(x[0]))[0]), 4321, 5, -1, 8999, 78, 88, 0, 900, N, 3, 2 ** 31 - 1])
    with np.errstate(invalid="ignore", divide="ignore"):
        check(run(ctx, x, ids, top), x, ids, top)


def test_rows_apart_and_anywhere(ctx):
    """Rows `ld` apart that start at any float; what lies between them (NaN) does not count."""
    rng = np.random.default_rng(6)
    for T, N, ld, offset in [(5, 1000, 1001, 1), (3, 4100, 4103, 3), (40, 77, 96, 2), (2, 30000, 30001, 1)]:
        wide = np.full((T, ld), np.nan, np.float32)
        wide[:, :N] = rng.standard_normal((T, N))
        ids = rng.integers(0, N, T)
        check(_run(ctx, wide, ids, 7, T, N, ld, offset), wide[:, :N], ids, 7)


def test_outputs_that_are_left_out(ctx):
    rng = np.random.default_rng(7)
    for T, N in ((2, 50000), (600, 100)):
        x, ids = rng.standard_normal((T, N)).astype(np.float32), rng.integers(0, N, T)
        dx, di, lp = ctx.upload(x), ctx.upload(ids.astype(np.int32)), ctx.zeros(T * 4)
        ctx.call("ti_logprobs", dx, di, lp, None, None, None, None, T, N, 0, 0)
        assert np.array_equal(ctx.download(lp, np.float32, T), run(ctx, x, ids, 5)["lp"])
        for b in (dx, di, lp):
            b.free()


def test_the_token_that_argmax_takes_ranks_first(ctx):
    """Beside ti_argmax and ti_gumbel_noise on the same buffer: the greedy token has rank 1 and heads the list."""
    rng = np.random.default_rng(8)
    N = 151936
    x = (3 * rng.standard_normal(N)).astype(np.float32)
    dx, hist = ctx.upload(x), ctx.zeros(64)
    ctx.call("ti_argmax", dx, N, hist, 3)
    lp, ent, rank, ti, tl = (ctx.zeros(80) for _ in range(5))
    ctx.call("ti_logprobs", dx, hist.at(12), lp, ent, rank, ti, tl, 1, N, 0, 20)
    tok = int(ctx.download(hist, np.uint32, 4)[3])
    assert tok == int(x.argmax()) == int(ctx.download(ti, np.int32, 1)[0]) and int(ctx.download(rank, np.int32, 1)[0]) == 1
    assert ctx.download(lp, np.float32, 1)[0] == ctx.download(tl, np.float32, 1)[0]
    for b in (dx, hist, lp, ent, rank, ti, tl):
        b.free()


def test_captured_call_follows_logits_and_ids(ctx):
    rng = np.random.default_rng(9)
    T, N, top = 3, 30000, 20
    dx, di = ctx.zeros(T * N * 4), ctx.zeros(T * 4)
    outs = [ctx.zeros(4 * n) for n in (T, T, T, T * top, T * top)]
    ctx.graph_begin()
    ctx.call("ti_logprobs", dx, di, *outs, T, N, 0, top)
    g = ctx.graph_end()
    for _ in range(4):
        x, ids = (3 * rng.standard_normal((T, N))).astype(np.float32), rng.integers(-1, N, T).astype(np.int32)
        ctx.write(dx, x)
        ctx.write(di, ids)
        ctx.graph_launch(g)
        got = dict(zip(("lp", "ent", "rank", "top_ids", "top_lp"), (ctx.download(o, dt, o.nbytes // 4) for o, dt in zip(outs, (np.float32, np.float32, np.int32, np.int32, np.float32)))))
        got["top_ids"], got["top_lp"] = got["top_ids"].reshape(T, top), got["top_lp"].reshape(T, top)
        check(got, x, ids, top)
        eager = run(ctx, x, ids, top)
        assert all(np.array_equal(got[k], eager[k]) for k in got)
    ctx.graph_destroy(g)
    for b in [dx, di] + outs:
        b.free()


@pytest.mark.parametrize("T", [127, 128, 129])
def test_rows_joined_by_their_last_workgroup_or_a_second_launch(ctx, T):
    """Two calls one behind the other on the same scratch; the second's rows as if it were alone."""
    rng = np.random.default_rng(T)
    for N, top in ((9001, 5), (20000, 64)):
        x = (2.5 * rng.standard_normal((T, N))).astype(np.float32)
        ids = rng.integers(0, N, T).astype(np.int32)
        check(run(ctx, x, ids, top), x, ids, top)


@pytest.mark.parametrize("T,N,top,far", [(1, 100, 5, 9.0), (4, 5000, 0, 12.0), (3, 151936, 20, 25.0), (200, 9001, 3, 18.0), (2, 3000, 1, 40.0)])
def test_near_certainty(ctx, T, N, top, far):
    """One token has almost all of the probability: its log probability and the row's entropy keep their digits. With s the others' sum of e^d, d
    their distances: ln S = log1p(s), s off by (N / 256 + 58) U of itself and 3 U of the sum of e^d |d|; the entropy's sum of e^d |d| likewise, by d^2 more."""
    rng = np.random.default_rng(N)
    x = (2 * rng.standard_normal((T, N))).astype(np.float32)
    ids = rng.integers(0, N, T).astype(np.int32)
    x[np.arange(T), ids] = x.max(1) + np.float32(far)
    got = run(ctx, x, ids, top)
    for t in range(T):
        d = np.delete(x[t].astype(np.float64) - x[t].max().astype(np.float64), ids[t])
        e = np.exp(d)
        s, sd, sdd = e.sum(), (e * -d).sum(), (e * d * d).sum()
        lp, ent = -np.log1p(s), np.log1p(s) + sd / (1 + s)
        tl = ((N / 256 + 58) * s + 3 * sd) * ref.U + 4 * ref.U * -lp + 2.0 ** -140
        te = tl + ((N / 256 + 62) * sd + 3 * sdd) * ref.U + 4 * ref.U * ent + 2.0 ** -140
        assert got["rank"][t] == 1 and abs(got["lp"][t] - lp) <= tl and abs(got["ent"][t] - ent) <= te, (t, got["lp"][t], lp, got["ent"][t], ent)
        if top:
            assert got["top_ids"][t, 0] == ids[t] and abs(got["top_lp"][t, 0] - lp) <= tl


@pytest.mark.parametrize("top", [15, 16, 20, 64])
@pytest.mark.parametrize("kind", ["few values", "zeros", "signed zeros", "mostly masked", "lowest", "one lane's", "large behind", "not numbers"])
def test_limits_of_a_first_step(ctx, kind, top):
    """Values that tie, that are next to no other, that lie in few lanes, in the first 4096 elements and behind them."""
    rng = np.random.default_rng(top)
    for T, N in ((2, 4096), (3, 4097), (2, 30011), (300, 9001)):
        x = rng.standard_normal((T, N)).astype(np.float32)
        if kind == "few values":
            x = np.round(x)
        elif kind == "zeros":
            x = np.minimum(x, 0)
        elif kind == "signed zeros":
            x = np.where(x > 0, np.copysign(np.float32(0), rng.standard_normal((T, N)).astype(np.float32)), x)
        elif kind == "mostly masked":
            x[rng.random((T, N)) > 30 / N] = -np.inf
        elif kind == "lowest":
            x[rng.random((T, N)) > 30 / N] = LOW
        elif kind == "one lane's":
            x[:, 4 * 7:4 * 7 + 4] += 100                   # of the first wave: more than its share
            x[:, 256 + 4 * 7:256 + 4 * 7 + 4] += 100
            x[:, :1024] += 5
        elif kind == "large behind":
            x[:, N - 40:] += np.arange(40, dtype=np.float32)
        else:
            x[rng.random((T, N)) > 0.5] = np.nan
        ids = rng.integers(0, N, T).astype(np.int32)
        check(run(ctx, x, ids, top), x, ids, top)


@pytest.mark.parametrize("top", [3, 20, 40])
def test_later_chunks_whose_few_lanes_are_far_above_the_others(ctx, top):
    """Just `top` lanes of every later chunk exceed the limit, by far more than what lies between it and the others, rising or all alike."""
    rng = np.random.default_rng(top)
    T, N = 4, 60000
    x = rng.uniform(0, 1.9, (T, N)).astype(np.float32)
    for t in range(T):
        x[t, 4 * rng.permutation(1024)[:4 * 64]] = 5
        for c in range(4, N // 1024):
            x[t, c * 1024 + 4 * rng.permutation(64)[:top] + rng.integers(0, 4, top)] = 6 + 0.01 * c * (t % 2) + 0.001 * rng.integers(0, 3, top) * (t // 2)
    ids = rng.integers(0, N, T).astype(np.int32)
    check(run(ctx, x, ids, top), x, ids, top)
