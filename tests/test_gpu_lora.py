"""Low-rank adapters of many requests beside a projection, against 64 bits (tests/serve_ref.py derives the tolerances)."""
import numpy as np
import pytest

import serve_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
GUARD = np.float32(-7.25)


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def weights(rng, shape, std, bf16):
    """(bit patterns, their values in 64 bits)."""
    x = (rng.standard_normal(shape) * std).astype(np.float32)
    if not bf16:
        h = x.astype(np.float16)
        return h.view(np.uint16), h.astype(np.float64)
    b = (x.view(np.uint32) >> 16).astype(np.uint16)
    return b, (b.astype(np.uint32) << 16).view(np.float32).astype(np.float64)


def requests(rng, T, n, turns):
    """`turns` requests behind each other, some with no adapter."""
    which = rng.integers(-1, n, turns)
    which[rng.integers(turns)] = rng.integers(n)
    return which[np.arange(T) * turns // T].astype(np.int32)


def run(ctx, x, y, idx, a, b, scale, N, bf16, ldx=0, ldy=0):
    T, (n, r, K) = len(idx), a.shape
    bufs = [ctx.upload(v) for v in (x, idx, a, b, scale)]
    out = ctx.upload(np.concatenate([y.ravel(), np.full(64, GUARD)]).astype(np.float32))
    ctx.call("ti_lora_add", *bufs, out, T, K, N, r, n, ldx, ldy, int(bf16))
    got = ctx.download(out, np.float32, y.size + 64)
    for v in bufs + [out]:
        v.free()
    assert np.all(got[y.size:] == GUARD)
    return got[:y.size].reshape(y.shape)


# T, K, N, r, n, turns
SHAPES = [(1, 32, 1, 1, 1, 1), (1, 2048, 2048, 16, 8, 1), (2, 64, 17, 8, 3, 2), (5, 96, 100, 7, 4, 5), (16, 2048, 512, 32, 40, 16), (17, 160, 31, 13, 2, 3), (48, 1024, 4096, 32, 16, 48),
          (33, 6144, 200, 64, 5, 4), (100, 224, 63, 128, 3, 7), (64, 512, 130, 100, 9, 64), (257, 2048, 300, 16, 6, 4), (700, 320, 65, 40, 8, 9), (1500, 1024, 257, 64, 6, 4), (2100, 96, 48, 9, 300, 2100)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,K,N,r,n,turns", SHAPES)
def test_adapters(ctx, T, K, N, r, n, turns, bf16):
    rng = np.random.default_rng(T + K + r)
    x = (rng.standard_normal((T, K)) * 10.0 ** rng.uniform(-3, 3, (T, 1))).astype(np.float32)
    y = rng.standard_normal((T, N)).astype(np.float32)
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale = rng.uniform(-2, 2, n).astype(np.float32)
    idx = requests(rng, T, n, turns)
    got = run(ctx, x, y, idx, a, b, scale, N, bf16)
    want, norm, tol = ref.lora(x.astype(np.float64), y.astype(np.float64), idx, a64, b64, scale.astype(np.float64))
    assert np.all(np.abs(got - want) <= tol)
    # row by row, as the rows' sizes differ
    some = rng.permutation(T)[:8]
    for t in some:
        _, norm, _ = ref.lora(x[t:t + 1].astype(np.float64), y[t:t + 1].astype(np.float64), idx[t:t + 1], a64, b64, scale.astype(np.float64))
        assert np.linalg.norm(got[t] - want[t]) <= norm + 1e-30
    none = idx < 0
    assert np.array_equal(got[none], y[none])


def test_rows_apart_and_unaligned_outputs(ctx):
    """Parts of wider rows: x a stretch of 4's, y any; what lies between is left alone. Indices out of range name no adapter."""
    rng = np.random.default_rng(2)
    T, K, N, r, n, ldx, ldy = 40, 256, 75, 16, 4, 300, 101
    for bf16 in (False, True):
        x, y = rng.standard_normal((T, ldx)).astype(np.float32), rng.standard_normal((T, ldy)).astype(np.float32)
        (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
        scale = rng.uniform(0.5, 2, n).astype(np.float32)
        idx = rng.choice(np.array([0, 1, 2, 3, 4, -1, 2 ** 31 - 1, -2 ** 31], np.int32), T)
        bufs = [ctx.upload(v) for v in (x, idx, a, b, scale, y)]
        ctx.call("ti_lora_add", bufs[0].at(16), bufs[1], bufs[2], bufs[3], bufs[4], bufs[5].at(20), T, K, N, r, n, ldx, ldy, int(bf16))
        got = ctx.download(bufs[5], np.float32, y.size).reshape(y.shape)
        for v in bufs:
            v.free()
        want, norm, tol = ref.lora(x[:, 4:4 + K].astype(np.float64), y[:, 5:5 + N].astype(np.float64), idx, a64, b64, scale.astype(np.float64))
        assert np.all(np.abs(got[:, 5:5 + N] - want) <= tol) and np.linalg.norm(got[:, 5:5 + N] - want) <= norm
        assert np.array_equal(got[:, :5], y[:, :5]) and np.array_equal(got[:, 5 + N:], y[:, 5 + N:])
        gone = (idx < 0) | (idx >= n)
        assert np.array_equal(got[gone], y[gone])


@pytest.mark.parametrize("bf16", [False, True])
def test_what_is_not_finite_stays_with_its_row(ctx, bf16):
    """NaN rows beside fine ones of the same tile and adapter; an adapter of NaN beside others; rows without an adapter hold anything."""
    rng = np.random.default_rng(3)
    T, K, N, r, n = 20, 512, 64, 24, 5
    x, y = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale = np.ones(n, np.float32)
    idx = (np.arange(T) % 4).astype(np.int32)
    idx[5] = -1
    want, _, tol = ref.lora(x.astype(np.float64), y.astype(np.float64), idx, a64, b64, scale.astype(np.float64))
    x[2, 100], x[5], x[7, 3] = np.nan, np.nan, np.inf
    a[4] = 0x7FFF                                          # nobody's adapter
    a[3, 0, 0] = 0x7FFF
    got = run(ctx, x, y, idx, a, b, scale, N, bf16)
    bad = np.isin(np.arange(T), [2, 7]) | (idx == 3)
    assert np.all(np.abs(got - want)[~bad] <= tol[~bad]) and not np.isfinite(got[bad]).any()


@pytest.mark.parametrize("bf16", [False, True])
def test_activations_of_any_size(ctx, bf16):
    """Rows far above and below f16's range, and rows of both: an element counts to 2^-39 of its row's largest."""
    rng = np.random.default_rng(4)
    T, K, N, r, n = 6, 384, 33, 16, 1
    x = rng.standard_normal((T, K)).astype(np.float32)
    x[0] *= np.float32(1e30)
    x[1] *= np.float32(1e-30)
    x[2, ::2] *= np.float32(1e7)
    x[3] = 0
    y = np.zeros((T, N), np.float32)
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale, idx = np.ones(1, np.float32), np.zeros(T, np.int32)
    got = run(ctx, x, y, idx, a, b, scale, N, bf16)
    for t in range(T):
        want, norm, _ = ref.lora(x[t:t + 1].astype(np.float64), y[t:t + 1].astype(np.float64), idx[t:t + 1], a64, b64, scale.astype(np.float64))
        assert np.linalg.norm(got[t] - want[0]) <= norm
    # subnormal weights count too
    s, s64 = (np.arange(1, r * K + 1, dtype=np.uint16) % 200).reshape(1, r, K), None
    s64 = s.view(np.float16).astype(np.float64) if not bf16 else (s.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
    if not bf16:
        got = run(ctx, x[4:], y[4:], idx[4:], s, b, scale, N, bf16)
        want, norm, tol = ref.lora(x[4:].astype(np.float64), y[4:].astype(np.float64), idx[4:], s64, b64, scale.astype(np.float64))
        assert np.linalg.norm(got - want) <= norm


def test_repeats_and_replays_bit_for_bit(ctx):
    """A captured call follows rows and indices from replay to replay; the same inputs give the same bits."""
    rng = np.random.default_rng(6)
    T, K, N, r, n = 50, 2048, 300, 32, 6
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, True), weights(rng, (n, N, r), 0.05, True)
    scale = rng.uniform(0.5, 2, n).astype(np.float32)
    da, db, ds = (ctx.upload(v) for v in (a, b, scale))
    dx, di, y1, y2 = ctx.zeros(T * K * 4), ctx.zeros(T * 4), ctx.zeros(T * N * 4), ctx.zeros(T * N * 4)
    call = lambda y: ctx.call("ti_lora_add", dx, di, da, db, ds, y, T, K, N, r, n, 0, 0, 1)  # noqa: E731
    ctx.graph_begin()
    call(y1)
    g = ctx.graph_end()
    for _ in range(4):
        x, y, idx = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32), rng.integers(-1, n, T).astype(np.int32)
        for d, v in ((dx, x), (di, idx), (y1, y), (y2, y)):
            ctx.write(d, v)
        ctx.graph_launch(g)
        call(y2)
        got = ctx.download(y1, np.float32, y.size).reshape(y.shape)
        want, norm, _ = ref.lora(x.astype(np.float64), y.astype(np.float64), idx, a64, b64, scale.astype(np.float64))
        assert np.array_equal(got.ravel(), ctx.download(y2, np.float32, y.size)) and np.linalg.norm(got - want) <= norm
    ctx.graph_destroy(g)
    for v in (da, db, ds, dx, di, y1, y2):
        v.free()
