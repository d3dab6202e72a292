"""Low-rank adapters of prompts, which the matrix cores take (T times the rank above 8192), against 64 bits: tests/test_gpu_lora.py's questions at
their sizes, and what is theirs alone. tests/serve_ref.py derives the tolerances.

f16 weights: an activation is the sum of two f16 under a power of two of the largest of its row's 32 elements from a multiple of 32 on, off by 2^-22
of itself or 2^-39 of that largest; h likewise, under its row's largest. bf16 weights: three bf16, exactly."""
import numpy as np
import pytest

import serve_ref as ref
from tabinfer_amd import abi
from test_gpu_lora import requests, run, weights

pytestmark = pytest.mark.gpu
MANY = 8192                                              # T times the rank from which on they are prompts


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def f64(*arrays):
    return [v.astype(np.float64) for v in arrays]


# T, K, N, r, n, turns: every rank's count of tiles, ranks of whole and of broken 16-byte pieces, one to four parts of K, short last stages
SHAPES = [(8200, 64, 20, 1, 3, 40), (1100, 416, 130, 8, 4, 9), (600, 1056, 257, 16, 6, 25), (500, 288, 33, 17, 3, 500), (400, 2048, 129, 24, 5, 3), (300, 4128, 300, 32, 64, 300),
          (200, 2080, 71, 50, 4, 11), (140, 1568, 40, 60, 2, 2), (100, 8192, 64, 100, 3, 8), (70, 4096, 513, 128, 9, 70), (97, 3104, 1, 96, 1, 1)]


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,K,N,r,n,turns", SHAPES)
def test_adapters(ctx, T, K, N, r, n, turns, bf16):
    assert T * r > MANY
    rng = np.random.default_rng(T + K + r)
    x = (rng.standard_normal((T, K)) * 10.0 ** rng.uniform(-3, 3, (T, 1))).astype(np.float32)
    y = rng.standard_normal((T, N)).astype(np.float32)
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale = rng.uniform(-2, 2, n).astype(np.float32)
    idx = requests(rng, T, n, turns)
    got = run(ctx, x, y, idx, a, b, scale, N, bf16)
    x64, y64, s64 = f64(x, y, scale)
    want, _, tol = ref.lora(x64, y64, idx, a64, b64, s64)
    assert np.all(np.abs(got - want) <= tol)
    for t in rng.permutation(T)[:12]:                     # row by row, as the rows' sizes differ
        _, norm, _ = ref.lora(x64[t:t + 1], y64[t:t + 1], idx[t:t + 1], a64, b64, s64)
        assert np.linalg.norm(got[t] - want[t]) <= norm + 1e-30
    none = idx < 0
    assert np.array_equal(got[none], y[none])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,K,N,r", [(560, 256, 75, 16), (150, 2080, 131, 60)])
def test_rows_apart_and_unaligned_outputs(ctx, T, K, N, r, bf16):
    """Parts of wider rows: x a stretch of 4's, y any; what lies between is left alone. Indices out of range name no adapter."""
    assert T * r > MANY
    rng = np.random.default_rng(2)
    n, ldx, ldy = 4, K + 44, N + 26
    x, y = rng.standard_normal((T, ldx)).astype(np.float32), rng.standard_normal((T, ldy)).astype(np.float32)
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale = rng.uniform(0.5, 2, n).astype(np.float32)
    idx = rng.choice(np.array([0, 1, 2, 3, 4, -1, 2 ** 31 - 1, -2 ** 31], np.int32), T)
    bufs = [ctx.upload(v) for v in (x, idx, a, b, scale, y)]
    ctx.call("ti_lora_add", bufs[0].at(16), bufs[1], bufs[2], bufs[3], bufs[4], bufs[5].at(20), T, K, N, r, n, ldx, ldy, int(bf16))
    got = ctx.download(bufs[5], np.float32, y.size).reshape(y.shape)
    for v in bufs:
        v.free()
    want, norm, tol = ref.lora(*f64(x[:, 4:4 + K], y[:, 5:5 + N]), idx, a64, b64, *f64(scale))
    assert np.all(np.abs(got[:, 5:5 + N] - want) <= tol) and np.linalg.norm(got[:, 5:5 + N] - want) <= norm
    assert np.array_equal(got[:, :5], y[:, :5]) and np.array_equal(got[:, 5 + N:], y[:, 5 + N:])
    gone = (idx < 0) | (idx >= n)
    assert np.array_equal(got[gone], y[gone])


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,K,r", [(400, 512, 24), (100, 2048, 100)])
def test_what_is_not_finite_stays_with_its_row(ctx, T, K, r, bf16):
    """NaN and infinite rows beside fine ones of the same tile and adapter; an adapter of NaN beside others; rows without an adapter hold anything, in
    x and in what an earlier call left behind."""
    assert T * r > MANY
    rng = np.random.default_rng(3)
    N, n = 64, 5
    x, y = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale = np.ones(n, np.float32)
    idx = (np.arange(T) % 4).astype(np.int32)
    idx[[5, 38, T - 1]] = -1
    run(ctx, np.full_like(x, np.nan), y, np.zeros(T, np.int32), a, b, scale, N, bf16)      # every row's h is NaN
    want, _, tol = ref.lora(*f64(x, y), idx, a64, b64, *f64(scale))
    x[2, 100], x[5], x[38], x[7, 3], x[T - 2, K - 1] = np.nan, np.nan, np.inf, np.inf, -np.inf
    a[4] = 0x7FFF                                          # nobody's adapter
    a[3, 0, 0] = 0x7FFF
    got = run(ctx, x, y, idx, a, b, scale, N, bf16)
    bad = np.isin(np.arange(T), [2, 7, T - 2]) | (idx == 3)
    assert np.all(np.abs(got - want)[~bad] <= tol[~bad]) and not np.isfinite(got[bad]).any()


@pytest.mark.parametrize("bf16", [False, True])
def test_activations_of_any_size(ctx, bf16):
    """Rows far above and below f16's range, and rows of both, each held to its own 2-norm; weights that are subnormal."""
    rng = np.random.default_rng(4)
    T, K, N, r, n = 520, 384, 33, 16, 1
    assert T * r > MANY
    x = rng.standard_normal((T, K)).astype(np.float32)
    kind = np.arange(T) % 5
    x[kind == 0] *= np.float32(1e30)
    x[kind == 1] *= np.float32(1e-30)
    x[kind == 2, ::2] *= np.float32(1e7)
    x[kind == 3] *= (10.0 ** rng.uniform(-12, 12, K)).astype(np.float32)
    x[7] = 0
    y = np.zeros((T, N), np.float32)
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale, idx = np.ones(1, np.float32), np.zeros(T, np.int32)
    got = run(ctx, x, y, idx, a, b, scale, N, bf16)
    x64, y64 = f64(x, y)
    for t in list(range(15)) + list(range(T - 15, T)):
        want, norm, _ = ref.lora(x64[t:t + 1], y64[t:t + 1], idx[t:t + 1], a64, b64, np.ones(1))
        assert np.linalg.norm(got[t] - want[0]) <= norm, (t, kind[t])
    if not bf16:
        s = (np.arange(1, r * K + 1, dtype=np.uint16) % 200).reshape(1, r, K)
        some = kind == 4
        pick = np.flatnonzero(some)
        x2 = x[np.resize(pick, T)]
        got = run(ctx, x2, y, idx, s, b, scale, N, bf16)
        want, norm, _ = ref.lora(x2.astype(np.float64), y64, idx, s.view(np.float16).astype(np.float64), b64, np.ones(1))
        assert np.linalg.norm(got - want) <= norm


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("size", [1e4, 1e7, 1e10])
def test_elements_beside_an_outlier(ctx, size, bf16):
    """Channels far above the others whose weights are zero: what is left of the elements near them. f16: sum |A| (2^-39 of the largest of the 32)
    and, h's largest being of the row, 2^-39 of it for each rank, beside the ordinary error of f32."""
    rng = np.random.default_rng(5)
    T, K, N, r, n = 600, 320, 48, 16, 2
    assert T * r > MANY
    x, y = rng.standard_normal((T, K)).astype(np.float32), np.zeros((T, N), np.float32)
    far = [5, 77, 200]
    x[:, far] *= np.float32(size)
    a32, b32 = rng.standard_normal((n, r, K)) * K ** -0.5, rng.standard_normal((n, N, r)) * 0.05
    a32[..., far] = 0
    if bf16:
        (a, b) = ((v.astype(np.float32).view(np.uint32) >> 16).astype(np.uint16) for v in (a32, b32))
        a64, b64 = ((v.astype(np.uint32) << 16).view(np.float32).astype(np.float64) for v in (a, b))
    else:
        a16, b16 = a32.astype(np.float16), b32.astype(np.float16)
        a, b, a64, b64 = a16.view(np.uint16), b16.view(np.uint16), a16.astype(np.float64), b16.astype(np.float64)
    scale, idx = np.ones(n, np.float32), rng.integers(0, n, T).astype(np.int32)
    got = run(ctx, x, y, idx, a, b, scale, N, bf16)
    x64 = x.astype(np.float64)
    want, _, tol = ref.lora(x64, y.astype(np.float64), idx, a64, b64, np.ones(n))
    if not bf16:
        near = np.abs(x64.reshape(T, K // 32, 32)).max(-1).repeat(32, -1)
        for t in range(T):
            A, B = a64[idx[t]], b64[idx[t]]
            tol[t] += 2.0 ** -39 * (np.abs(B) @ (np.abs(A) @ near[t])) + 2.0 ** -39 * np.abs(B).sum(-1) * np.abs(A @ x64[t]).max() * (1 + 2.0 ** -10)
    assert np.all(np.abs(got - want) <= tol)
    if size == 1e10 and not bf16:                          # the bound is of this: f32 alone would not leave as much
        assert np.abs(got - want).max() > 1e3 * ref.U * np.abs(want).max()


@pytest.mark.parametrize("bf16", [False, True])
def test_repeats_and_replays_bit_for_bit(ctx, bf16):
    """A captured call follows rows and indices from replay to replay, with another size's call on the same scratch between."""
    rng = np.random.default_rng(6)
    T, K, N, r, n = 300, 2048, 300, 32, 6
    assert T * r > MANY
    (a, a64), (b, b64) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    scale = rng.uniform(0.5, 2, n).astype(np.float32)
    da, db, ds = (ctx.upload(v) for v in (a, b, scale))
    dx, di, y1, y2 = ctx.zeros(T * K * 4), ctx.zeros(T * 4), ctx.zeros(T * N * 4), ctx.zeros(T * N * 4)
    call = lambda y, T: ctx.call("ti_lora_add", dx, di, da, db, ds, y, T, K, N, r, n, 0, 0, int(bf16))  # noqa: E731
    ctx.graph_begin()
    call(y1, T)
    g = ctx.graph_end()
    for _ in range(4):
        x, y, idx = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32), rng.integers(-1, n, T).astype(np.int32)
        for d, v in ((dx, x), (di, idx), (y1, y), (y2, y)):
            ctx.write(d, v)
        ctx.graph_launch(g)
        call(y2, T - 7)
        ctx.write(y2, y)
        call(y2, T)
        got = ctx.download(y1, np.float32, y.size).reshape(y.shape)
        want, norm, _ = ref.lora(*f64(x, y), idx, a64, b64, *f64(scale))
        assert np.array_equal(got.ravel(), ctx.download(y2, np.float32, y.size)) and np.linalg.norm(got - want) <= norm
    ctx.graph_destroy(g)
    for v in (da, db, ds, dx, di, y1, y2):
        v.free()


def plain(x, y, idx, a64, b64, scale):
    """The formula as it stands in 64 bits, infinities and NaN included (no library product, which may add zeros times infinity of its own)."""
    want = y.astype(np.float64)
    with np.errstate(invalid="ignore"):
        for t, i in enumerate(idx):
            h = (a64[i] * x[t].astype(np.float64)).sum(-1) * float(scale[i])
            want[t] += (b64[i] * h).sum(-1)
    return want


@pytest.mark.parametrize("bf16", [False, True])
@pytest.mark.parametrize("T,K,r", [(30, 320, 1), (30, 544, 16), (8300, 64, 1), (530, 544, 16), (130, 2080, 66)])
def test_infinite_activations_give_what_the_formula_does(ctx, T, K, r, bf16):
    """However many rows a call has: infinities of the weights' signs, NaN where two of them meet, beside elements of any size."""
    rng = np.random.default_rng(7)
    N, n = 21, 3
    x, y = rng.standard_normal((T, K)).astype(np.float32), rng.standard_normal((T, N)).astype(np.float32)
    (a, _), (b, _) = weights(rng, (n, r, K), K ** -0.5, bf16), weights(rng, (n, N, r), 0.05, bf16)
    if r > 1:                                              # adapters 0 and 1 of one sign each, so that infinities do not cancel
        a[0], b[0], a[1], b[1] = a[0] & 0x7FFF, b[0] & 0x7FFF, a[1] & 0x7FFF, b[1] | 0x8000
    f = (lambda v: (v.astype(np.uint32) << 16).view(np.float32).astype(np.float64)) if bf16 else (lambda v: v.view(np.float16).astype(np.float64))
    a64, b64 = f(a), f(b)
    scale = np.array([0.5, 1.5, -2.0], np.float32)
    idx = rng.integers(0, n, T).astype(np.int32)
    hit = rng.random(T) < 0.5
    for t in np.flatnonzero(hit):
        at = rng.choice(K, int(rng.integers(1, 3)), replace=False)
        x[t, rng.integers(0, K, 5)] = 10.0 ** rng.uniform(-30, 30, 5) * rng.choice([-1, 1], 5)
        x[t, at] = np.inf * rng.choice([1, 1, 1, -1], len(at))
    got, want = run(ctx, x, y, idx, a, b, scale, N, bf16), plain(x, y, idx, a64, b64, scale)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    for s in (np.inf, -np.inf):
        assert np.any(want == s) and np.array_equal(got == s, want == s)
    fine = ~hit
    _, _, tol = ref.lora(*f64(x[fine], y[fine]), idx[fine], a64, b64, *f64(scale))
    assert np.all(np.abs(got[fine] - want[fine]) <= tol)
