"""The attention over a part of the KV cache as near to 64 bits, in the 2-norm, as f32 arithmetic comes (tests/span_norm.py derives the
bound, tests/test_span_norm.py shows what it sees): under a window, over pages, and the weights that are added up."""
import numpy as np
import pytest

import span_norm as norm
import span_ref as ref
from span_cases import CHAIN, NORM_WINDOWS, inputs
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


@pytest.mark.parametrize("T,pos0,nHq,nKv,hd,window,sinks", NORM_WINDOWS)
def test_window(ctx, T, pos0, nHq, nKv, hd, window, sinks):
    q, (kc, ks, vc, vs) = inputs(T, pos0, nHq, nKv, hd)
    dev = [ctx.upload(a) for a in (q, kc, ks, vc, vs)]
    o = ctx.zeros(q.nbytes)
    ctx.call("ti_attn_window_q8", *dev, o, T, pos0, nHq, nKv, hd, window, sinks)
    got = ctx.download(o, np.float32, q.size).reshape(q.shape)
    seen = ref.visible(pos0 + np.arange(T), np.arange(pos0 + T), window, sinks)
    want, _, tol, _ = norm.attend(q, ref.values(kc, ks), ref.values(vc, vs), seen, CHAIN)
    assert norm.off(got, want) <= tol
    for x in dev + [o]:
        x.free()


@pytest.mark.parametrize("page", [1, 16, 64])
@pytest.mark.parametrize("pos0,nHq,nKv,hd,window,sinks", [c[1:] for c in NORM_WINDOWS if c[0] == 1])
def test_pages(ctx, pos0, nHq, nKv, hd, window, sinks, page):
    """The same tokens over pages in no order, three in one call."""
    rng = np.random.default_rng(page)
    q, (kc, ks, vc, vs) = inputs(3, pos0 - 2, nHq, nKv, hd)
    S = pos0 + 1
    width = (S + page - 1) // page
    table = rng.permutation(width + 3)[:width].astype(np.int32)
    rows = table[np.arange(S) // page].astype(np.int64) * page + np.arange(S) % page
    pool = []
    for a in (kc, ks, vc, vs):
        p = np.zeros(((width + 3) * page,) + a.shape[1:], a.dtype)
        p[rows] = a
        pool.append(p)
    lens = np.array([S - 2, S - 1, S], np.int32)
    dev = [ctx.upload(a) for a in [q] + pool + [np.stack([table] * 3), lens]]
    o = ctx.zeros(q.nbytes)
    ctx.call("ti_attn_paged_q8", *dev, o, 3, nHq, nKv, hd, page, width + 3, width, window, sinks)
    got = ctx.download(o, np.float32, q.size).reshape(q.shape)
    want, _, tol, _ = norm.attend(q, ref.values(kc, ks), ref.values(vc, vs), ref.visible(lens - 1, np.arange(S), window, sinks), CHAIN)
    assert norm.off(got, want) <= tol
    for x in dev + [o]:
        x.free()


@pytest.mark.parametrize("T,pos0,nHq,nKv,hd", [(1, 1000, 16, 8, 128), (1, 3333, 40, 8, 96), (1, 900, 20, 1, 64), (3, 500, 16, 1, 32), (17, 600, 6, 2, 96),
                                               (64, 0, 4, 2, 128), (100, 700, 16, 8, 128), (204, 1, 20, 1, 32), (256, 300, 16, 4, 64)])
def test_weights_added_up(ctx, T, pos0, nHq, nKv, hd):
    q, (kc, ks, vc, vs) = inputs(T, pos0, nHq, nKv, hd)
    S = pos0 + T
    dev = [ctx.upload(a) for a in (q, kc, ks, vc, vs)]
    o, dm = ctx.zeros(q.nbytes), ctx.zeros(S * nKv * 4)
    ctx.call("ti_attn_mass_q8", *dev, o, dm, T, pos0, nHq, nKv, hd)
    got, mass = ctx.download(o, np.float32, q.size).reshape(q.shape), ctx.download(dm, np.float32, S * nKv).reshape(S, nKv)
    seen = ref.visible(pos0 + np.arange(T), np.arange(S), -1, 0)
    want, w, tol, wtol = norm.attend(q, ref.values(kc, ks), ref.values(vc, vs), seen, CHAIN)
    assert norm.off(got, want) <= tol
    # of T nHq / nKv weights a key the sum, a rounding each: below n / 9 of the bound's terms
    assert norm.off(mass, w.reshape(T, nKv, -1, S).sum((0, 2)).T) <= wtol + 3 * norm.U * np.sqrt(T * nHq / nKv / 9)
    for x in dev + [o, dm]:
        x.free()
