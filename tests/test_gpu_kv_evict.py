"""Eviction from the int8 KV cache by accumulated attention weight: which slots stay, where they go and what they hold,
exactly; and a generation that attends, adds up and evicts as it goes."""
import numpy as np
import pytest

import span_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def masses(rng, kind, n, nKv):
    if kind == "equal":
        return np.full((n, nKv), 0.5, np.float32)
    if kind == "few":                                   # many ties, both zeros among them
        return rng.choice(np.array([0.0, -0.0, 1.0, 2.0, 1e-30], np.float32), (n, nKv))
    m = np.exp(4 * rng.standard_normal((n, nKv))).astype(np.float32)
    if kind == "odd":                                   # what no attention leaves: negative, infinite, not a number
        m = m * rng.choice(np.array([1, -1], np.float32), m.shape)
        for x in (np.nan, np.inf, -np.inf, -np.nan, np.finfo(np.float32).tiny / 4):
            m[rng.random(m.shape) < 0.05] = x
    return m


# n, known, keep, sinks, recent, nKv, hd
CASES = [(1, 0, 1, 0, 0, 1, 32), (2, 0, 1, 0, 0, 2, 64), (2, 2, 1, 1, 0, 1, 32), (65, 64, 64, 4, 16, 8, 128), (100, 0, 10, 0, 10, 5, 96),
         (100, 40, 99, 0, 0, 3, 64), (300, 300, 20, 20, 0, 2, 128), (1024, 0, 512, 4, 100, 8, 128), (1025, 1000, 1, 0, 1, 1, 32),
         (4097, 4096, 4096, 4, 512, 8, 128), (5000, 17, 2500, 3, 3, 4, 64), (30000, 0, 4096, 4, 1024, 2, 32), (70001, 60000, 300, 1, 9, 1, 32),
         (50, 50, 50, 2, 2, 2, 32), (50, 20, 400, 2, 2, 2, 32)]


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("kind", ["plain", "equal", "few", "odd"])
@pytest.mark.parametrize("n,known,keep,sinks,recent,nKv,hd", CASES)
def test_evict(ctx, n, known, keep, sinks, recent, nKv, hd, kind, in_place):
    rng = np.random.default_rng(n + keep)
    kept = min(keep, n)
    nxt = n + 500 if known else n
    old = nxt - (n - known)
    where = np.stack([rng.permutation(old)[:known] for _ in range(nKv)], 1).astype(np.int32) if known else None
    mass = masses(rng, kind, n, nKv)
    kc, ks, vc, vs = ref.cache(rng, n + 2, nKv, hd)     # two rows behind the last slot
    dev = [ctx.upload(a) for a in (kc, ks, vc, vs)]
    full = np.full((n + 1, nKv), -77, np.int32)
    if known:
        full[:known] = where
    dm, dw = ctx.upload(np.concatenate([mass, np.full((1, nKv), -5, np.float32)])), ctx.upload(full)
    mo, wo = (dm, dw) if in_place else (ctx.upload(np.full((kept + 1, nKv), -5, np.float32)), ctx.upload(np.full((kept + 1, nKv), -77, np.int32)))
    ctx.call("ti_kv_evict_q8", *dev, dm, dw if known else None, mo, wo, n, known, keep, sinks, recent, nxt, nKv, hd)
    src, pos = ref.evict(mass, where, n, known, keep, sinks, recent, nxt)
    h = np.arange(nKv)[None]
    rows = n + 1 if in_place else kept + 1
    gm, gw = ctx.download(mo, np.uint32, rows * nKv).reshape(rows, nKv), ctx.download(wo, np.int32, rows * nKv).reshape(rows, nKv)
    assert np.array_equal(gw[:kept], pos)
    assert np.array_equal(gm[:kept], mass.view(np.uint32)[src, h])
    if in_place:                                        # what is behind the kept slots stays
        assert np.array_equal(gm[kept:n], mass.view(np.uint32)[kept:]) and np.all(gm[n] == np.float32(-5).view(np.uint32))
        assert np.array_equal(gw[kept:], full[kept:])
    else:
        assert np.all(gm[kept] == np.float32(-5).view(np.uint32)) and np.all(gw[kept] == -77)
    for d, a in zip(dev, (kc, ks, vc, vs)):
        got = ctx.download(d, a.dtype, a.size).reshape(a.shape)
        assert np.array_equal(got[:kept], a[src, h]) and np.array_equal(got[kept:], a[kept:])
    for b in dev + [dm, dw] + ([] if in_place else [mo, wo]):
        b.free()


def test_generation_under_eviction(ctx, orc):
    """A prompt and 60 tokens in a cache of 40 slots: every token written to the next slot, its attention over the
    slots against 64 bits, the weights added up, and the cache cut to 32 slots whenever it is full. The slots chosen
    are compared given the accumulated weights that the device holds (which are themselves held to 64 bits)."""
    rng = np.random.default_rng(5)
    nHq, nKv, hd, cap, keep, sinks, recent, theta, eps = 16, 8, 128, 40, 32, 2, 8, 1e6, 1e-6
    cache = [ctx.zeros(cap * nKv * hd), ctx.zeros(cap * nKv * hd // 8), ctx.zeros(cap * nKv * hd), ctx.zeros(cap * nKv * hd // 8)]
    dm, dw = ctx.upload(np.full((cap, nKv), np.nan, np.float32)), ctx.upload(np.full((cap, nKv), -1, np.int32))
    nw = ctx.upload((1 + 0.1 * rng.standard_normal(hd)).astype(np.float16).view(np.uint16))
    n = known = nxt = 0
    where = np.zeros((0, nKv), np.int32)
    for step in range(61):
        T = 25 if step == 0 else 1
        bufs = [ctx.upload(rng.standard_normal((T, h, hd)).astype(np.float32)) for h in (nHq, nKv, nKv)]
        qr, kr, do = ctx.zeros(T * nHq * hd * 4), ctx.zeros(T * nKv * hd * 4), ctx.zeros(T * nHq * hd * 4)
        ctx.call("ti_rope_qk", bufs[0], nw, qr, T, nHq, hd, nxt, np.float32(theta), np.float32(eps))
        ctx.call("ti_rope_qk", bufs[1], nw, kr, T, nKv, hd, nxt, np.float32(theta), np.float32(eps))
        ctx.call("ti_kv_write_q8", kr, bufs[2], *cache, T, nKv, hd, n)
        before = ctx.download(dm, np.float32, cap * nKv).reshape(cap, nKv)
        ctx.call("ti_attn_mass_q8", qr, *cache, do, dm, T, n, nHq, nKv, hd)
        got, q = (ctx.download(b, np.float32, T * nHq * hd).reshape(T, nHq, hd) for b in (do, qr))
        mass = ctx.download(dm, np.float32, cap * nKv).reshape(cap, nKv)
        S = n + T
        kv = [ctx.download(cache[i], np.int8, S * nKv * hd).reshape(S, nKv, hd) for i in (0, 2)]
        sc = [ctx.download(cache[i], np.float32, S * nKv * hd // 32).reshape(S, nKv, hd // 32) for i in (1, 3)]
        seen = ref.visible(n + np.arange(T), np.arange(S), -1, 0)
        want, tol, w, rel = ref.attend(q, ref.values(kv[0], sc[0]), ref.values(kv[1], sc[1]), seen)
        assert np.all(np.abs(got - want) <= tol), step
        add = w.reshape(T, nKv, 2, S).sum((0, 2)).T
        old = np.where(np.arange(S)[:, None] < n, before[:S], 0)
        assert np.all(np.abs(mass[:S] - old - add) <= rel.max() * add + (2 * T + 3) * ref.U * (np.abs(old) + add)), step
        n, nxt = S, nxt + T
        for b in bufs + [qr, kr, do]:
            b.free()
        if n == cap:
            ctx.call("ti_kv_evict_q8", *cache, dm, dw, dm, dw, n, known, keep, sinks, recent, nxt, nKv, hd)
            src, pos = ref.evict(mass, where, n, known, keep, sinks, recent, nxt)
            gw = ctx.download(dw, np.int32, keep * nKv).reshape(keep, nKv)
            assert np.array_equal(gw, pos)
            for i in range(2):
                c = ctx.download(cache[2 * i], np.int8, keep * nKv * hd).reshape(keep, nKv, hd)
                assert np.array_equal(c, kv[i][src, np.arange(nKv)[None]])
            assert np.all((gw < sinks).sum(0) == sinks) and np.all((gw >= nxt - recent).sum(0) == recent)
            n = known = keep
            where = gw
    assert nxt == 85 and known == keep
    for b in cache + [dm, dw, nw]:
        b.free()
