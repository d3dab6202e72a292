"""The operators over a part of the KV cache where their launches, scratch and callers meet: captured runs, two contexts,
the largest calls, the shortest chunks, and the launchers of the JavaScript host."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import span_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
NODE = shutil.which("node")


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def queries(rng, T, nHq, hd):
    return rng.standard_normal((T, nHq, hd)).astype(np.float32)


class Step:
    """A decode step or a chunk of one sequence: rows written, attention under a window, attention with the weights added
    up, the cache cut by one slot into buffers of its own."""

    def __init__(self, ctx, T, pos0, nHq, nKv, hd, keep):
        self.ctx, self.dims, self.S = ctx, (T, pos0, nHq, nKv, hd), pos0 + T
        self.keep = keep
        S = self.S
        self.src = [ctx.zeros(T * nHq * hd * 4), ctx.zeros(T * nKv * hd * 4), ctx.zeros(T * nKv * hd * 4)]
        self.cache = [ctx.zeros(S * nKv * hd), ctx.zeros(S * nKv * hd // 8), ctx.zeros(S * nKv * hd), ctx.zeros(S * nKv * hd // 8)]
        self.pos = ctx.upload(np.arange(pos0, S, dtype=np.int32))
        self.outs = [ctx.zeros(T * nHq * hd * 4), ctx.zeros(T * nHq * hd * 4), ctx.zeros(S * nKv * 4), ctx.zeros(keep * nKv * 4),
                     ctx.zeros(keep * nKv * 4)]

    def fill(self, seed):
        T, pos0, nHq, nKv, hd = self.dims
        rng = np.random.default_rng(seed)
        for d, a in zip(self.src, (queries(rng, T, nHq, hd), queries(rng, T, nKv, hd), queries(rng, T, nKv, hd))):
            self.ctx.write(d, a)
        for d, a in zip(self.cache, ref.cache(rng, self.S, nKv, hd)):
            self.ctx.write(d, a)
        self.ctx.write(self.outs[2], rng.uniform(0, 3, self.S * nKv).astype(np.float32))

    def run(self):
        T, pos0, nHq, nKv, hd = self.dims
        q, k, v = self.src
        c = self.ctx
        c.call("ti_kv_write_paged_q8", k, v, *self.cache, None, None, self.pos, T, 1, nKv, hd, 1, self.S, 0)
        c.call("ti_attn_window_q8", q, *self.cache, self.outs[0], T, pos0, nHq, nKv, hd, 60, 4)
        c.call("ti_attn_mass_q8", q, *self.cache, self.outs[1], self.outs[2], T, pos0, nHq, nKv, hd)
        c.call("ti_kv_evict_q8", *self.cache, self.outs[2], None, self.outs[3], self.outs[4], self.S, 0, self.keep, 4, 16, self.S, nKv, hd)

    def results(self):
        return [self.ctx.download(b, np.uint32, b.nbytes // 4) for b in self.outs + self.cache]

    def free(self):
        for b in self.src + self.cache + self.outs + [self.pos]:
            b.free()


@pytest.mark.parametrize("T,pos0,nHq,nKv,hd,less", [(1, 400, 16, 8, 128, 1), (1, 90, 6, 2, 96, 7), (4, 300, 16, 8, 128, 1), (70, 200, 8, 4, 64, 100)])
def test_a_captured_run_replays_like_eager(ctx, T, pos0, nHq, nKv, hd, less):
    """Four operators captured together; replays over other data, with eager calls of the same ones and waits between."""
    a, b = (Step(ctx, T, pos0, nHq, nKv, hd, pos0 + T - less) for _ in range(2))
    a.fill(0)
    a.run()                                              # the kernels are loaded
    ctx.graph_begin()
    a.run()
    g = ctx.graph_end()
    try:
        for seed in range(1, 5):
            a.fill(seed)
            b.fill(seed)
            ctx.graph_launch(g)
            if seed % 2:
                ctx.sync()
            b.run()
            assert all(np.array_equal(x, y) for x, y in zip(a.results(), b.results())), seed
    finally:
        ctx.graph_destroy(g)
        a.free()
        b.free()


def test_two_contexts_at_once():
    """Each with its stream and scratch: calls that alternate between them give what each gives alone."""
    with abi.Ctx(0) as c1, abi.Ctx(0) as c2:
        dims = [(1, 3000, 16, 8, 128, 3000), (90, 700, 16, 8, 64, 500)]
        alone = []
        for c, d in ((c1, dims[0]), (c2, dims[1])):
            s = Step(c, *d)
            s.fill(7)
            s.run()
            alone.append(s.results())
            s.free()
        s1, s2 = Step(c1, *dims[0]), Step(c2, *dims[1])
        for _ in range(5):
            s1.fill(7)
            s2.fill(7)
            s1.run()
            s2.run()
            assert all(np.array_equal(x, y) for x, y in zip(s1.results(), alone[0]))
            assert all(np.array_equal(x, y) for x, y in zip(s2.results(), alone[1]))
        s1.free()
        s2.free()


def test_the_most_sequences_and_heads(ctx):
    """2048 sequences of 64 heads; every 97th against 64 bits."""
    rng = np.random.default_rng(3)
    B, nHq, nKv, hd, page, pages, width = 2048, 64, 16, 32, 8, 500, 12
    lens = rng.integers(0, page * width + 1, B).astype(np.int32)
    lens[[0, 1, 5, -1]] = [0, page * width, 1, page * width]
    table = rng.integers(0, pages, (B, width)).astype(np.int32)
    q, (kc, ks, vc, vs) = queries(rng, B, nHq, hd), ref.cache(rng, pages * page, nKv, hd)
    dev = [ctx.upload(a) for a in (q, kc, ks, vc, vs, table, lens)]
    o = ctx.upload(np.full(q.size, np.nan, np.float32))
    ctx.call("ti_attn_paged_q8", *dev, o, B, nHq, nKv, hd, page, pages, width, 70, 5)
    got = ctx.download(o, np.float32, q.size).reshape(q.shape)
    assert np.all(np.isfinite(got)) and np.all(got[lens == 0] == 0)
    for b in sorted({0, 1, 5, B - 1} | set(range(0, B, 97))):
        j = np.arange(lens[b])
        if len(j) == 0:
            continue
        rows = table[b, j // page].astype(np.int64) * page + j % page
        seen = ref.visible([lens[b] - 1], j, 70, 5)
        want, tol, _, _ = ref.attend(q[b:b + 1], ref.values(kc[rows], ks[rows]), ref.values(vc[rows], vs[rows]), seen)
        assert np.all(np.abs(got[b] - want[0]) <= tol[0]), b
    for x in dev + [o]:
        x.free()


@pytest.mark.parametrize("T", [2, 3, 4, 5, 8, 9, 16, 17])
@pytest.mark.parametrize("nHq,nKv,hd", [(2, 1, 128), (4, 4, 96), (6, 2, 32)])
def test_short_chunks(ctx, T, nHq, nKv, hd):
    """On either side of the row counts where one kernel ends and the other begins."""
    rng = np.random.default_rng(T)
    pos0, window, sinks = 150, 64, 3
    S = pos0 + T
    q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
    dev = [ctx.upload(a) for a in (q, kc, ks, vc, vs)]
    o, o2, dm = ctx.zeros(q.nbytes), ctx.zeros(q.nbytes), ctx.zeros(S * nKv * 4)
    ctx.call("ti_attn_window_q8", *dev, o, T, pos0, nHq, nKv, hd, window, sinks)
    ctx.call("ti_attn_mass_q8", *dev, o2, dm, T, pos0, nHq, nKv, hd)
    K, V = ref.values(kc, ks), ref.values(vc, vs)
    for b, w, s in ((o, window, sinks), (o2, -1, 0)):
        want, tol, p, rel = ref.attend(q, K, V, ref.visible(pos0 + np.arange(T), np.arange(S), w, s))
        assert np.all(np.abs(ctx.download(b, np.float32, q.size).reshape(q.shape) - want) <= tol)
    add = p.reshape(T, nKv, -1, S).sum((0, 2)).T
    mtol = (p * rel[..., None]).reshape(T, nKv, -1, S).sum((0, 2)).T + (T * nHq // nKv + 3) * ref.U * add
    assert np.all(np.abs(ctx.download(dm, np.float32, S * nKv).reshape(S, nKv) - add) <= mtol)
    for x in dev + [o, o2, dm]:
        x.free()


def test_weights_over_two_to_the_29_keys(ctx):
    """2^23 and some positions of 64 heads, every score 0: each key's weight is 1 over the count, exactly summed (integers
    below 2^24): three roundings a row, one of the sum."""
    T, pos0, n, hd = 2, 2 ** 23 + 77, 64, 32
    S = pos0 + T

    def filled(words, value):
        b = ctx.alloc(4 * words)
        for at in range(0, words, 1 << 28):
            ctx.fill_u32(b.at(4 * at), value, min(1 << 28, words - at))
        return b

    one = int(np.float32(1).view(np.uint32))
    cache = [filled(S * n * hd // 4, 0), filled(S * n, one), filled(S * n * hd // 4, 0), filled(S * n, one)]
    mass = filled(S * n, 0)
    v = np.zeros((n, hd), np.int8)
    v[63] = 127
    ctx.write(cache[2], v, (2 ** 23 + 5) * n * hd)
    q = ctx.upload(queries(np.random.default_rng(0), T, n, hd))
    o = ctx.zeros(T * n * hd * 4)
    ctx.call("ti_attn_mass_q8", q, *cache, o, mass, T, pos0, n, n, hd)
    rows = 1.0 / (pos0 + 1 + np.arange(T))               # a key's weight in each row
    for a in (0, 4096 * 32 - 5, 2 ** 22, 2 ** 23 - 10, pos0 - 20):
        m = min(40, S - a)
        got = ctx.download(mass, np.float32, m * n, a * n * 4).reshape(m, n)
        want = np.array([rows[max(0, j - pos0):].sum() for j in range(a, a + m)])[:, None]
        assert np.all(np.abs(got - want) <= 4 * ref.U * want), a
    got = ctx.download(o, np.float32, T * n * hd).reshape(T, n, hd)
    want = np.zeros(got.shape)
    want[:, 63] = rows[:, None]
    assert np.all(np.abs(got - want) <= 4 * ref.U * want)
    for b in cache + [mass, q, o]:
        b.free()


@pytest.mark.parametrize("n,known,nKv,kind", [(2, 2, 3, "plain"), (64, 0, 2, "equal"), (65, 30, 2, "nan"), (8193, 8192, 2, "plain"), (20000, 0, 3, "equal"),
                                              (20000, 20000, 2, "nan"), (70001, 5, 1, "plain")])
def test_one_slot_too_many(ctx, n, known, nKv, kind):
    rng = np.random.default_rng(n)
    hd, keep, sinks, recent, nxt = 32, n - 1, min(1, n - 2), 0, n + 3
    mass = rng.uniform(0.5, 1, (n, nKv)).astype(np.float32)
    if kind == "equal":
        mass[:] = 1.0
    if kind == "nan":
        mass[rng.integers(1, n, 3)] = np.nan
        mass[rng.integers(1, n, 3)] = -np.inf
    where = np.stack([rng.permutation(nxt - (n - known))[:known] for _ in range(nKv)], 1).astype(np.int32) if known else None
    kc, ks, vc, vs = ref.cache(rng, n, nKv, hd)
    dev = [ctx.upload(a) for a in (kc, ks, vc, vs, mass)]
    dw = ctx.upload(np.concatenate([where, np.full((n - known, nKv), -77, np.int32)]) if known else np.full((n, nKv), -77, np.int32))
    ctx.call("ti_kv_evict_q8", *dev, dw if known else None, dev[4], dw, n, known, keep, sinks, recent, nxt, nKv, hd)
    src, pos = ref.evict(mass, where, n, known, keep, sinks, recent, nxt)
    h = np.arange(nKv)[None]
    assert np.array_equal(ctx.download(dw, np.int32, n * nKv).reshape(n, nKv)[:keep], pos)
    for d, a in zip(dev, (kc, ks, vc, vs, mass)):
        got = ctx.download(d, a.dtype, a.size).reshape(a.shape)
        assert np.array_equal(got[:keep].view(np.uint8), np.ascontiguousarray(a[src, h]).view(np.uint8))
    for b in dev + [dw]:
        b.free()


def test_half_of_a_million_slots(ctx):
    """A head's slots go through the select in many chunks, equal masses among them."""
    rng = np.random.default_rng(6)
    n, keep, nKv, hd = 1_000_000, 500_000, 1, 32
    mass = rng.integers(0, 3000, (n, nKv)).astype(np.float32)
    kc, ks, vc, vs = ref.cache(rng, n, nKv, hd)
    dev = [ctx.upload(a) for a in (kc, ks, vc, vs, mass)]
    mo, wo = ctx.zeros(keep * 4), ctx.zeros(keep * 4)
    ctx.call("ti_kv_evict_q8", *dev, None, mo, wo, n, 0, keep, 4, 1000, n, nKv, hd)
    src, pos = ref.evict(mass, None, n, 0, keep, 4, 1000, n)
    h = np.arange(nKv)[None]
    assert np.array_equal(ctx.download(wo, np.int32, keep).reshape(keep, 1), pos)
    for d, a in zip(dev[:4] + [mo], (kc, ks, vc, vs, mass)):
        got = ctx.download(d, a.dtype, keep * a[0].size).reshape((keep,) + a.shape[1:])
        assert np.array_equal(got, a[src, h])
    for x in dev + [mo, wo]:
        x.free()


def test_a_cache_without_a_table_needs_no_sequences(ctx):
    rng = np.random.default_rng(1)
    T, nKv, hd = 4, 2, 64
    k = rng.standard_normal((T, nKv, hd)).astype(np.float32)
    cache = [ctx.zeros(8 * nKv * hd), ctx.zeros(8 * nKv * hd // 8), ctx.zeros(8 * nKv * hd), ctx.zeros(8 * nKv * hd // 8)]
    dk, pos, back = ctx.upload(k), ctx.upload(np.array([6, 1, 7, 0], np.int32)), [ctx.zeros(k.nbytes) for _ in range(2)]
    ctx.call("ti_kv_write_paged_q8", dk, dk, *cache, None, None, pos, T, 0, nKv, hd, 8, 1, 0)
    ctx.call("ti_kv_read_paged_q8", *cache, None, None, pos, *back, T, 0, nKv, hd, 8, 1, 0)
    for b in back:                                       # half a step of a group's 127 codes, and f32 roundings
        got = ctx.download(b, np.float32, k.size).reshape(T, nKv, 2, 32)
        x = k.reshape(T, nKv, 2, 32)
        assert np.all(np.abs(got - x) <= np.abs(x).max(-1, keepdims=True) * (0.5 / 127 + 8 * ref.U))
    for b in cache + back + [dk, pos]:
        b.free()


@pytest.mark.parametrize("T", [1, 3, 12, 150])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_a_rows_query_is_its_own(ctx, T, bad):
    """A query that is not finite (a padded row's) leaves the other heads and tokens as they are."""
    rng = np.random.default_rng(T)
    nHq, nKv, hd, pos0, window, sinks = 8, 4, 64, 300, 100, 2
    S = pos0 + T
    q, (kc, ks, vc, vs) = queries(rng, T, nHq, hd), ref.cache(rng, S, nKv, hd)
    dirty = q.copy()
    dirty[T // 2, 3, 5:9] = bad
    o = ctx.zeros(q.nbytes)
    dev = [ctx.upload(a) for a in (dirty, kc, ks, vc, vs)]
    ctx.call("ti_attn_window_q8", *dev, o, T, pos0, nHq, nKv, hd, window, sinks)
    got = ctx.download(o, np.float32, q.size).reshape(q.shape)
    want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), ref.visible(pos0 + np.arange(T), np.arange(S), window, sinks))
    ok = np.ones((T, nHq), bool)
    ok[T // 2, 3] = False
    assert np.all((np.abs(got - want) <= tol)[ok]) and np.all(np.isnan(got[T // 2, 3]))
    for x in dev + [o]:
        x.free()


def test_padded_rows_of_a_batch(ctx):
    """Rows without a sequence (length 0, garbage in the query and the table) give zeros, the others their own results."""
    rng = np.random.default_rng(2)
    B, nHq, nKv, hd, page, pages, width = 5, 16, 8, 128, 16, 30, 6
    lens = np.array([90, 0, 17, -3, 40], np.int32)
    table = np.stack([rng.permutation(pages)[:width] for _ in range(B)]).astype(np.int32)
    q, (kc, ks, vc, vs) = queries(rng, B, nHq, hd), ref.cache(rng, pages * page, nKv, hd)
    q[1], q[3] = np.nan, np.inf
    table[1], table[3] = 2 ** 31 - 1, -2 ** 31
    dev = [ctx.upload(a) for a in (q, kc, ks, vc, vs, table, lens)]
    o = ctx.upload(np.full(q.size, np.nan, np.float32))
    ctx.call("ti_attn_paged_q8", *dev, o, B, nHq, nKv, hd, page, pages, width, -1, 0)
    got = ctx.download(o, np.float32, q.size).reshape(q.shape)
    assert np.all(got[[1, 3]] == 0)
    for b in (0, 2, 4):
        j = np.arange(lens[b])
        rows = table[b, j // page].astype(np.int64) * page + j % page
        want, tol, _, _ = ref.attend(q[b:b + 1], ref.values(kc[rows], ks[rows]), ref.values(vc[rows], vs[rows]), ref.visible([lens[b] - 1], j, -1, 0))
        assert np.all(np.abs(got[b] - want[0]) <= tol[0]), b
    for x in dev + [o]:
        x.free()


@pytest.mark.parametrize("n,keep", [(300, 299), (300, 120), (5000, 4000)])
@pytest.mark.parametrize("mass_in_place", [True, False])
def test_one_of_the_slots_buffers_in_place(ctx, n, keep, mass_in_place):
    """Masses cut in place and positions elsewhere, or the other way round."""
    rng = np.random.default_rng(n)
    nKv, hd, known, nxt = 3, 32, n - 7, n + 50
    mass = rng.uniform(0, 1, (n, nKv)).astype(np.float32)
    where = np.stack([rng.permutation(nxt - 7)[:known] for _ in range(nKv)], 1).astype(np.int32)
    kc, ks, vc, vs = ref.cache(rng, n, nKv, hd)
    dev = [ctx.upload(a) for a in (kc, ks, vc, vs, mass, np.concatenate([where, np.full((7, nKv), -77, np.int32)]))]
    mo = dev[4] if mass_in_place else ctx.zeros(keep * nKv * 4)
    wo = ctx.zeros(keep * nKv * 4) if mass_in_place else dev[5]
    ctx.call("ti_kv_evict_q8", *dev, mo, wo, n, known, keep, 3, 20, nxt, nKv, hd)
    src, pos = ref.evict(mass, where, n, known, keep, 3, 20, nxt)
    h = np.arange(nKv)[None]
    assert np.array_equal(ctx.download(wo, np.int32, keep * nKv).reshape(keep, nKv), pos)
    assert np.array_equal(ctx.download(mo, np.float32, keep * nKv).reshape(keep, nKv), mass[src, h])
    assert np.array_equal(ctx.download(dev[0], np.int8, kc.size).reshape(kc.shape)[:keep], kc[src, h])
    for x in dev + [mo, wo]:
        x.free()


@pytest.mark.skipif(NODE is None, reason="node is not installed")
def test_javascript_launchers(tmp_path):
    """The host's six launchers: a paged prompt and token, a window, weights added up, an eviction and what it leaves."""
    d = str(tmp_path)
    rng = np.random.default_rng(4)
    T, nHq, nKv, hd, page, pages, width = 21, 8, 2, 64, 8, 9, 4
    S, keep = T, 12
    table = np.array([[4, 0, 7, -1], [2, -1, -1, -1]], np.int32)
    k, v, q = queries(rng, T, nKv, hd), queries(rng, T, nKv, hd), queries(rng, T, nHq, hd)
    seq, pos = np.array([0] * 20 + [1], np.int32), np.array(list(range(20)) + [0], np.int32)
    kc, ks, vc, vs = ref.cache(rng, S, nKv, hd)
    files = dict(table=table, k=k, v=v, q=q, seq=seq, pos=pos, lens=np.array([20, 1], np.int32), kc=kc, ks=ks, vc=vc, vs=vs)
    for n, a in files.items():
        np.ascontiguousarray(a).tofile(os.path.join(d, n))
    json.dump(dict(T=T, nHq=nHq, nKv=nKv, hd=hd, page=page, pages=pages, width=width, S=S, keep=keep, files=sorted(files)),
              open(os.path.join(d, "spec.json"), "w"))
    r = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "run_kv.js"), d], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert r.returncode == 0, r.stdout

    def out(name, dt, shape):
        return np.fromfile(os.path.join(d, name), dt).reshape(shape)

    # paged: what was read back is what the attention saw
    K, V = out("k.out", np.float32, k.shape).astype(np.float64), out("v.out", np.float32, v.shape).astype(np.float64)
    for got, want in ((K, k), (V, v)):
        x = want.reshape(T, nKv, 2, 32)
        assert np.all(np.abs(got.reshape(x.shape) - x) <= np.abs(x).max(-1, keepdims=True) * (0.5 / 127 + 8 * ref.U))
    paged = out("paged.out", np.float32, (2, nHq, hd))
    for b, rows in ((0, slice(0, 20)), (1, slice(20, 21))):
        n = len(K[rows])
        want, tol, _, _ = ref.attend(q[b:b + 1], K[rows], V[rows], ref.visible([n - 1], np.arange(n), 9, 2))
        # two more roundings of each value that was read back
        more = 2 * ref.U * (1 + 2 * (np.abs(q[b]).sum(-1).max() * np.abs(K).max())) * np.abs(V).max()
        assert np.all(np.abs(paged[b] - want[0]) <= tol[0] + more)
    Kc, Vc = ref.values(kc, ks), ref.values(vc, vs)
    p = np.arange(T)
    want, tol, _, _ = ref.attend(q, Kc, Vc, ref.visible(p, p, 7, 2))
    assert np.all(np.abs(out("window.out", np.float32, q.shape) - want) <= tol)
    want, tol, w, rel = ref.attend(q, Kc, Vc, ref.visible(p, p, -1, 0))
    assert np.all(np.abs(out("mass_attn.out", np.float32, q.shape) - want) <= tol)
    mass = out("mass.out", np.float32, (S, nKv))
    add = w.reshape(T, nKv, -1, S).sum((0, 2)).T
    assert np.all(np.abs(mass - add) <= rel.max() * add + 100 * ref.U * add)
    src, at = ref.evict(mass, None, S, 0, keep, 2, 3, S)
    assert np.array_equal(out("where.out", np.int32, (S, nKv))[:keep], at)
    assert np.array_equal(out("kc.out", np.int8, kc.shape)[:keep], kc[src, np.arange(nKv)[None]])
    assert np.array_equal(out("cut.out", np.float32, (S, nKv))[:keep], mass[src, np.arange(nKv)[None]])
