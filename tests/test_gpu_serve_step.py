"""A served batch's step made of the calls in their order: projection and adapters, rows into pages, attention of groups, logits and log
probabilities. Captured once and replayed, each stage against its 64-bit reference from what the stage before left (tests/serve_ref.py and
tests/span_ref.py derive the tolerances); and the same calls from JavaScript."""
import json
import os
import shutil
import subprocess

import numpy as np
import pytest

import serve_ref as ref
import span_ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
NODE = shutil.which("node")
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
THETA, EPS = 1e6, 1e-6


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def int4(ctx, rng, N, K):
    return (ctx.upload(rng.integers(0, 2 ** 32, (N, K // 8), dtype=np.uint32)),
            ctx.upload((rng.uniform(0.2, 1, (N, K // 32)) * 0.2 * K ** -0.5).astype(np.float16)))


def adapters(ctx, rng, n, r, K, N):
    a, b = (rng.standard_normal((n, r, K)) * K ** -0.5).astype(np.float16), (rng.standard_normal((n, N, r)) * 0.1).astype(np.float16)
    s = rng.uniform(0.5, 2, n).astype(np.float32)
    return [ctx.upload(x) for x in (a, b, s)], [x.astype(np.float64) for x in (a, b, s)]


class Step:
    """One layer's attention and a head over one pool of pages; B sequences in groups."""
    H, nHq, nKv, hd, V, top, n, r = 256, 8, 4, 64, 1003, 7, 5, 16
    page, pages, width = 8, 200, 24

    def __init__(self, ctx, rng, B, P):
        self.ctx, self.B, self.P = ctx, B, P
        self.N = (self.nHq + 2 * self.nKv) * self.hd
        self.dim = self.nHq * self.hd
        rows = self.pages * self.page * self.nKv
        self.pool = [ctx.zeros(rows * self.hd), ctx.zeros(rows * self.hd // 8), ctx.zeros(rows * self.hd), ctx.zeros(rows * self.hd // 8)]
        self.wqkv, self.wo, self.head = int4(ctx, rng, self.N, self.H), int4(ctx, rng, self.H, self.dim), int4(ctx, rng, self.V, self.H)
        self.qkv_ad, self.qkv_ad64 = adapters(ctx, rng, self.n, self.r, self.H, self.N)
        self.o_ad, self.o_ad64 = adapters(ctx, rng, self.n, self.r, self.dim, self.H)
        self.norms = [rng.uniform(0.8, 1.2, d).astype(np.float16) for d in (self.H, self.hd, self.hd, self.H)]
        self.dnorms = [ctx.upload(w) for w in self.norms]
        self.ins = {k: ctx.zeros(4 * s) for k, s in dict(x=B * self.H, idx=B, table=B * self.width, pos=B, rot=B, lens=B, starts=P + 1, shared=P, ids=B).items()}

    def outs(self):
        B = self.B
        sizes = dict(xn=B * self.H, qkv=B * self.N, qr=B * self.dim, o=B * self.dim, y=B * self.H, yn=B * self.H, logits=B * self.V, lp=B, ent=B, rank=B,
                     top_ids=B * self.top, top_lp=B * self.top)
        return {k: self.ctx.zeros(4 * s) for k, s in sizes.items()}

    def run(self, u):
        c, i, B = self.ctx.call, self.ins, self.B
        c("ti_rmsnorm", i["x"], self.dnorms[0], u["xn"], B, self.H, EPS)
        c("ti_linear_q4", u["xn"], *self.wqkv, u["qkv"], B, self.N, self.H, 0)
        c("ti_lora_add", u["xn"], i["idx"], *self.qkv_ad, u["qkv"], B, self.H, self.N, self.r, self.n, 0, 0, 0)
        k, v = u["qkv"].at(4 * self.dim), u["qkv"].at(4 * (self.dim + self.nKv * self.hd))
        c("ti_attn_prep_paged_q8", u["qkv"], k, v, self.dnorms[1], self.dnorms[2], u["qr"], *self.pool, i["table"], None, i["pos"], i["rot"], B, B, self.nHq,
          self.nKv, self.hd, self.page, self.pages, self.width, self.N, self.N, THETA, EPS)
        c("ti_attn_shared_q8", u["qr"], *self.pool, i["table"], i["lens"], i["starts"], i["shared"], u["o"], B, self.P, self.nHq, self.nKv, self.hd, self.page,
          self.pages, self.width)
        c("ti_linear_q4", u["o"], *self.wo, u["y"], B, self.H, self.dim, 0)
        c("ti_lora_add", u["o"], i["idx"], *self.o_ad, u["y"], B, self.dim, self.H, self.r, self.n, 0, 0, 0)
        c("ti_rmsnorm", u["y"], self.dnorms[3], u["yn"], B, self.H, EPS)
        c("ti_linear_q4", u["yn"], *self.head, u["logits"], B, self.V, self.H, 0)
        c("ti_logprobs", u["logits"], i["ids"], u["lp"], u["ent"], u["rank"], u["top_ids"], u["top_lp"], B, self.V, 0, self.top)

    def linear(self, x, w, N, K):
        d, y = self.ctx.upload(x), self.ctx.zeros(4 * len(x) * N)
        self.ctx.call("ti_linear_q4", d, *w, y, len(x), N, K, 0)
        got = self.ctx.download(y, np.float32, len(x) * N).reshape(len(x), N)
        d.free()
        y.free()
        return got

    def cache(self):
        rows = self.pages * self.page
        return [self.ctx.download(b, t, rows * self.nKv * n).reshape(rows, self.nKv, n) for b, (t, n) in zip(self.pool, ((np.int8, self.hd), (np.float32, self.hd // 32)) * 2)]


def rows_of(table, page, starts, shared, b, n):
    """Pool rows of sequence b's n positions."""
    j, row = np.arange(n), np.full(n, b)
    for g in range(len(shared)):
        if starts[g] <= b < starts[g + 1] and starts[g + 1] - starts[g] > 1:
            row[j < shared[g]] = starts[g]
    return table[row, j // page].astype(np.int64) * page + j % page


def test_prompts_and_steps_of_a_batch(ctx):
    rng = np.random.default_rng(3)
    starts, shared, B = [0, 4, 7], [37, 90], 8
    st = Step(ctx, rng, B, 2)
    lens = np.array([37 + 5, 38, 37 + 20, 37 + 11, 91, 90 + 7, 99, 60], np.int32)
    table = np.arange(B * st.width, dtype=np.int32).reshape(B, st.width)[:, rng.permutation(st.width)]
    # the prompts: shared positions by their group's first sequence, then everyone's own; rows of any order in one call
    where = [(b, p) for b in range(B) for p in range(lens[b] - 1) if rows_of(table, st.page, starts, shared, b, p + 1)[-1] // st.page in table[b]]
    order = rng.permutation(len(where))
    seq, pos = np.array(where, np.int32)[order].T
    T = len(seq)
    kv = rng.standard_normal((T, 2, st.nKv, st.hd)).astype(np.float32)
    bufs = [ctx.upload(a) for a in (kv, np.ascontiguousarray(table), np.ascontiguousarray(seq), np.ascontiguousarray(pos))]
    ld = 2 * st.nKv * st.hd
    ctx.call("ti_attn_prep_paged_q8", None, bufs[0], bufs[0].at(2 * ld), None, st.dnorms[2], None, *st.pool, bufs[1], bufs[2], bufs[3], None, T, B, 0, st.nKv, st.hd,
             st.page, st.pages, st.width, 0, ld, THETA, EPS)
    for x in bufs:
        x.free()

    u, eager = st.outs(), st.outs()
    ctx.write(st.ins["table"], np.ascontiguousarray(table))
    ctx.graph_begin()
    st.run(u)
    graph = ctx.graph_end()
    x = (rng.standard_normal((B, st.H)) * rng.uniform(0.5, 3, (B, 1))).astype(np.float32)
    for turn in range(5):
        idx = rng.integers(-1, st.n, B).astype(np.int32)
        ids = rng.integers(0, st.V, B).astype(np.int32)
        rot = lens - 1 + 1000 * turn
        new = dict(x=x, idx=idx, ids=ids, pos=lens - 1, rot=rot, lens=lens, starts=starts, shared=shared)
        for name, a in new.items():
            ctx.write(st.ins[name], np.ascontiguousarray(a, np.float32 if name == "x" else np.int32))
        before = st.cache()
        ctx.graph_launch(graph)
        got = {k: ctx.download(b, np.int32 if k in ("rank", "top_ids") else np.float32, b.nbytes // 4) for k, b in u.items()}
        after = st.cache()
        # the program's own call of the same: the same bits
        st.run(eager)
        for k, b in eager.items():
            assert np.array_equal(ctx.download(b, np.uint32, b.nbytes // 4), got[k].view(np.uint32)), (turn, k)

        xn, qkv = got["xn"].reshape(B, -1), got["qkv"].reshape(B, -1)
        want, _, tol = ref.lora(xn.astype(np.float64), st.linear(xn, st.wqkv, st.N, st.H).astype(np.float64), idx, *st.qkv_ad64)
        assert np.all(np.abs(qkv - want) <= tol)
        q, k, v = np.split(qkv, [st.dim, st.dim + st.nKv * st.hd], 1)
        want, tol = ref.turn(q.reshape(B, st.nHq, st.hd), st.norms[1], rot, THETA, EPS)
        qr = got["qr"].reshape(B, st.nHq, st.hd)
        assert np.all(np.abs(qr - want) <= tol)
        at = np.array([rows_of(table, st.page, starts, shared, b, lens[b])[-1] for b in range(B)])
        rest = np.setdiff1d(np.arange(st.pages * st.page), at)
        for a, b in zip(after, before):
            assert np.array_equal(a[rest], b[rest])
        c, top, _ = ref.codes(v.reshape(B, st.nKv, st.hd))
        assert np.array_equal(after[2][at], c) and np.array_equal(after[3][at], top)
        c, top, far = ref.codes(ref.turn32(k.reshape(B, st.nKv, st.hd), st.norms[2], rot, THETA, EPS))
        off = np.abs(after[0][at].astype(int) - c)
        assert np.all((off == 0) | ((off == 1) & (far < 1e-4))) and np.all(np.abs(after[1][at] - top) <= 4 * ref.U * top)
        K, Vv = span_ref.values(after[0], after[1]), span_ref.values(after[2], after[3])
        o = got["o"].reshape(B, st.nHq, st.hd)
        for b in range(B):
            r = rows_of(table, st.page, starts, shared, b, lens[b])
            want, tol, _, _ = span_ref.attend(qr[b:b + 1], K[r], Vv[r], np.ones((1, len(r)), bool))
            assert np.all(np.abs(o[b] - want[0]) <= tol[0]), (turn, b)
        o = got["o"].reshape(B, -1)
        want, _, tol = ref.lora(o.astype(np.float64), st.linear(o, st.wo, st.H, st.dim).astype(np.float64), idx, *st.o_ad64)
        assert np.all(np.abs(got["y"].reshape(B, -1) - want) <= tol)
        want, tol = ref.logprobs(got["logits"].reshape(B, st.V), ids, st.top)
        assert np.array_equal(got["rank"], want["rank"]) and np.array_equal(got["top_ids"].reshape(B, -1), want["top_ids"])
        for name in ("lp", "ent", "top_lp"):
            assert np.all(np.abs(got[name].reshape(want[name].shape) - want[name]) <= tol[name]), (turn, name)
        x, lens = got["y"].reshape(B, -1) + x, lens + 1
        assert np.isfinite(x).all()
    ctx.graph_destroy(graph)


@pytest.mark.skipif(NODE is None, reason="node is not installed")
def test_javascript_launchers(ctx, tmp_path):
    """The same bits as through the C ABI from Python."""
    d, rng = str(tmp_path), np.random.default_rng(4)
    s = dict(T=60, B=3, nHq=8, nKv=2, hd=64, page=8, pages=30, width=5, P=1, K=96, N=75, r=8, n=4, V=5003, top=6)
    T, B, nHq, nKv, hd, page, pages, width, P, K, N, r, n, V, top = s.values()
    seq, pos = np.repeat([0, 1, 2], [40, 10, 10]), np.concatenate([np.arange(40), 25 + np.arange(10), 25 + np.arange(10)])
    ld = (nHq + 2 * nKv) * hd
    f32, f16, i32 = np.float32, np.float16, np.int32
    files = dict(table=rng.permutation(pages)[:B * width].reshape(B, width).astype(i32), qkv=rng.standard_normal((T, ld)).astype(f32), qw=rng.uniform(0.5, 1.5, hd).astype(f16),
                 kw=rng.uniform(0.5, 1.5, hd).astype(f16), seq=seq.astype(i32), pos=pos.astype(i32), rot=(pos + 3).astype(i32), lens=np.array([40, 35, 35], i32),
                 starts=np.array([0, 3], i32), shared=np.array([25], i32), x=rng.standard_normal((B, K)).astype(f32), idx=np.array([3, -1, 0], i32),
                 a=(0.1 * rng.standard_normal((n, r, K))).astype(f16), b=rng.standard_normal((n, N, r)).astype(f16), scale=rng.uniform(1, 2, n).astype(f32),
                 y=rng.standard_normal((B, N)).astype(f32), logits=(3 * rng.standard_normal((B, V))).astype(f32), ids=np.array([5, 5002, -1], i32))
    for name, a in files.items():
        np.ascontiguousarray(a).tofile(os.path.join(d, name))
    json.dump(dict(s, files=sorted(files)), open(os.path.join(d, "spec.json"), "w"))
    done = subprocess.run([NODE, os.path.join(ROOT, "tests", "js", "run_serve.js"), d], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True, timeout=100)
    assert done.returncode == 0, done.stdout

    g = {k: ctx.upload(a) for k, a in files.items()}
    rows = page * pages * nKv
    pool = [ctx.zeros(rows * hd), ctx.zeros(rows * hd // 8), ctx.zeros(rows * hd), ctx.zeros(rows * hd // 8)]
    qr, o = ctx.zeros(T * nHq * hd * 4), ctx.zeros(B * nHq * hd * 4)
    k, v = g["qkv"].at(nHq * hd * 4), g["qkv"].at((nHq + nKv) * hd * 4)

    def same(name, buf, nbytes):
        assert np.array_equal(np.fromfile(os.path.join(d, name + ".out"), np.uint8), ctx.download(buf, np.uint8, nbytes)), name

    ctx.call("ti_attn_prep_paged_q8", g["qkv"], k, v, g["qw"], g["kw"], qr, *pool, g["table"], g["seq"], g["pos"], g["rot"], T, B, nHq, nKv, hd, page, pages, width, ld, ld, THETA, EPS)
    for name, buf, nbytes in (("qr", qr, T * nHq * hd * 4), ("kq", pool[0], rows * hd), ("ks", pool[1], rows * hd // 8), ("vq", pool[2], rows * hd)):
        same(name, buf, nbytes)
    ctx.call("ti_attn_shared_q8", qr, *pool, g["table"], g["lens"], g["starts"], g["shared"], o, B, P, nHq, nKv, hd, page, pages, width)
    same("o", o, B * nHq * hd * 4)
    ctx.call("ti_attn_prep_paged_q8", None, k, v, None, None, None, *pool, g["table"], g["seq"], g["pos"], None, T, B, 0, nKv, hd, page, pages, width, ld, ld, THETA, EPS)
    same("kq2", pool[0], rows * hd)
    ctx.call("ti_lora_add", g["x"], g["idx"], g["a"], g["b"], g["scale"], g["y"], B, K, N, r, n, 0, 0, 0)
    same("y", g["y"], B * N * 4)
    out = [ctx.zeros(B * 4 * m) for m in (1, 1, 1, top, top)]
    ctx.call("ti_logprobs", g["logits"], g["ids"], *out, B, V, 0, top)
    for name, buf in zip(("lp", "entropy", "rank", "topIds", "topLp"), out):
        same(name, buf, buf.nbytes)
    same("only", out[0], B * 4)
    assert "top" in open(os.path.join(d, "refused.out")).read()


def test_two_contexts_at_once(ctx):
    """Steps of two batches on two contexts' streams, neither waiting for the other: the bits of each alone."""
    rng = np.random.default_rng(8)
    other = abi.Ctx(0)
    steps, alone, outs = [], [], []
    for c, B, starts, shared in ((ctx, 8, [0, 4, 7], [37, 90]), (other, 5, [0, 5, 5], [60, 9])):
        st = Step(c, rng, B, 2)
        lens = rng.integers(91, 180, B).astype(np.int32)
        table = np.arange(B * st.width, dtype=np.int32).reshape(B, st.width)
        new = dict(x=rng.standard_normal((B, st.H)).astype(np.float32), idx=rng.integers(-1, st.n, B), ids=rng.integers(0, st.V, B), pos=lens - 1, rot=lens - 1, lens=lens, starts=starts,
                   shared=shared, table=table)
        for name, a in new.items():
            c.write(st.ins[name], np.ascontiguousarray(a, np.float32 if name == "x" else np.int32))
        rows = st.pages * st.page * st.nKv
        for b, a in zip(st.pool, (rng.integers(-127, 128, rows * st.hd).astype(np.int8), rng.uniform(0.5, 2, rows * st.hd // 32).astype(np.float32)) * 2):
            c.write(b, a)
        u = st.outs()
        st.run(u)
        alone.append({k: c.download(b, np.uint32, b.nbytes // 4) for k, b in u.items()})
        steps.append(st)
        outs.append([st.outs() for _ in range(10)])
    for i in range(10):
        for st, o in zip(steps, outs):
            st.run(o[i])
    for st, o, want in zip(steps, outs, alone):
        for u in o:
            for k, b in u.items():
                assert np.array_equal(st.ctx.download(b, np.uint32, b.nbytes // 4), want[k]), k
    other.close()
