"""ti_attn_prep_paged_q8 and ti_attn_prep_q8 on the same rows at near and far positions: the same operations on angles of 64 bits that differ by their
last bits (tests/serve_ref.py derives the tolerance of either against 64 bits)."""
import numpy as np
import pytest

import serve_ref as ref
from tabinfer_amd import abi
from test_gpu_prep_paged import new_pool

pytestmark = pytest.mark.gpu
EPS = 1e-6
# A frequency is off by 2^-52 of itself on either side (one ulp of a power), the angle by its rounding too; both sides together
ANGLE = 2 * 1.5 * 2.0 ** -52


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


@pytest.mark.parametrize("theta", [1e4, 1e6])
@pytest.mark.parametrize("nHq,nKv,hd", [(16, 2, 128), (6, 1, 96), (8, 2, 64), (4, 1, 32)])
def test_as_the_single_token_call(ctx, nHq, nKv, hd, theta):
    rng = np.random.default_rng(hd)
    pos = np.array([0, 1, 899, 4095, 9999, 10 ** 5 - 1, 123457, 399999, 654321, 10 ** 6], np.int32)
    T, cap = len(pos), 10 ** 6 + 1
    q, k, v = (rng.standard_normal((T, n, hd)).astype(np.float32) for n in (nHq, nKv, nKv))
    qw, kw = ((1 + 0.2 * rng.standard_normal(hd)).astype(np.float16) for _ in range(2))
    dq, dk, dv, dqw, dkw, dp = [ctx.upload(a) for a in (q, k, v, qw, kw, pos)]
    a, b, qr, out = new_pool(ctx, cap, nKv, hd), new_pool(ctx, cap, nKv, hd), ctx.zeros(q.nbytes), ctx.zeros(q.nbytes)
    for t in range(T):
        ctx.call("ti_attn_prep_q8", dq.at(t * q[0].nbytes), dk.at(t * k[0].nbytes), dv.at(t * v[0].nbytes), dqw, dkw, qr.at(t * q[0].nbytes), *a, nHq, nKv, hd,
                 int(pos[t]), theta, EPS)
    ctx.call("ti_attn_prep_paged_q8", dq, dk, dv, dqw, dkw, out, *b, None, None, dp, None, T, 1, nHq, nKv, hd, 1, cap, 0, 0, 0, theta, EPS)
    one, many = (ctx.download(o, np.float32, q.size).reshape(q.shape) for o in (qr, out))

    def terms(x, w):                                       # of the rotation, in size: what a cosine's or sine's change is multiplied by
        y = np.abs(x.astype(np.float64) / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + EPS) * w.astype(np.float64))
        half = y[..., :hd // 2] + y[..., hd // 2:]
        return np.concatenate([half, half], -1)
    # a cosine's and a sine's rounding turned on one side: 2 U each of terms up to y; then the products' and the sum's own
    slack = (6 * ref.U + ANGLE * pos[:, None, None]) * terms(q, qw)
    assert np.array_equal(one[pos < 10 ** 4], many[pos < 10 ** 4]) and np.all(np.abs(one.astype(np.float64) - many) <= slack)
    assert np.count_nonzero(one != many) <= 1e-3 * one.size
    off = 0
    for t in range(T):
        rows = [[ctx.download(p, np.int8 if i % 2 == 0 else np.float32, nKv * hd // (1 if i % 2 == 0 else 32), int(pos[t]) * p.nbytes // cap) for i, p in enumerate(x)] for x in (a, b)]
        (kc, ks, vc, vs), (kc2, ks2, vc2, vs2) = rows
        assert np.array_equal(vc, vc2) and np.array_equal(vs, vs2)
        if pos[t] < 10 ** 4:
            assert np.array_equal(kc, kc2) and np.array_equal(ks, ks2)
        g = terms(k[t], kw).reshape(-1, 32).max(-1)
        assert np.all(np.abs(ks.astype(np.float64) - ks2) <= (6 * ref.U + ANGLE * pos[t]) * g)
        d = np.abs(kc.astype(int) - kc2)
        assert d.max() <= 1
        off += np.count_nonzero(d)
    assert off <= 1e-3 * k.size + 1
    for x in a + b + [dq, dk, dv, dqw, dkw, dp, qr, out]:
        x.free()
