"""The partials of few-row attention joined a whole row a workgroup, as where a batch has as many rows as the device has CUs: one partial,
a few and hundreds of a sequence, and none that sees anything."""
import numpy as np
import pytest

import span_norm as norm
import span_ref as ref
from span_cases import CHAIN
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
# partials: one a 32 keys of a sequence at most; eight a group of threads and round are 64, 80 and 128 of 128, 96 and 64 dims
LENS = [12000, 0, 1, 33, 700, 64, 5000, 31, 300, -5, 97]


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


# heads of a KV head on either side of what fits a column a 32-dim group
@pytest.mark.parametrize("B,nHq,nKv,hd,window,sinks", [(40, 8, 4, 64, -1, 0), (40, 10, 1, 64, -1, 0), (22, 16, 8, 128, -1, 0), (32, 10, 2, 128, -1, 0), (40, 8, 4, 96, -1, 0),
                                                       (32, 12, 2, 96, -1, 0), (66, 5, 5, 96, 900, 40), (44, 8, 2, 128, 250, 3), (320, 1, 1, 64, 0, 70),
                                                       (40, 8, 8, 32, -1, 0)])
@pytest.mark.parametrize("page", [16, 64])
def test_batches_of_many_rows(ctx, B, nHq, nKv, hd, window, sinks, page):
    rng = np.random.default_rng(B + hd)
    assert B * nHq >= 320
    lens = np.array((LENS * B)[:B], np.int32)
    lens[len(LENS):] = np.minimum(lens[len(LENS):], 400)                    # the long ones once
    need = (np.maximum(lens, 0) + page - 1) // page
    width, pages = int(need.max()), int(need.sum()) + 2
    ids, table, at = rng.permutation(pages).astype(np.int32), np.full((B, width), -1, np.int32), 0
    for b, n in enumerate(need):
        table[b, :n] = ids[at:at + n]
        at += n
    q, (kc, ks, vc, vs) = rng.standard_normal((B, nHq, hd)).astype(np.float32), ref.cache(rng, pages * page, nKv, hd)
    dev = [ctx.upload(a) for a in (q, kc, ks, vc, vs, table, lens)]
    o = ctx.upload(np.full(q.size + 64, np.nan, np.float32))
    ctx.call("ti_attn_paged_q8", *dev, o, B, nHq, nKv, hd, page, pages, width, window, sinks)
    got = ctx.download(o, np.float32, q.size + 64)
    for x in dev + [o]:
        x.free()
    assert np.all(np.isnan(got[q.size:]))
    got = got[:q.size].reshape(q.shape)
    for b, n in enumerate(lens):
        if n <= 0:
            assert np.all(got[b] == 0)
            continue
        j = np.arange(n)
        rows = table[b, j // page].astype(np.int64) * page + j % page
        K, V, seen = ref.values(kc[rows], ks[rows]), ref.values(vc[rows], vs[rows]), ref.visible([n - 1], j, window, sinks)
        if not seen.any():
            assert np.all(got[b] == 0)
            continue
        want, tol, _, _ = ref.attend(q[b:b + 1], K, V, seen)
        assert np.all(np.abs(got[b] - want[0]) <= tol[0]), b
        assert norm.off(got[b], want[0]) <= norm.attend(q[b:b + 1], K, V, seen, CHAIN)[2], b


@pytest.mark.parametrize("T,nHq,nKv,hd", [(5, 64, 64, 128), (8, 64, 64, 64), (7, 60, 60, 96), (3, 128 // 2, 32, 96), (8, 48, 48, 32)])
def test_a_few_tokens_of_many_heads(ctx, T, nHq, nKv, hd):
    """A short chunk with a row for every CU, under a window that reaches far and one that cuts a block."""
    rng = np.random.default_rng(T + hd)
    pos0 = 3000
    q, cache = rng.standard_normal((T, nHq, hd)).astype(np.float32), ref.cache(rng, pos0 + T, nKv, hd)
    dev = [ctx.upload(a) for a in (q,) + cache]
    K, V = ref.values(*cache[:2]), ref.values(*cache[2:])
    for window, sinks in ((-1, 0), (1000, 45), (13, 2), (0, 0)):
        o = ctx.upload(np.full(q.size + 64, np.nan, np.float32))
        ctx.call("ti_attn_window_q8", *dev, o, T, pos0, nHq, nKv, hd, window, sinks)
        got = ctx.download(o, np.float32, q.size + 64)
        o.free()
        assert np.all(np.isnan(got[q.size:]))
        got = got[:q.size].reshape(q.shape)
        seen = ref.visible(pos0 + np.arange(T), np.arange(pos0 + T), window, sinks)
        if not seen.any():
            assert np.all(got == 0)
            continue
        want, tol, _, _ = ref.attend(q, K, V, seen)
        assert np.all(np.abs(got - want) <= tol), window
        assert norm.off(got, want) <= norm.attend(q, K, V, seen, CHAIN)[2], window
    for x in dev:
        x.free()
