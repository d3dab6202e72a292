"""Paged attention of sequences whose length is below zero, the lowest value of its type among them: zeros, and the others
their own results."""
import numpy as np
import pytest

import span_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("window,sinks", [(-1, 0), (20, 3), (0, 2), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("lens", [[-2 ** 31], [-2 ** 31, 45, -2 ** 31 + 1, 0, 64, -1]])
def test_lengths_below_zero_give_zeros(lens, window, sinks):
    rng = np.random.default_rng(len(lens))
    B, nHq, nKv, hd, page, pages, width = len(lens), 8, 4, 64, 16, 30, 4
    table = np.stack([rng.permutation(pages)[:width] for _ in range(B)]).astype(np.int32)
    table[np.array(lens) <= 0] = 2 ** 31 - 1
    q, (kc, ks, vc, vs) = rng.standard_normal((B, nHq, hd)).astype(np.float32), ref.cache(rng, pages * page, nKv, hd)
    with abi.Ctx(0) as ctx:
        dev = [ctx.upload(a) for a in (q, kc, ks, vc, vs, table, np.array(lens, np.int32))]
        o = ctx.upload(np.full(q.size, np.nan, np.float32))
        ctx.call("ti_attn_paged_q8", *dev, o, B, nHq, nKv, hd, page, pages, width, window, sinks)
        got = ctx.download(o, np.float32, q.size).reshape(q.shape)
        for x in dev + [o]:
            x.free()
    for b, n in enumerate(lens):
        if n <= 0:
            assert np.all(got[b] == 0)
            continue
        j = np.arange(n)
        rows = table[b, j // page].astype(np.int64) * page + j % page
        want, tol, _, _ = ref.attend(q[b:b + 1], ref.values(kc[rows], ks[rows]), ref.values(vc[rows], vs[rows]), ref.visible([n - 1], j, window, sinks))
        assert np.all(np.abs(got[b] - want[0]) <= tol[0]), b
