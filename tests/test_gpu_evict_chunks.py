"""Evictions on either side of the slot counts where a head's keys no longer fit its registers and go through in chunks."""
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


@pytest.mark.parametrize("kind", ["plain", "equal", "few"])
@pytest.mark.parametrize("n", [2047, 2048, 2049, 8191, 8192, 8193, 16383, 16384, 16385, 32767, 32768, 32769, 49153])
def test_slots_next_to_a_chunk(ctx, n, kind):
    rng = np.random.default_rng(n)
    nKv, hd, sinks, recent = 2, 32, 3, 50
    mass = {"plain": np.exp(3 * rng.standard_normal((n, nKv))), "equal": np.ones((n, nKv)), "few": rng.integers(0, 3, (n, nKv))}[kind].astype(np.float32)
    kc, ks, vc, vs = ref.cache(rng, n, nKv, hd)
    h = np.arange(nKv)[None]
    for keep in (100, n // 2, n - 2):
        dev = [ctx.upload(a) for a in (kc, ks, vc, vs, mass)]
        wo = ctx.zeros(keep * nKv * 4)
        ctx.call("ti_kv_evict_q8", *dev, None, dev[4], wo, n, 0, keep, sinks, recent, n, nKv, hd)
        src, pos = ref.evict(mass, None, n, 0, keep, sinks, recent, n)
        assert np.array_equal(ctx.download(wo, np.int32, keep * nKv).reshape(keep, nKv), pos)
        for d, a in zip(dev, (kc, ks, vc, vs, mass)):
            got = ctx.download(d, a.dtype, a.size).reshape(a.shape)
            assert np.array_equal(got[:keep], a[src, h]) and np.array_equal(got[keep:], a[keep:])
        for x in dev + [wo]:
            x.free()
