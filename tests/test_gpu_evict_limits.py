"""The largest evictions that the header promises, n * nKv = 16 million with half of the slots kept: each row carries its slot's
number, so what the kept slots hold says where it came from."""
import numpy as np
import pytest

from tabinfer_amd import abi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("n,nKv", [(16_000_000, 1), (2_000_000, 8), (250_000, 64)])
def test_as_many_slots_as_fit(n, nKv, in_place):
    rng = np.random.default_rng(nKv)
    hd, keep, sinks, recent = 32, n // 2, 4, 1000
    slot = np.broadcast_to(np.arange(n, dtype=np.uint32)[:, None], (n, nKv))
    mass = rng.integers(0, 5000, (n, nKv)).astype(np.float32)           # many equal ones
    codes = np.zeros((n, nKv, 8), np.uint32)
    codes[..., 3], codes[..., 6] = slot, ~slot
    src = np.zeros((keep, nKv), np.uint32)
    for h in range(nKv):
        key = mass[:, h].copy()
        key[:sinks] = key[n - recent:] = np.inf
        last = np.partition(key, n - keep)[n - keep]
        stay = key > last
        stay[np.flatnonzero(key == last)[:keep - int(stay.sum())]] = True
        src[:, h] = np.arange(keep)
        src[~stay[:keep], h] = keep + np.flatnonzero(stay[keep:])
    with abi.Ctx(0) as ctx:
        kq, vq = ctx.upload(codes), ctx.upload(codes[..., ::-1])
        ks, vs = ctx.upload(slot.astype(np.float32)), ctx.upload(-slot.astype(np.float32))
        dm = ctx.upload(mass)
        mo, wo = (dm if in_place else ctx.zeros(4 * keep * nKv)), ctx.zeros(4 * keep * nKv)
        ctx.call("ti_kv_evict_q8", kq, ks, vq, vs, dm, None, mo, wo, n, 0, keep, sinks, recent, n, nKv, hd)
        count = keep * nKv
        assert np.array_equal(ctx.download(wo, np.uint32, count).reshape(keep, nKv), src)
        assert np.array_equal(ctx.download(mo, np.float32, count).reshape(keep, nKv), np.take_along_axis(mass, src.astype(np.int64), 0))
        assert np.array_equal(ctx.download(ks, np.float32, count).reshape(keep, nKv), src.astype(np.float32))
        assert np.array_equal(ctx.download(vs, np.float32, count).reshape(keep, nKv), -src.astype(np.float32))
        k, v = (ctx.download(b, np.uint32, 8 * count).reshape(keep, nKv, 8) for b in (kq, vq))
        for got, at in ((k, (3, 6)), (v, (4, 1))):
            assert np.array_equal(got[..., at[0]], src) and np.array_equal(got[..., at[1]], ~src)
            got[..., at] = 0
            assert not got.any()
        for b in {id(x): x for x in (kq, vq, ks, vs, dm, mo, wo)}.values():
            b.free()
