"""The operators over a part of the KV cache on a decoder's own buffers: refused where its positions have a spare code slot, which
they would read other rows of, and right where they have none."""
import numpy as np
import pytest

import span_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
HD, CTX = 64, 64


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def decoder(ctx, kv_heads):
    return abi.Qwen3(ctx, layers=2, hidden=256, intermediate=256, n_heads=kv_heads, n_kv_heads=kv_heads, head_dim=HD, vocab=64, rope_theta=1e6,
                     rms_eps=1e-6, max_ctx=CTX, max_tokens=8)


def calls(cache, nKv, b):
    """Each operator with the cache's four arrays and buffers b of its own."""
    pages = (b, b, b, 1, 1, nKv, HD, 16, 4, 4)          # table, seq, pos; T, B, heads, dims, page, pages, width
    return {
        "ti_attn_window_q8": (b, *cache, b.at(4096), 1, 7, nKv, nKv, HD, 4, 0),
        "ti_attn_mass_q8": (b, *cache, b.at(4096), b.at(8192), 1, 7, nKv, nKv, HD),
        "ti_attn_paged_q8": (b, *cache, b, b, b.at(4096), 1, nKv, nKv, HD, 16, 4, 4, -1, 0),
        "ti_kv_write_paged_q8": (b, b, *cache, *pages),
        "ti_kv_read_paged_q8": (*cache, *pages[:3], b.at(4096), b.at(8192), *pages[3:]),
        "ti_kv_evict_q8": (*cache, b, None, b.at(4096), b.at(8192), 8, 0, 4, 0, 0, 8, nKv, HD),
    }


@pytest.mark.parametrize("kv_heads", [4, 8])
def test_a_cache_with_a_spare_slot_is_refused(ctx, kv_heads):
    m, other = decoder(ctx, kv_heads), decoder(ctx, 2)
    b = ctx.zeros(1 << 16)
    own = [ctx.zeros(CTX * kv_heads * HD) for _ in range(4)]
    assert m.kv_slots() == kv_heads + 1 and other.kv_slots() == 2
    try:
        for layer in range(2):
            kv = m.kv(layer)
            last = CTX * (kv_heads + 1) * HD - 16       # the last bytes of the codes
            for i, at in ((0, 0), (2, 0), (0, last), (2, last)):
                cache = [int(x) for x in own]
                cache[i] = kv[i] + at
                for name, args in calls(cache, kv_heads, b).items():
                    with pytest.raises(abi.TIError, match="%d code slots" % (kv_heads + 1)) as e:
                        ctx.call(name, *args)
                    assert e.value.code == abi.TI_ERR_INVALID and name in str(e.value)
    finally:
        m.close()
        other.close()
        for x in own + [b]:
            x.free()


def test_a_cache_without_one_is_a_cache(ctx):
    """Two KV heads: the decoder's rows, written by it, as the window sees them; and again in the next decoder's memory."""
    rng = np.random.default_rng(0)
    for _ in range(3):
        big, m = decoder(ctx, 8), decoder(ctx, 2)
        big.close()                                      # its memory is anyone's from here on
        kc, ks, vc, vs = ref.cache(rng, CTX, 2, HD)
        for d, a in zip(m.kv(1), (kc, ks, vc, vs)):
            ctx.write(d, a)
        q = rng.standard_normal((1, 2, HD)).astype(np.float32)
        dq, o = ctx.upload(q), ctx.zeros(q.nbytes)
        ctx.call("ti_attn_window_q8", dq, *m.kv(1), o, 1, CTX - 1, 2, 2, HD, 20, 3)
        want, tol, _, _ = ref.attend(q, ref.values(kc, ks), ref.values(vc, vs), ref.visible([CTX - 1], np.arange(CTX), 20, 3))
        assert np.all(np.abs(ctx.download(o, np.float32, q.size).reshape(q.shape) - want) <= tol)
        m.close()
        own = [ctx.zeros(CTX * 8 * HD) for _ in range(4)]
        ctx.call("ti_attn_window_q8", dq, *own, o, 1, CTX - 1, 2, 2, HD, 20, 3)
        ctx.sync()
        for x in own + [dq, o]:
            x.free()


def test_a_decoder_is_destroyed_once(ctx):
    m = decoder(ctx, 4)
    h = m.h
    m.close()
    assert abi.lib().ti_qwen3_destroy(ctx.h, h) == abi.TI_ERR_INVALID
    assert b"no such decoder" in abi.lib().ti_last_error()
