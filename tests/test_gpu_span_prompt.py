"""Whole prompts under a window: enough rows that each wave takes two tiles of 16, with ragged ends, against 64 bits on a sample of tokens,
and in full against the same prompt in chunks, which take one tile a wave."""
import numpy as np
import pytest

import span_norm as norm
import span_ref as ref
from tabinfer_amd import abi

pytestmark = pytest.mark.gpu
CHUNK = 150                                  # tokens: fewer rows than any switch

# T, pos0, nHq, nKv, hd, window, sinks. Two tiles a wave need a workgroup of 128 rows for every CU of a KV head's share: 320 and
# more here, so that a device of a few more CUs takes them too. The rows behind the last whole 128, a KV head: 2, 80, 40, 52, 112, 20
PROMPTS = [(2561, 0, 16, 8, 128, 300, 4), (5200, 33, 8, 8, 128, 77, 0), (2600, 517, 16, 16, 64, 1000, 65), (1700, 100, 25, 5, 96, 33, 3),
           (1100, 7, 40, 2, 32, 500, 20), (4100, 3, 40, 8, 64, 1, 1), (2700, 64, 16, 16, 96, 700, 0), (2600, 900, 16, 16, 32, 129, 40)]


@pytest.fixture(scope="module")
def ctx():
    c = abi.Ctx(0)
    yield c
    c.close()


def sample(rng, T, G):
    """Tokens of the first and last rows, of those on either side of some workgroups' edges and tiles, and a few more."""
    rows = np.array([0, 15, 16, 31, 32, 127, 128, 129, 255, 256, 1024, 1023])
    last = G * T - 1
    rows = np.concatenate([rows, last - rows[:7], last // 128 * 128 - np.arange(3)])
    return np.unique(np.concatenate([rows[(rows >= 0) & (rows <= last)] // G, rng.integers(0, T, 12)]))


def run(ctx, q, cache, T, pos0, nHq, nKv, hd, window, sinks, shift=0):
    """Outputs of the call, and of the same one in chunks; shift: queries and outputs that many floats off their alignment."""
    dq = ctx.upload(np.concatenate([np.zeros(shift, np.float32), q.ravel()]))
    whole, parts = (ctx.upload(np.full(q.size + 64, np.nan, np.float32)) for _ in range(2))
    dev = [ctx.upload(a) for a in cache]
    at = 4 * shift
    ctx.call("ti_attn_window_q8", dq.at(at), *dev, whole.at(at), T, pos0, nHq, nKv, hd, window, sinks)
    for t in range(0, T, CHUNK):
        n, off = min(CHUNK, T - t), at + 4 * t * nHq * hd
        ctx.call("ti_attn_window_q8", dq.at(off), *dev, parts.at(off), n, pos0 + t, nHq, nKv, hd, window, sinks)
    out = []
    for b in (whole, parts):
        a = ctx.download(b, np.float32, q.size + 64)
        assert np.all(np.isnan(a[:shift])) and np.all(np.isnan(a[shift + q.size:]))
        out.append(a[shift:shift + q.size].reshape(q.shape))
    for b in dev + [dq, whole, parts]:
        b.free()
    return out


def check(q, cache, got, parts, pos0, window, sinks, tokens):
    kc, ks, vc, vs = cache
    S = len(kc)
    seen = ref.visible(pos0 + tokens, np.arange(S), window, sinks)
    # the keys that some sampled token sees
    any_ = seen.any(0)
    K, V = ref.values(kc[any_], ks[any_]), ref.values(vc[any_], vs[any_])
    want, _, tol, _ = norm.attend(q[tokens], K, V, seen[:, any_])
    assert norm.off(got[tokens], want) <= tol
    elem = ref.attend(q[tokens], K, V, seen[:, any_])[1]
    assert np.all(np.abs(got[tokens] - want) <= elem)
    # both are within the bound of the truth
    assert np.all(np.isfinite(parts)) and norm.off(got, parts.astype(np.float64)) <= 2.1 * tol


@pytest.mark.parametrize("T,pos0,nHq,nKv,hd,window,sinks", PROMPTS)
def test_whole_prompts(ctx, T, pos0, nHq, nKv, hd, window, sinks):
    rng = np.random.default_rng(T + hd)
    G = nHq // nKv
    assert nKv * -(-G * T // 128) >= 320 > nKv * -(-G * CHUNK // 128)
    q, cache = rng.standard_normal((T, nHq, hd)).astype(np.float32), ref.cache(rng, pos0 + T, nKv, hd)
    got, parts = run(ctx, q, cache, T, pos0, nHq, nKv, hd, window, sinks, shift=T % 4)
    check(q, cache, got, parts, pos0, window, sinks, sample(rng, T, G))


def test_a_prompt_without_a_window(ctx):
    """Every key before it is seen, 3000 tokens behind 1111 cached ones; sampled tokens, whose rows see up to 4110 keys in one wave."""
    rng = np.random.default_rng(5)
    T, pos0, nHq, nKv, hd = 3000, 1111, 16, 16, 64
    q, cache = rng.standard_normal((T, nHq, hd)).astype(np.float32), ref.cache(rng, pos0 + T, nKv, hd)
    got, parts = run(ctx, q, cache, T, pos0, nHq, nKv, hd, -1, 0)
    check(q, cache, got, parts, pos0, -1, 0, sample(rng, T, 1))


@pytest.mark.parametrize("nHq,nKv,hd", [(16, 8, 128), (25, 5, 96), (16, 16, 64), (40, 2, 32)])
def test_a_prompt_that_sees_nothing(ctx, nHq, nKv, hd):
    rng = np.random.default_rng(hd)
    T = 42000 // nHq
    q, cache = rng.standard_normal((T, nHq, hd)).astype(np.float32), ref.cache(rng, 10 + T, nKv, hd)
    for out in run(ctx, q, cache, T, 10, nHq, nKv, hd, 0, 0):
        assert np.all(out == 0)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("T,pos0,nHq,nKv,hd,window,sinks", [(2561, 600, 16, 8, 128, 90, 5), (1700, 500, 25, 5, 96, 50, 0), (2600, 517, 16, 16, 64, 1, 33),
                                                            (1100, 800, 40, 2, 32, 300, 2)])
def test_masked_keys_of_a_prompt_do_not_count(ctx, T, pos0, nHq, nKv, hd, window, sinks, bad):
    """Scales of keys between the sinks and the first token's window, and of the last key, that only the last token sees."""
    rng = np.random.default_rng(T)
    q, cache = rng.standard_normal((T, nHq, hd)).astype(np.float32), ref.cache(rng, pos0 + T, nKv, hd)
    dirty = [a.copy() for a in cache]
    for i in (1, 3):
        dirty[i][sinks:pos0 + 1 - window] = bad
        dirty[i][-1] = bad
    got, parts = run(ctx, q, dirty, T, pos0, nHq, nKv, hd, window, sinks)
    assert np.all(np.isnan(got[-1])) and np.all(np.isnan(parts[-1]))
    tokens = sample(rng, T, nHq // nKv)
    check(q[:-1], [a[:-1] for a in cache], got[:-1], parts[:-1], pos0, window, sinks, tokens[tokens < T - 1])


def test_a_row_of_a_prompt_is_its_own(ctx):
    """A token whose queries are not finite leaves the others as they are."""
    rng = np.random.default_rng(8)
    T, pos0, nHq, nKv, hd, window, sinks = 2600, 40, 16, 8, 64, 100, 2
    q, cache = rng.standard_normal((T, nHq, hd)).astype(np.float32), ref.cache(rng, pos0 + T, nKv, hd)
    bad = np.array([0, 9, 64, 1300, T - 1])
    dirty = q.copy()
    dirty[bad] = np.nan
    got, parts = run(ctx, dirty, cache, T, pos0, nHq, nKv, hd, window, sinks)
    assert np.all(np.isnan(got[bad]))
    clean = run(ctx, q, cache, T, pos0, nHq, nKv, hd, window, sinks)[0]
    rest = np.setdiff1d(np.arange(T), bad)
    assert np.array_equal(got[rest], clean[rest])
    tokens = np.setdiff1d(sample(rng, T, 2), bad)
    check(q, cache, clean, clean, pos0, window, sinks, tokens)
