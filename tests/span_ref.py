"""64-bit references of the attention over a part of the int8 KV cache: which keys a query sees, softmax attention over
them with the error that f32 arithmetic may leave, and a cache's eviction."""
import numpy as np

U = 2.0 ** -24                                   # half a step of f32, relative


def visible(p, j, window, sinks):
    """Which keys j the queries at positions p see."""
    p, j = np.asarray(p)[:, None], np.asarray(j)[None]
    ok = j <= p
    return ok if window < 0 else ok & ((j > p - window) | (j < sinks))


def cache(rng, n, nKv, hd, wide=False):
    """Codes and scales of n positions; wide: V scales over six decades."""
    kc, vc = (rng.integers(-127, 128, (n, nKv, hd)).astype(np.int8) for _ in range(2))
    ks, vs = (rng.uniform(0.5, 3.0, (n, nKv, hd // 32)).astype(np.float32) for _ in range(2))
    if wide:
        vs *= (10.0 ** rng.uniform(-3, 3, vs.shape)).astype(np.float32)
    return kc, ks, vc, vs


def values(codes, scales):
    with np.errstate(invalid="ignore"):                 # 0 * inf of a key that nobody sees
        return codes.astype(np.float64) * np.repeat(scales.astype(np.float64) / 127, 32, -1)


def attend(q, K, V, seen):
    """q [T, nHq, hd] over K, V [n, nKv, hd] where seen [T, n]: (out, tolerance, weights, their relative error).

    A score is a sum of hd products in f32: 32 a group, at most 32 roundings of the running sum, the groups' sums scaled
    and added with 8 more, whatever the order: 40 U of sum |q k| (an f16 hi + lo split of q is off by 2^-22 of
    each product, 4 U). Scaling and the difference to the maximum add 4 U. So 48 U = ds, on either side of the softmax.
    A weight's exponential and its product with the V scale: 2^-20. The sums over n keys, and their rescalings by
    the running maximum once in 32: 2 n U on either side."""
    T, nHq, hd = q.shape
    n, nKv = K.shape[:2]
    G = nHq // nKv
    out, tol = np.zeros((T, nHq, hd)), np.zeros((T, nHq, hd))
    w, rel = np.zeros((T, nHq, n)), np.zeros((T, nHq))
    for h in range(nHq):
        k, v, x = K[:, h // G], V[:, h // G], q[:, h].astype(np.float64)
        s = np.where(seen, x @ np.where(np.isfinite(k), k, 0).T / np.sqrt(hd), -np.inf)
        m = s.max(-1, keepdims=True)
        p = np.exp(s - np.where(np.isfinite(m), m, 0))
        l = p.sum(-1, keepdims=True)
        p = np.divide(p, l, out=np.zeros_like(p), where=l > 0)
        z = np.where(np.isfinite(v), v, 0)
        ds = 48 * U * np.where(seen, np.abs(x) @ np.abs(np.where(np.isfinite(k), k, 0)).T / np.sqrt(hd), 0).max(-1)
        out[:, h], w[:, h] = p @ z, p
        rel[:, h] = 2 * ds + 2.0 ** -20 + 4 * n * U
        tol[:, h] = rel[:, h][:, None] * (p @ np.abs(z))
    return out, tol, w, rel


def evict(mass, where, n, known, keep, sinks, recent, nxt):
    """(source slot of each kept slot, positions they hold): [min(keep, n)][nKv] each."""
    nKv, kept = mass.shape[1], min(keep, n)
    src, pos = np.zeros((kept, nKv), np.int64), np.zeros((kept, nKv), np.int32)
    for h in range(nKv):
        at = np.array([where[i, h] if i < known else nxt - (n - i) for i in range(n)])
        m = np.where(np.isnan(mass[:n, h]), -np.inf, mass[:n, h].astype(np.float64))
        guarded = (at < sinks) | (at >= nxt - recent)
        # protected first (lower slot), then larger mass (lower slot); NaN after -inf
        order = np.lexsort((np.arange(n), np.where(guarded, 0, np.isnan(mass[:n, h])), np.where(guarded, 0, -m), ~guarded))
        stay = np.zeros(n, bool)
        stay[order[:kept]] = True
        src[:, h] = np.arange(kept)
        src[~stay[:kept], h] = kept + np.flatnonzero(stay[kept:])
        pos[:, h] = at[src[:, h]]
    return src, pos
