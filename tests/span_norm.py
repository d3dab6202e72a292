"""How near the attention over a part of the KV cache has to come to 64 bits in the 2-norm, and attention with a mistake planted
in it, to show that the bound sees the mistake.

The bound is what roundings of f32 leave where they fall independently: each changes its value by U / sqrt(3) of it in the mean
square (U = 2^-24, half a step, uniform). With S^2 the scores' mean square (natural units), n the keys a row sees:

- a score, in units of U: a group's running sum takes at most 64 roundings (32 products with each half of q), of values that
  grow to the group's share of S: 64 NG x (S^2 / NG) / 2 / 3 = 32 S^2 / 3; its scaling and the groups' sum with the factor
  afterwards 7 S^2 / 3; the halves of q leave up to 4 U of an element, 16 S^2 / 3: together 18.4 S^2;
- a weight: its exponent's argument, of up to 4 where weights are large, in units of the natural logarithm 4 ln 2: 2.6; the
  exponential 1 ulp = 2 U: 4 / 3; scaled and multiplied with the V scale: 2 / 3: together 4.6;
- P V: three products a key, a running sum that grows like its square root: 3 n / 2 / 3 = n / 2; the sum of the weights
  below n / 9; and the same again for the partials that are merged, which is far more than they are: 0.7 n in all, where n is
  at most the chain that one wave adds up.

Three times the root of their sum is the bound: a 2-norm over hundreds of elements stays near its mean. Weights alone have no P V.
"""
import numpy as np

import span_ref as ref

U = ref.U


def bound(S2, n):
    return 3 * U * np.sqrt(18.4 * S2 + 4.6 + 0.7 * n)


def scores(q, K, seen):
    """Natural-logarithm scores [T, nHq, n]."""
    T, nHq, hd = q.shape
    G = nHq // K.shape[1]
    out = np.empty((T, nHq, K.shape[0]))
    for h in range(nHq):
        out[:, h] = q[:, h].astype(np.float64) @ K[:, h // G].T / np.sqrt(hd)
    return out


def softmax(s, seen):
    s = np.where(seen[:, None], s, -np.inf)
    m = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(m), m, 0))
    return np.divide(p, p.sum(-1, keepdims=True), out=np.zeros_like(p), where=p.sum(-1, keepdims=True) > 0)


def attend(q, K, V, seen, chain=None):
    """(out [T, nHq, hd], weights [T, nHq, n], bound of out's relative 2-norm error, of the weights')."""
    s = scores(q, K, seen)
    p = softmax(s, seen)
    some = np.broadcast_to(seen[:, None], s.shape)
    S2 = float(np.mean(s[some] ** 2)) if some.any() else 0.0
    n = int(seen.sum(-1).max())
    return mix(p, V), p, bound(S2, min(n, chain or n)), bound(S2, 0)


def mix(p, V):
    G = p.shape[1] // V.shape[1]
    return np.stack([p[:, h] @ V[:, h // G] for h in range(p.shape[1])], 1)


def off(got, want):
    """Relative 2-norm error."""
    return float(np.linalg.norm(np.asarray(got, np.float64) - want) / np.linalg.norm(want))


# ---- planted mistakes --------------------------------------------------------------------------------
def top_bits(x, bits):
    """x cut (not rounded) to its leading bits."""
    m, e = np.frexp(x)
    return np.ldexp(np.trunc(np.ldexp(m, bits)), e - bits)


def two_pieces(p, vc, vs):
    """P V with each weight's product with its V scale cut to two pieces of 8 bits in place of three."""
    hd = vc.shape[-1]
    G = p.shape[1] // vc.shape[1]
    out = np.empty(p.shape[:2] + (hd,))
    for h in range(p.shape[1]):
        for g in range(hd // 32):
            w = top_bits(p[:, h] * vs[:, h // G, g] / 127, 16)
            out[:, h, 32 * g:32 * g + 32] = w @ vc[:, h // G, 32 * g:32 * g + 32].astype(np.float64)
    return out


def upper_half(q):
    """Queries with f16's 11 bits."""
    m, e = np.frexp(q.astype(np.float64))
    return np.ldexp(np.rint(np.ldexp(m, 11)), e - 11)
