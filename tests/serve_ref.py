"""64-bit references of the operators around a served batch's step: norm and rotation of heads, the cache's codes of f32 rows, low-rank
adapters, log probabilities; with the errors that f32 arithmetic may leave."""
import numpy as np

U = 2.0 ** -24                                   # half a step of f32, relative


def angles(hd, rot, theta):
    return np.asarray(rot, np.float64)[:, None, None] * np.float64(np.float32(theta)) ** (-2.0 * np.arange(hd // 2) / hd)


def turn(x, w, rot, theta, eps):
    """x [T, heads, hd] normed (w None: not) and rotated: (values, tolerance).

    The squares' sum takes 7 additions and a product, its mean a division, eps an addition, the root and the reciprocal one rounding each, which
    the root halves: (7 + 1 + 1 + 1) / 2 + 2 = 7 U; two products: 9 U of the normed value. Its cosine or sine is rounded, the product and the
    difference too: 12 U of each of the two terms, whose factors are at most 1."""
    x, hd = x.astype(np.float64), x.shape[-1]
    y = x if w is None else x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(eps))) * w.astype(np.float64)
    a, b, t = y[..., :hd // 2], y[..., hd // 2:], angles(hd, rot, theta)
    c, s = np.cos(t), np.sin(t)
    tol = 12 * U * (np.abs(a) + np.abs(b)) + 2.0 ** -140
    return np.concatenate([a * c - b * s, b * c + a * s], -1), np.concatenate([tol, tol], -1)


def turn32(x, w, rot, theta, eps):
    """The same with every operation rounded to f32 in ti_attn_prep_q8's order, angles in 64 bits: what the cache's codes are of."""
    f, hd = np.float32, x.shape[-1]
    y = x
    if w is not None:
        t = np.zeros(x.shape[:-1] + (128,), f)
        t[..., :hd] = x * x
        while t.shape[-1] > 1:
            t = t[..., :t.shape[-1] // 2] + t[..., t.shape[-1] // 2:]
        y = x * (f(1) / np.sqrt(t / f(hd) + f(eps))) * w.astype(f)
    t = angles(hd, rot, theta)
    c, s = np.cos(t).astype(f), np.sin(t).astype(f)
    a, b = y[..., :hd // 2], y[..., hd // 2:]
    return np.concatenate([a * c + -b * s, b * c + a * s], -1)


def codes(x):
    """(codes [.., hd] int8, scales [.., hd / 32], distance of each code's quotient from the border of another) of f32 rows."""
    g = x.reshape(x.shape[:-1] + (x.shape[-1] // 32, 32))
    top = np.maximum(np.abs(g).max(-1), np.float32(1e-12))
    e = 0.5 + 127.0 * np.clip(g / top[..., None], -1, 1).astype(np.float64)
    far = np.abs(e - np.rint(e))
    return np.floor(np.nan_to_num(e)).astype(np.int8).reshape(x.shape), top, far.reshape(x.shape)


def lora(x, y, idx, a, b, scale):
    """(y + s B A x, bound of the 2-norm of its error, tolerance of each value), weights and rows as 64-bit arrays.

    A value of h sums K products of each of an activation's pieces, of y's change r: running sums of f32, each rounding independent, add up to
    U / sqrt(3) of their size, half of the last one's in the mean square: with three pieces sqrt(3 (K + r) / 2) U / sqrt(3); the pieces themselves leave
    2^-22 of an element or 2^-39 of the largest, 4 U; scaling and joining parts 8 roundings. Three times that for the 2-norm. At worst they all add up:
    3 (K + r) + 32 of the sums of magnitudes."""
    d, worst = np.zeros(y.shape), np.zeros(y.shape)
    for t, i in enumerate(idx):
        if 0 <= i < len(a):
            d[t] = scale[i] * (b[i] @ (a[i] @ x[t]))
            worst[t] = abs(scale[i]) * (np.abs(b[i]) @ (np.abs(a[i]) @ np.abs(x[t])))
    K, r = x.shape[1], a.shape[1]
    norm = 3 * U * np.sqrt((K + r) / 2 + 16 + 8 / 3) * np.linalg.norm(d) + U * np.linalg.norm(y + d)
    tol = (3 * (K + r) + 32) * U * worst + 2 * U * np.abs(y + d)
    return y + d, norm, tol


def logprobs(x, ids, top):
    """x [T, N] f32: dict of lp, ent, rank, top_ids, top_lp, and tolerances of lp, ent and top_lp.

    With d = x - M: its rounding and that of d log2 e, U |d| each, the exponential 2 U; a lane adds up N / 256 of them at most, and joins follow:
    lane by lane, wave by wave and part by part, 12 of 4 roundings each: the sum is off by (N / 256 + 56 + 2 E|d|) U, E over the probabilities. ln S
    is off by that and by 2 U of itself, lp by U of x - M and of itself more. u sums e d the same way: (N / 256 + 60) U E|d| + 2 U E d^2."""
    T, N = x.shape
    r = dict(lp=np.full(T, -np.inf), ent=np.zeros(T), rank=np.zeros(T, np.int32), top_ids=np.full((T, top), -1, np.int32), top_lp=np.full((T, top), -np.inf))
    tl, te = np.zeros(T), np.zeros(T)
    for t in range(T):
        v = x[t].astype(np.float64)
        with np.errstate(invalid="ignore", over="ignore", divide="ignore"):
            M = np.nanmax(v) if not np.isnan(v).all() else np.nan
            d = v - M
            e = np.exp(d)
            S = e.sum()
            lse = M + np.log(S)
            p, dd = e / S, np.where(e > 0, d, 0)
            r["ent"][t] = np.log(S) - (p * dd).sum()
            Ed, Ed2 = -(p * dd).sum(), (p * dd * dd).sum()
            tl[t] = (N / 256 + 60 + 2 * Ed) * U + 2 * U * abs(np.log(S))
            te[t] = tl[t] + (N / 256 + 62) * U * (Ed + 1) * 2 + 2 * U * (Ed2 + Ed * Ed)
            there = 0 <= ids[t] < N
            if there:
                r["lp"][t], r["rank"][t] = (v[ids[t]] - M) - np.log(S), 1 + (v > v[ids[t]]).sum()
            ok = np.flatnonzero(~np.isnan(v))
            order = ok[np.lexsort((ok, -v[ok]))][:top]
            r["top_ids"][t, :len(order)] = order
            r["top_lp"][t, :len(order)] = (v[order] - M) - np.log(S)
    with np.errstate(invalid="ignore"):
        lp_tol = tl + 4 * U * np.abs(np.where(np.isfinite(r["lp"]), r["lp"], 0))
        top_tol = tl[:, None] + 4 * U * np.abs(np.where(np.isfinite(r["top_lp"]), r["top_lp"], 0))
    return r, dict(lp=lp_tol, ent=te, top_lp=top_tol)
