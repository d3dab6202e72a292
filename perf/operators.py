"""Performance cases of the operators that bound and share the int8 KV cache, through the C ABI's Python binding:

  window   T queries of one sequence over its cache, a sliding window and the first tokens (sinks) visible
  paged    one new token of each of B sequences over a cache in pages
  write    T rows of K and V into the pages, read back as the values that the codes stand for
  mass     causal attention that also adds up the weight each cached key receives
  evict    a cache cut to the keys of most accumulated weight, read back as values

A case is a dict of plain values; `kind` picks the operator. Where `own` is false, run() computes the same in
elementary torch operations. The cache's format: int8 codes of 32-dim groups, one float scale (the group's largest
magnitude) each, value = code * scale / 127; position-major, then KV head, then dim. Head layouts are those of the
models the repository is configured for (16 query heads over 8 of 128; 32 over 8 of 64) and generic ones.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
if torch.cuda.is_available():
    torch.backends.cuda.matmul.allow_tf32 = False


def listed():
    q3, lfm = dict(heads=16, kv_heads=8, hd=128), dict(heads=32, kv_heads=8, hd=64)
    return [
        # a generated token of a long chat that keeps a 4k window and four sinks: bound by latency
        dict(name="window_token_32k", kind="window", T=1, pos0=32101, window=4096, sinks=4, **q3),
        # a whole prompt at once under a 1k window
        dict(name="window_prompt_4k", kind="window", T=4096, pos0=0, window=1024, sinks=4, **q3),
        # one ragged chunk of a long prompt, four query heads a KV head
        dict(name="window_chunk_250", kind="window", T=250, pos0=7777, window=2000, sinks=16, **lfm),
        # one conversation in small pages
        dict(name="paged_1_of_8k", kind="paged", B=1, longest=8191, even=True, page=16, window=-1, sinks=0, **q3),
        # a served batch of conversations of very different lengths
        dict(name="paged_32_ragged", kind="paged", B=32, longest=8192, even=False, page=64, window=-1, sinks=0, **q3),
        # a batch under a window: pages outside it are gone from the table
        dict(name="paged_8_window", kind="paged", B=8, longest=32000, even=False, page=32, window=2048, sinks=16, **lfm),
        # a prompt's chunk into pages; a token of each of 64 conversations
        dict(name="write_chunk_256", kind="write", T=256, B=1, longest=1300, page=16, **q3),
        dict(name="write_64_tokens", kind="write", T=64, B=64, longest=3000, page=64, **q3),
        # a generated token whose attention weights are added up; a prompt's last chunk
        dict(name="mass_token_4k", kind="mass", T=1, pos0=4095, **q3),
        dict(name="mass_chunk_256", kind="mass", T=256, pos0=1792, **q3),
        # a full cache that makes room for one token; a prompt cut to a quarter
        dict(name="evict_one_of_4k", kind="evict", n=4097, known=4096, keep=4096, sinks=4, recent=512, **q3),
        dict(name="evict_16k_to_4k", kind="evict", n=16384, known=0, keep=4096, sinks=4, recent=1024, **q3),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _row(c):
    """Bytes of K and V of one position: codes and scales."""
    return 2 * c["kv_heads"] * (c["hd"] + c["hd"] // 8)


def draw(rng):
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (8, 8), (6, 2), (12, 4), (40, 8), (16, 1), (5, 5)])
    hd = rng.choice([32, 64, 96, 128, 128])
    h = dict(heads=heads, kv_heads=kv_heads, hd=hd)
    kind = rng.choice(["window", "window", "paged", "paged", "paged", "write", "mass", "mass", "evict"])
    if kind == "window":
        # a chunk's cost is its rows times what they see: at most the whole prompt's above
        T = _log(rng, 1, 4096)
        window = min(_log(rng, 1, 8192), max(1, 4096 * 1024 * 16 * 128 // (T * heads * hd)))
        return dict(kind=kind, T=T, pos0=rng.choice([0, _log(rng, 1, 30000)]), window=window, sinks=rng.choice([0, _log(rng, 1, 64)]), **h)
    if kind == "paged":
        B = _log(rng, 1, 64)
        longest = _log(rng, 1, min(32000, 200_000_000 // (B * _row(h))))
        return dict(kind=kind, B=B, longest=longest, even=rng.random() < 0.4, page=2 ** rng.randint(0, 8),
                    window=rng.choice([-1, -1, _log(rng, 1, 4096)]), sinks=rng.choice([0, _log(rng, 1, 64)]), **h)
    if kind == "write":
        T = _log(rng, 1, 1024)
        B = rng.choice([1, T])
        return dict(kind=kind, T=T, B=B, longest=T + _log(rng, 1, 3000) if B == 1 else _log(rng, 1, 3000), page=2 ** rng.randint(0, 8), **h)
    if kind == "mass":
        T = _log(rng, 1, max(1, min(256, 4096 // heads)))
        return dict(kind=kind, T=T, pos0=rng.choice([0, _log(rng, 1, 16000)]), **h)
    n = _log(rng, 2, 32000)
    keep = rng.randint(1, n)
    sinks = rng.randint(0, min(8, keep))
    return dict(kind=kind, n=n, known=rng.choice([0, rng.randint(0, n)]), keep=keep, sinks=sinks, recent=rng.randint(0, keep - sinks), **h)


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 29)
    return g


def _cache(g, rows, c):
    """`rows` cached positions of unit-variance heads: codes [rows][kv_heads][hd], scales [rows][kv_heads][hd / 32]."""
    n = rows * c["kv_heads"] * c["hd"] // 32
    codes, scales = torch.empty(n, 32, dtype=torch.int8, device=DEV), torch.empty(n, device=DEV)
    step = 1 << 20
    for i in range(0, n, step):
        _quant_into(torch.randn(min(step, n - i), 32, generator=g, device=DEV), codes[i:i + step], scales[i:i + step])
    return codes.view(rows, c["kv_heads"], c["hd"]), scales.view(rows, c["kv_heads"], c["hd"] // 32)


def _quant_into(x, codes, scales):
    s = x.abs().amax(-1).clamp_(min=1e-12)
    codes.copy_(torch.floor(0.5 + 127.0 * (x / s[:, None]).clamp_(-1, 1).double()))
    scales.copy_(s)


def _lens(c):
    """The sequences' lengths: alike, or from short to the longest."""
    B = c["B"]
    return [c["longest"] if c["even"] else max(1, round(c["longest"] * ((b + 1) / B) ** 2)) for b in range(B)]


def _seen(c, length):
    """How many keys the token at length - 1 sees."""
    if c["window"] < 0:
        return length
    return min(length, c["window"] + min(c["sinks"], max(0, length - c["window"])))


def _table(g, c, lens):
    """A table of pages in no order, -1 where no key is seen any more, and how many pages there are."""
    page = c["page"]
    width = max((n + page - 1) // page for n in lens)
    first = torch.arange(width, device=DEV) * page
    L = torch.tensor(lens, device=DEV)[:, None]
    live = first[None] < L
    if c.get("window", -1) >= 0:
        live &= (first[None] + page > L - c["window"]) | (first[None] < c["sinks"])
    pages = int(live.sum())
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    table[live] = torch.randperm(pages, generator=g, device=DEV).int()
    return table, pages, width


def prepare(case, seed):
    c, g = case, _gen(seed)
    kind, h = c["kind"], dict(heads=c["heads"], kv_heads=c["kv_heads"], hd=c["hd"])
    s = dict(c=c)
    if kind in ("window", "mass"):
        S = c["pos0"] + c["T"]
        s["kq"], s["ks"] = _cache(g, S, c)
        s["vq"], s["vs"] = _cache(g, S, c)
        # query rows of the size that normalised heads have
        s["q"] = 1.5 * torch.randn(c["T"], c["heads"], c["hd"], generator=g, device=DEV)
        s["out"] = torch.empty_like(s["q"])
        if kind == "mass":
            s["mass"] = torch.rand(S, c["kv_heads"], generator=g, device=DEV)
    elif kind == "paged":
        lens = _lens(c)
        s["table"], s["pages"], s["width"] = _table(g, c, lens)
        s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
        s["kq"], s["ks"] = _cache(g, s["pages"] * c["page"], c)
        s["vq"], s["vs"] = _cache(g, s["pages"] * c["page"], c)
        s["q"] = 1.5 * torch.randn(c["B"], c["heads"], c["hd"], generator=g, device=DEV)
        s["out"] = torch.empty_like(s["q"])
    elif kind == "write":
        s["table"], s["pages"], s["width"] = _table(g, c, [c["longest"]] * c["B"])
        if c["B"] == 1:     # a chunk at the end of its sequence
            s["seq"] = torch.zeros(c["T"], dtype=torch.int32, device=DEV)
            s["pos"] = torch.arange(c["longest"] - c["T"], c["longest"], dtype=torch.int32, device=DEV)
        else:               # one token of each
            s["seq"] = torch.arange(c["T"], dtype=torch.int32, device=DEV)
            s["pos"] = torch.randint(0, c["longest"], (c["T"],), generator=g, device=DEV).int()
        rows, n = s["pages"] * c["page"], (c["T"], c["kv_heads"], c["hd"])
        for a in ("k", "v"):
            s[a] = torch.randn(*n, generator=g, device=DEV)
            s[a + "_out"] = torch.empty(*n, device=DEV)
            s[a + "q"] = torch.zeros(rows, *n[1:], dtype=torch.int8, device=DEV)
            s[a + "s"] = torch.zeros(rows, n[1], n[2] // 32, device=DEV)
    else:
        n, kv = c["n"], c["kv_heads"]
        s["kq"], s["ks"] = _cache(g, n, c)
        s["vq"], s["vs"] = _cache(g, n, c)
        # what the attention left: weights over many orders of magnitude, some of them none at all
        mass = torch.exp(3 * torch.randn(n, kv, generator=g, device=DEV))
        s["mass"] = torch.where(torch.rand(n, kv, generator=g, device=DEV) < 0.05, torch.zeros_like(mass), mass)
        # the first `known` slots hold earlier positions, each head in an order of its own; the next token's position
        s["next"] = c["n"] + 1000 if c["known"] else c["n"]
        old = s["next"] - (n - c["known"])
        order = [torch.randperm(max(1, old), generator=g, device=DEV)[:c["known"]] for _ in range(kv)]
        s["where"] = torch.stack(order, 1).int().contiguous() if c["known"] else torch.zeros(1, kv, dtype=torch.int32, device=DEV)
        k = min(c["keep"], n)
        s["mass_out"] = torch.empty(k, kv, device=DEV)
        s["where_out"] = torch.empty(k, kv, dtype=torch.int32, device=DEV)
        s["rows"] = torch.arange(k, dtype=torch.int32, device=DEV)
        s["k_out"], s["v_out"] = (torch.empty(k, kv, c["hd"], device=DEV) for _ in range(2))
    s.update(h)
    if own:
        _ctx()
    torch.cuda.synchronize()
    return s


# ---- the operators ------------------------------------------------------------------------------
_CTX = []


def _ctx():
    if not _CTX:
        from tabinfer_amd import abi
        _CTX.append(abi.Ctx(0))
    return _CTX[0]


def _p(t):
    return None if t is None else t.data_ptr()


def _own(s):
    c, ctx = s["c"], _ctx()
    h = (c["heads"], c["kv_heads"], c["hd"])
    cache = tuple(_p(s[a]) for a in ("kq", "ks", "vq", "vs"))
    if c["kind"] == "window":
        ctx.call("ti_attn_window_q8", _p(s["q"]), *cache, _p(s["out"]), c["T"], c["pos0"], *h, c["window"], c["sinks"])
        return s["out"]
    if c["kind"] == "paged":
        ctx.call("ti_attn_paged_q8", _p(s["q"]), *cache, _p(s["table"]), _p(s["lens"]), _p(s["out"]), c["B"], *h, c["page"],
                 s["pages"], s["width"], c["window"], c["sinks"])
        return s["out"]
    if c["kind"] == "write":
        place = (_p(s["table"]), _p(s["seq"]), _p(s["pos"]))
        size = (c["T"], c["B"], c["kv_heads"], c["hd"], c["page"], s["pages"], s["width"])
        ctx.call("ti_kv_write_paged_q8", _p(s["k"]), _p(s["v"]), *cache, *place, *size)
        ctx.call("ti_kv_read_paged_q8", *cache, *place, _p(s["k_out"]), _p(s["v_out"]), *size)
        return dict(k=s["k_out"], v=s["v_out"])
    if c["kind"] == "mass":
        ctx.call("ti_attn_mass_q8", _p(s["q"]), *cache, _p(s["out"]), _p(s["mass"]), c["T"], c["pos0"], *h)
        return dict(out=s["out"], mass=s["mass"])
    k = min(c["keep"], c["n"])
    ctx.call("ti_kv_evict_q8", *cache, _p(s["mass"]), _p(s["where"]) if c["known"] else None, _p(s["mass_out"]), _p(s["where_out"]),
             c["n"], c["known"], c["keep"], c["sinks"], c["recent"], s["next"], c["kv_heads"], c["hd"])
    ctx.call("ti_kv_read_paged_q8", *cache, None, None, _p(s["rows"]), _p(s["k_out"]), _p(s["v_out"]), k, 1, c["kv_heads"], c["hd"],
             1, c["n"], 0)
    return dict(k=s["k_out"], v=s["v_out"], mass=s["mass_out"], where=s["where_out"])


def _values(codes, scales):
    """Codes [.., hd] and scales [.., hd / 32] as float values."""
    g = codes.float().unflatten(-1, (-1, 32))
    return (g * (scales / 127.0).unsqueeze(-1)).flatten(-2)


def _attend(q, k, v, ok, weights=False):
    """q [b, T, heads, hd] over k, v [b, n, kv, hd] where ok [b, T, n]: out like q, and the weights added up over
    queries and a KV head's query heads [b, n, kv]."""
    b, T, heads, hd = q.shape
    kv = k.shape[2]
    G = heads // kv
    x = q.view(b, T, kv, G, hd).permute(0, 2, 3, 1, 4).reshape(b * kv, G * T, hd)
    s = torch.bmm(x, k.permute(0, 2, 3, 1).reshape(b * kv, hd, -1).contiguous()).view(b, kv, G, T, -1) / math.sqrt(hd)
    s = s.masked_fill_(~ok[:, None, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    l = p.sum(-1, keepdim=True)
    p = torch.where(l > 0, p / l, 0.0)
    o = torch.bmm(p.view(b * kv, G * T, -1), v.permute(0, 2, 1, 3).reshape(b * kv, -1, hd).contiguous())
    o = o.view(b, kv, G, T, hd).permute(0, 3, 1, 2, 4).reshape(b, T, heads, hd)
    return (o, p.double().sum((2, 3)).permute(0, 2, 1)) if weights else o


def _visible(p, j, window, sinks):
    ok = j <= p
    return ok if window < 0 else ok & ((j > p - window) | (j < sinks))


def _plain(s):
    c = s["c"]
    if c["kind"] == "window":
        # the keys that any query sees, in order
        S = c["pos0"] + c["T"]
        low = max(0, c["pos0"] + 1 - c["window"]) if c["window"] >= 0 else 0
        first = min(c["sinks"], low)
        j = torch.cat([torch.arange(first, device=DEV), torch.arange(low, S, device=DEV)])
        k, v = _values(s["kq"][j], s["ks"][j])[None], _values(s["vq"][j], s["vs"][j])[None]
        p = torch.arange(c["pos0"], S, device=DEV)[:, None]
        return _attend(s["q"][None], k, v, _visible(p, j[None], c["window"], c["sinks"])[None])[0]
    if c["kind"] == "paged":
        p = s["lens"].long()[:, None] - 1
        # the first `sinks` positions, then each sequence's own last `window`; all of them without a window
        first, last = (0, c["longest"]) if c["window"] < 0 else (c["sinks"], min(c["window"], c["longest"]))
        i = torch.arange(first + last, device=DEV)[None]
        j = torch.where(i < first, i, (i - first + p + 1 - last).clamp(min=first)) if c["window"] >= 0 else i
        ok = (j <= p) & ((i < first) | (i - first + p + 1 - last >= first) | (c["window"] < 0))
        j = torch.minimum(j, p)
        row = s["table"].long().gather(1, j // c["page"]) * c["page"] + j % c["page"]
        row = row.clamp(min=0)
        k, v = _values(s["kq"][row], s["ks"][row]), _values(s["vq"][row], s["vs"][row])
        return _attend(s["q"][:, None], k, v, ok[:, None])[:, 0]
    if c["kind"] == "write":
        pos = s["pos"].long()
        row = s["table"].long()[s["seq"].long(), pos // c["page"]] * c["page"] + pos % c["page"]
        return dict(k=_write(s["k"], s["kq"], s["ks"], row), v=_write(s["v"], s["vq"], s["vs"], row))
    if c["kind"] == "mass":
        S = c["pos0"] + c["T"]
        k, v = _values(s["kq"], s["ks"])[None], _values(s["vq"], s["vs"])[None]
        ok = _visible(torch.arange(c["pos0"], S, device=DEV)[:, None], torch.arange(S, device=DEV)[None], -1, 0)
        out, w = _attend(s["q"][None], k, v, ok[None], weights=True)
        new = torch.arange(S, device=DEV)[:, None] >= c["pos0"]
        s["mass"].copy_((torch.where(new, 0.0, s["mass"].double()) + w[0]).float())
        return dict(out=out[0], mass=s["mass"])
    n, keep = c["n"], min(c["keep"], c["n"])
    slot = torch.arange(n, device=DEV)[:, None].expand(n, c["kv_heads"])
    late = (s["next"] - n + slot).int()
    where = torch.cat([s["where"][:c["known"]], late[c["known"]:]])
    guarded = (where < c["sinks"]) | (where >= s["next"] - c["recent"])
    order = torch.sort(torch.where(guarded, math.inf, s["mass"]), dim=0, descending=True, stable=True).indices
    kept = torch.zeros_like(guarded).scatter_(0, order[:keep], True)
    # the i-th freed slot below keep takes the i-th kept one above it
    hole = ~kept[:keep]
    tail = torch.sort(torch.where(kept & (slot >= keep), slot, n), dim=0).values
    src = torch.where(hole, tail.gather(0, (hole.cumsum(0) - 1).clamp(min=0)), slot[:keep])
    head = torch.arange(c["kv_heads"], device=DEV)[None]
    return dict(k=_values(s["kq"][src, head], s["ks"][src, head]), v=_values(s["vq"][src, head], s["vs"][src, head]),
                mass=s["mass"].gather(0, src), where=where.gather(0, src))


def _write(x, codes, scales, row):
    """Rows x [T, kv, hd] into the cache at `row`, and what they then stand for."""
    g = x.unflatten(-1, (-1, 32))
    m = g.abs().amax(-1).clamp(min=1e-12)
    codes[row] = torch.floor(0.5 + 127.0 * (g / m.unsqueeze(-1)).clamp(-1, 1).double()).flatten(-2).to(torch.int8)
    scales[row] = m
    return _values(codes[row], scales[row])


def run(state):
    return _own(state) if own else _plain(state)


# ---- 64 bits --------------------------------------------------------------------------------------
def _deq64(codes, scales):
    return codes.double() * (scales.double() / 127).repeat_interleave(32, -1)


def _softmax64(q, k, v, seen):
    """One head's rows q [n, hd] over k, v [m, hd], seen [n, m]: outputs and weights in 64 bits."""
    z = (q.double() @ k.T) * k.shape[-1] ** -0.5
    z = torch.where(seen, z, -math.inf)
    e = torch.where(seen, (z - z.amax(-1, keepdim=True)).exp(), 0.0)
    w = torch.nan_to_num(e / e.sum(-1, keepdim=True))
    return w @ v, w


def exact(case, seed):
    c, s = case, prepare(case, seed)
    G = c["heads"] // c["kv_heads"]
    if c["kind"] in ("window", "mass"):
        out = torch.zeros(c["T"], c["heads"], c["hd"], dtype=torch.float64, device=DEV)
        mass = torch.zeros(c["pos0"] + c["T"], c["kv_heads"], dtype=torch.float64, device=DEV)
        if c["kind"] == "mass":
            mass[:c["pos0"]] = s["mass"][:c["pos0"]].double()
        W, sinks = (c["window"], c["sinks"]) if c["kind"] == "window" else (-1, 0)
        for t0 in range(0, c["T"], 512):        # queries in runs, over the part of the cache that they may see
            t1 = min(c["T"], t0 + 512)
            at = c["pos0"] + torch.arange(t0, t1, device=DEV)[:, None]
            lo = 0 if W < 0 else max(0, c["pos0"] + t0 - W + 1)
            rows = sorted(set(range(min(sinks, c["pos0"] + t1))) | set(range(lo, c["pos0"] + t1)))
            rows = torch.tensor(rows, device=DEV)
            behind = at - rows[None]
            seen = behind >= 0
            if W >= 0:
                seen &= (behind < W) | (rows[None] < sinks)
            for hq in range(c["heads"]):
                h = hq // G
                o, w = _softmax64(s["q"][t0:t1, hq], _deq64(s["kq"][rows, h], s["ks"][rows, h]), _deq64(s["vq"][rows, h], s["vs"][rows, h]), seen)
                out[t0:t1, hq] = o
                mass[rows, h] += w.sum(0)
        return out if c["kind"] == "window" else dict(out=out, mass=mass)
    if c["kind"] == "paged":
        out = torch.zeros(c["B"], c["heads"], c["hd"], dtype=torch.float64, device=DEV)
        table = s["table"].cpu().numpy()
        for b, n in enumerate(_lens(c)):
            see = [j for j in range(n) if c["window"] < 0 or j >= n - c["window"] or j < c["sinks"]]
            if not see:
                continue
            see = np.array(see)
            rows = torch.from_numpy(table[b, see // c["page"]].astype(np.int64) * c["page"] + see % c["page"]).to(DEV)
            k, v = _deq64(s["kq"][rows], s["ks"][rows]), _deq64(s["vq"][rows], s["vs"][rows])
            for hq in range(c["heads"]):
                all_ = torch.ones(1, len(see), dtype=torch.bool, device=DEV)
                out[b, hq] = _softmax64(s["q"][b, hq][None], k[:, hq // G], v[:, hq // G], all_)[0][0]
        return out
    if c["kind"] == "write":
        res = {}
        for a in ("k", "v"):
            x = s[a].cpu().numpy().reshape(-1, 32)
            top = np.maximum(np.abs(x).max(1), np.float32(1e-12))[:, None]
            part = np.clip((x / top).astype(np.float32), -1, 1)         # the format takes the quotient in 32 bits
            res[a] = (np.floor(0.5 + 127 * part.astype(np.float64)) * top.astype(np.float64) / 127).reshape(s[a].shape)
        return res
    n, keep, kv = c["n"], min(c["keep"], c["n"]), c["kv_heads"]
    mass, known = s["mass"].cpu().numpy(), s["where"].cpu().numpy()
    k, v = _deq64(s["kq"], s["ks"]).cpu().numpy(), _deq64(s["vq"], s["vs"]).cpu().numpy()
    res = dict(k=np.zeros((keep, kv, c["hd"])), v=np.zeros((keep, kv, c["hd"])), mass=np.zeros((keep, kv)), where=np.zeros((keep, kv), np.int32))
    for h in range(kv):
        at = [int(known[i, h]) if i < c["known"] else s["next"] - n + i for i in range(n)]
        free = [c["sinks"] <= p < s["next"] - c["recent"] for p in at]
        rank = sorted(range(n), key=lambda i: (free[i], -mass[i, h] if free[i] else 0.0, i))
        stay = set(rank[:keep])
        late = iter(sorted(i for i in stay if i >= keep))
        final = [i if i in stay else next(late) for i in range(keep)]
        res["k"][:, h], res["v"][:, h], res["mass"][:, h] = k[final, h], v[final, h], mass[final, h].astype(np.float64)
        res["where"][:, h] = [at[i] for i in final]
    return res


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    c = case
    row = _row(c)
    if c["kind"] in ("window", "mass"):
        T, p0 = c["T"], c["pos0"]
        w = dict(window=c.get("window", -1), sinks=c.get("sinks", 0))
        pairs = sum(_seen(w, p0 + t + 1) for t in range(T))
        keys = _seen(w, p0 + 1) + T - 1 if w["window"] else min(w["sinks"], p0 + T)
        add = 4 * c["kv_heads"] * (2 * p0 + T) if c["kind"] == "mass" else 0
        return dict(bytes=keys * row + 8 * T * c["heads"] * c["hd"] + add, flops=4 * pairs * c["heads"] * c["hd"])
    if c["kind"] == "paged":
        keys = sum(_seen(c, n) for n in _lens(c))
        return dict(bytes=keys * row + 8 * c["B"] * c["heads"] * c["hd"] + 4 * (keys // c["page"] + c["B"]), flops=4 * keys * c["heads"] * c["hd"])
    values = 8 * c["kv_heads"] * c["hd"]                         # K and V of a position as floats
    if c["kind"] == "write":                                     # rows in, the cache's rows out; and in again, values out
        return dict(bytes=c["T"] * (2 * values + 2 * row + 16), flops=0)
    moved = min(c["keep"], c["n"] - c["keep"]) if c["keep"] < c["n"] else 0
    keep = min(c["keep"], c["n"])
    return dict(bytes=8 * c["kv_heads"] * (c["n"] + keep) + 2 * moved * row * keep // max(1, c["n"]) + keep * (row + values), flops=0)
