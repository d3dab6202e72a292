"""Performance cases of the operators around a served batch's step, through the C ABI's Python binding:

  append   rows of Q, K and V of any sequences: per-head norm and rotation, K and V into the int8 cache in pages, read back as
           the values that the codes stand for
  shared   one new token of each of B sequences in groups that share their first positions, which are read once a group
  lora     rows of a projection's output, each with the low-rank adapter of its request added
  logprobs log probability and rank of given tokens under rows of logits, the rows' entropy and their likeliest tokens

A case is a dict of plain values; `kind` picks the operator. Where `own` is false, run() computes the same in elementary
torch operations. The cache's format: int8 codes of 32-dim groups, one float scale (the group's largest magnitude) each, value =
code * scale / 127; position-major, then KV head, then dim. Head layouts are those of the models the repository is configured
for (16 query heads over 8 of 128; 32 over 8 of 64) and generic ones.
"""
import math

import numpy as np
import torch

own = False
DEV = "cuda"
EPS, THETA = 1e-6, 1e6
VOCAB = 151936
if torch.cuda.is_available():
    torch.backends.cuda.matmul.allow_tf32 = False


def listed():
    q3, lfm = dict(heads=16, kv_heads=8, hd=128), dict(heads=32, kv_heads=8, hd=64)
    return [
        # a generated token of one conversation: bound by latency
        dict(name="append_token", kind="append", T=1, B=1, longest=8191, page=16, merged=False, turn=0, **q3),
        # a token of each of 64 conversations, Q, K and V as one projection leaves them
        dict(name="append_64_merged", kind="append", T=64, B=64, longest=3001, page=64, merged=True, turn=0, **q3),
        # a whole prompt's rows, in a cache that was cut: the rotation's positions lie behind the slots'
        dict(name="append_prompt_2000", kind="append", T=2000, B=1, longest=5003, page=32, merged=True, turn=100000, **lfm),
        # four samples of one short prompt
        dict(name="shared_4_samples_1k", kind="shared", P=1, each=4, prefix=1000, tail=77, even=True, page=16, **q3),
        # 32 conversations behind one long system prompt
        dict(name="shared_32_of_8k", kind="shared", P=1, each=32, prefix=8192, tail=500, even=False, page=64, **q3),
        # six prompts of different lengths, up to 8 samples each
        dict(name="shared_6_groups", kind="shared", P=6, each=8, prefix=6000, tail=1200, even=False, page=32, **lfm),
        # one request's adapter beside a generated token's projection
        dict(name="lora_token", kind="lora", T=1, K=2048, N=2048, r=16, n=8, turns=1, bf16=True, pad=0),
        # a batch of 48 requests over 16 adapters, beside Q, K and V as one projection
        dict(name="lora_48_requests", kind="lora", T=48, K=2048, N=4096, r=32, n=16, turns=48, bf16=False, pad=0),
        # prompts of four requests in one batch, beside the down projection
        dict(name="lora_prompts_1500", kind="lora", T=1500, K=6144, N=2048, r=64, n=6, turns=4, bf16=True, pad=0),
        # a generated token with its five likeliest
        dict(name="logprobs_token", kind="logprobs", T=1, N=VOCAB, top=5, pad=0, masked=0.0),
        # a batch of requests, part of the vocabulary masked away
        dict(name="logprobs_48_masked", kind="logprobs", T=48, N=VOCAB, top=20, pad=64, masked=0.4),
        # a prompt scored
        dict(name="logprobs_prompt_400", kind="logprobs", T=400, N=VOCAB, top=0, pad=0, masked=0.0),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _row(c):
    """Bytes of K and V of one position: codes and scales."""
    return 2 * c["kv_heads"] * (c["hd"] + c["hd"] // 8)


def draw(rng):
    heads, kv_heads = rng.choice([(16, 8), (16, 8), (32, 8), (8, 8), (6, 2), (12, 4), (40, 8), (16, 1), (5, 5)])
    h = dict(heads=heads, kv_heads=kv_heads, hd=rng.choice([32, 64, 96, 128, 128]))
    kind = rng.choice(["append", "shared", "shared", "lora", "lora", "logprobs"])
    if kind == "append":
        T = _log(rng, 1, 2000)
        B = rng.choice([1, T])
        return dict(kind=kind, T=T, B=B, longest=T + _log(rng, 1, 3000) if B == 1 else _log(rng, 1, 3000), page=2 ** rng.randint(0, 8),
                    merged=rng.random() < 0.5, turn=rng.choice([0, _log(rng, 1, 200000)]), **h)
    if kind == "shared":
        P, each = _log(rng, 1, 12), _log(rng, 1, 32)
        room = 40_000_000 // _row(h)                 # positions of K and V that a pass reads, at most
        return dict(kind=kind, P=P, each=each, prefix=_log(rng, 1, min(16000, room // P)), tail=_log(rng, 1, max(1, min(2000, room // (P * each)))),
                    even=rng.random() < 0.4, page=2 ** rng.randint(0, 8), **h)
    if kind == "lora":
        T, r = _log(rng, 1, 1500), rng.choice([1, 8, 16, 16, 32, 64, 128, rng.randint(1, 128)])
        return dict(kind=kind, T=T, K=32 * _log(rng, 1, 192 if T < 800 else 64), N=_log(rng, 1, 6144 if T < 800 else 2048), r=r, n=_log(rng, 1, 32),
                    turns=_log(rng, 1, T), bf16=rng.random() < 0.5, pad=rng.choice([0, 0, rng.randint(1, 9)]))
    N = _log(rng, 50, VOCAB)
    return dict(kind=kind, T=_log(rng, 1, max(1, min(1000, 400 * VOCAB // N))), N=N, top=min(N, rng.choice([0, 1, 5, 20, rng.randint(0, 64)])),
                pad=rng.choice([0, 0, rng.randint(1, 70)]), masked=rng.choice([0.0, 0.0, 0.3, 0.99]))


# ---- inputs ------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 2654435761 % (1 << 62) + 41)
    return g


def _cache(g, rows, c):
    """`rows` cached positions of unit-variance heads: codes [rows][kv_heads][hd], scales [rows][kv_heads][hd / 32]."""
    n = rows * c["kv_heads"] * c["hd"] // 32
    codes, scales = torch.empty(n, 32, dtype=torch.int8, device=DEV), torch.empty(n, device=DEV)
    step = 1 << 20
    for i in range(0, n, step):
        x = torch.randn(min(step, n - i), 32, generator=g, device=DEV)
        s = x.abs().amax(-1)
        codes[i:i + step] = torch.floor(0.5 + 127.0 * (x / s[:, None]).clamp_(-1, 1).double()).to(torch.int8)
        scales[i:i + step] = s
    return codes.view(rows, c["kv_heads"], c["hd"]), scales.view(rows, c["kv_heads"], c["hd"] // 32)


def _groups(c):
    """The groups' sizes and shared lengths, and each sequence's length: alike, or from small to large."""
    P = c["P"]
    sizes = [c["each"] if c["even"] else max(1, round(c["each"] * (p + 1) / P)) for p in range(P)]
    shared = [c["prefix"] if c["even"] else max(1, round(c["prefix"] * (p + 1) / P)) for p in range(P)]
    lens = [shared[p] + (c["tail"] if c["even"] else max(1, round(c["tail"] * ((j + 1) / sizes[p]) ** 2))) for p in range(P) for j in range(sizes[p])]
    return sizes, shared, lens


def prepare(case, seed):
    c, g = case, _gen(seed)
    s = dict(c=c)
    if c["kind"] == "append":
        _prepare_append(s, c, g)
    elif c["kind"] == "shared":
        _prepare_shared(s, c, g)
    elif c["kind"] == "lora":
        dt = torch.bfloat16 if c["bf16"] else torch.float16
        T, K, N, r, n, pad = c["T"], c["K"], c["N"], c["r"], c["n"], c["pad"]
        # rows of a residual stream after its norm, some larger than others
        s["x"] = torch.randn(T, K + 4 * pad, generator=g, device=DEV)[:, :K] * (0.5 + torch.rand(T, 1, generator=g, device=DEV))
        if pad:
            s["x"] = torch.nn.functional.pad(s["x"], (0, 4 * pad))[:, :K]
        s["y"] = torch.randn(T, N + pad, generator=g, device=DEV)[:, :N]
        s["a"] = (torch.randn(n, r, K, generator=g, device=DEV) / math.sqrt(K)).to(dt)
        s["b"] = (0.05 * torch.randn(n, N, r, generator=g, device=DEV)).to(dt)
        s["scale"] = 0.5 + 1.5 * torch.rand(n, generator=g, device=DEV)
        # `turns` requests behind each other, each with an adapter or none
        which = torch.randint(0, n + max(1, n // 8), (c["turns"],), generator=g, device=DEV)
        which[0] = 0
        which = torch.where(which < n, which, -1).int()
        s["idx"] = which[torch.arange(T, device=DEV) * c["turns"] // T].contiguous()
    else:
        T, N = c["T"], c["N"]
        x = torch.empty(T, N + c["pad"], device=DEV)
        x.normal_(generator=g)
        x *= 2.5
        # a few tokens stand out in every row
        like = torch.randint(0, N, (T, 8), generator=g, device=DEV)
        x.scatter_(1, like, 8 + 4 * torch.randn(T, 8, generator=g, device=DEV))
        if c["masked"]:
            x.masked_fill_(torch.rand(T, N + c["pad"], generator=g, device=DEV) < c["masked"], -math.inf)
            x.scatter_(1, like[:, :1], 9.0)
        s["x"] = x[:, :N]
        # the sampled tokens: likely ones and any; a padded row has none
        ids = torch.where(torch.rand(T, generator=g, device=DEV) < 0.7, like[:, 0], torch.randint(0, N, (T,), generator=g, device=DEV))
        s["ids"] = torch.where(torch.rand(T, generator=g, device=DEV) < (0.05 if T > 8 else 0.0), -1, ids).int()
        s["lp"], s["ent"] = torch.empty(T, device=DEV), torch.empty(T, device=DEV)
        s["rank"] = torch.empty(T, dtype=torch.int32, device=DEV)
        s["top_ids"], s["top_lp"] = torch.empty(T, c["top"], dtype=torch.int32, device=DEV), torch.empty(T, c["top"], device=DEV)
    if own:
        _ctx()
    torch.cuda.synchronize()
    return s


def _prepare_append(s, c, g):
    T, H, kv, hd, page = c["T"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    width = (c["longest"] + page - 1) // page
    pages = width * c["B"]
    s["table"] = torch.randperm(pages, generator=g, device=DEV).int().view(c["B"], width)
    s["width"], s["pages"] = width, pages
    if c["B"] == 1:         # a chunk at the end of its sequence
        s["seq"] = torch.zeros(T, dtype=torch.int32, device=DEV)
        s["pos"] = torch.arange(c["longest"] - T, c["longest"], dtype=torch.int32, device=DEV)
    else:                   # one token of each
        s["seq"] = torch.arange(T, dtype=torch.int32, device=DEV)
        s["pos"] = torch.randint(0, c["longest"], (T,), generator=g, device=DEV).int()
    s["rot"] = (s["pos"] + c["turn"]).contiguous() if c["turn"] else None
    if c["merged"]:
        qkv = torch.randn(T, (H + 2 * kv) * hd, generator=g, device=DEV)
        q, k, v = qkv.split([H * hd, kv * hd, kv * hd], 1)
    else:
        q, k, v = (torch.randn(T, n * hd, generator=g, device=DEV) for n in (H, kv, kv))
    s["q"], s["k"], s["v"] = q.view(T, H, hd), k.view(T, kv, hd), v.view(T, kv, hd)
    s["qw"], s["kw"] = ((1.0 + 0.1 * torch.randn(hd, generator=g, device=DEV)).half() for _ in range(2))
    s["qr"] = torch.empty(T, H, hd, device=DEV)
    rows = pages * page
    for a in ("k", "v"):
        s[a + "q"] = torch.zeros(rows, kv, hd, dtype=torch.int8, device=DEV)
        s[a + "s"] = torch.zeros(rows, kv, hd // 32, device=DEV)
        s[a + "_out"] = torch.empty(T, kv, hd, device=DEV)


def _prepare_shared(s, c, g):
    page = c["page"]
    sizes, shared, lens = _groups(c)
    B, width = len(lens), max((n + page - 1) // page for n in lens)
    table, used, b = np.full((B, width), -1, np.int32), 0, 0
    for p, m in enumerate(sizes):       # the pages that hold shared positions alone are one group's, the others a sequence's
        whole = shared[p] // page
        table[b:b + m, :whole] = used + np.arange(whole)
        used += whole
        for j in range(b, b + m):
            more = (lens[j] + page - 1) // page - whole
            table[j, whole:whole + more] = used + np.arange(more)
            used += more
        b += m
    order = torch.randperm(used, generator=g, device=DEV)
    table = torch.from_numpy(table).to(DEV)
    s["table"] = torch.where(table < 0, -1, order[table.clamp(min=0).long()]).int().contiguous()
    s["pages"], s["width"], s["B"] = used, width, B
    s["kq"], s["ks"] = _cache(g, used * page, c)
    s["vq"], s["vs"] = _cache(g, used * page, c)
    up = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
    s["starts"], s["shared"], s["lens"] = up(np.concatenate([[0], np.cumsum(sizes)]).tolist()), up(shared), up(lens)
    # query rows of the size that normalised heads have
    s["q"] = 1.5 * torch.randn(B, c["heads"], c["hd"], generator=g, device=DEV)
    s["out"] = torch.empty_like(s["q"])


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
    if c["kind"] == "append":
        H, kv, hd, T = c["heads"], c["kv_heads"], c["hd"], c["T"]
        cache = (_p(s["kq"]), _p(s["ks"]), _p(s["vq"]), _p(s["vs"]))
        table, seq, pos = _p(s["table"]), _p(s["seq"]), _p(s["pos"])
        pool = (c["page"], s["pages"], s["width"])
        ctx.call("ti_attn_prep_paged_q8", _p(s["q"]), _p(s["k"]), _p(s["v"]), _p(s["qw"]), _p(s["kw"]), _p(s["qr"]), *cache, table, seq, pos,
                 _p(s["rot"]), T, c["B"], H, kv, hd, *pool, s["q"].stride(0), s["k"].stride(0), THETA, EPS)
        ctx.call("ti_kv_read_paged_q8", *cache, table, seq, pos, _p(s["k_out"]), _p(s["v_out"]), T, c["B"], kv, hd, *pool)
        return dict(q=s["qr"], k=s["k_out"], v=s["v_out"])
    if c["kind"] == "shared":
        ctx.call("ti_attn_shared_q8", _p(s["q"]), _p(s["kq"]), _p(s["ks"]), _p(s["vq"]), _p(s["vs"]), _p(s["table"]), _p(s["lens"]), _p(s["starts"]),
                 _p(s["shared"]), _p(s["out"]), s["B"], c["P"], c["heads"], c["kv_heads"], c["hd"], c["page"], s["pages"], s["width"])
        return s["out"]
    if c["kind"] == "lora":
        ctx.call("ti_lora_add", _p(s["x"]), _p(s["idx"]), _p(s["a"]), _p(s["b"]), _p(s["scale"]), _p(s["y"]), c["T"], c["K"], c["N"], c["r"], c["n"],
                 s["x"].stride(0), s["y"].stride(0), int(c["bf16"]))
        return s["y"]
    top = (_p(s["top_ids"]), _p(s["top_lp"])) if c["top"] else (None, None)
    ctx.call("ti_logprobs", _p(s["x"]), _p(s["ids"]), _p(s["lp"]), _p(s["ent"]), _p(s["rank"]), *top, c["T"], c["N"], s["x"].stride(0), c["top"])
    out = dict(lp=s["lp"], ent=s["ent"], rank=s["rank"])
    return dict(out, top_ids=s["top_ids"], top_lp=s["top_lp"]) if c["top"] else out


def _values(codes, scales):
    """Codes [.., hd] and scales [.., hd / 32] as float values."""
    g = codes.float().unflatten(-1, (-1, 32))
    return (g * (scales / 127.0).unsqueeze(-1)).flatten(-2)


# The codes are those of f32 values, each operation rounded in the order that the format's writers keep, so that none lies on the other
# side of a code's border. A quotient or root of doubles rounded to f32 is the f32 operation's.
def _div(a, b):
    return (a.double() / b.double()).float()


def _tree(x):
    """The sum over the last axis, halves on halves."""
    h = x.shape[-1] // 2
    return x if h == 0 else _tree(x[..., :h] + x[..., h:])


def _norm(x, w):
    hd = x.shape[-1]
    sq = torch.nn.functional.pad(x * x, (0, 128 - hd))
    m = _div(_tree(sq), torch.tensor(float(hd), device=DEV)) + torch.tensor(EPS, device=DEV)
    inv = _div(torch.ones_like(m), m.double().sqrt().float())
    return x * inv * w.float()


def _rotate(x, at):
    half = x.shape[-1] // 2
    i = torch.arange(half, device=DEV, dtype=torch.float64)
    angle = at.double()[:, None, None] * float(np.float32(THETA)) ** (-2.0 * i / x.shape[-1])
    c, s = angle.cos().float(), angle.sin().float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c + -b * s, b * c + a * s], -1)


def _write(x, codes, scales, row):
    """Rows x [T, kv, hd] into the cache at `row`, and what they then stand for."""
    g = x.unflatten(-1, (-1, 32))
    m = g.abs().amax(-1).clamp(min=1e-12)
    codes[row] = torch.floor(0.5 + 127.0 * _div(g, m.unsqueeze(-1)).clamp(-1, 1).double()).flatten(-2).to(torch.int8)
    scales[row] = m
    return _values(codes[row], scales[row])


def _plain_append(s):
    c = s["c"]
    pos, at = s["pos"].long(), s["pos"] if s["rot"] is None else s["rot"]
    row = s["table"].long()[s["seq"].long(), pos // c["page"]] * c["page"] + pos % c["page"]
    s["qr"].copy_(_rotate(_norm(s["q"], s["qw"]), at))
    return dict(q=s["qr"], k=_write(_rotate(_norm(s["k"], s["kw"]), at), s["kq"], s["ks"], row), v=_write(s["v"], s["vq"], s["vs"], row))


def _rows(s, b, j):
    """Cache rows of positions j [n, m] of sequences b [n]."""
    page = s["c"]["page"]
    k = (j // page).clamp(max=s["width"] - 1)
    return (s["table"].long()[b].gather(1, k) * page + j % page).clamp(min=0)


def _products(q, k):
    """q [n, r, kv, hd] against k [n, m, kv, hd]: [n, kv, r, m]."""
    n, r, kv, hd = q.shape
    x, y = q.permute(0, 2, 1, 3).reshape(n * kv, r, hd), k.permute(0, 2, 3, 1).reshape(n * kv, hd, -1).contiguous()
    return torch.bmm(x, y).view(n, kv, r, -1)


def _mix(p, v):
    """Weights p [n, kv, r, m] of v [n, m, kv, hd]: [n, r, kv, hd]."""
    n, kv, r, m = p.shape
    o = torch.bmm(p.reshape(n * kv, r, m), v.permute(0, 2, 1, 3).reshape(n * kv, m, -1).contiguous())
    return o.view(n, kv, r, -1).permute(0, 2, 1, 3)


def _plain_shared(s):
    """The groups' rows against the groups' keys, once; every sequence's own; one softmax over both."""
    c = s["c"]
    B, P, H, kv, hd = s["B"], c["P"], c["heads"], c["kv_heads"], c["hd"]
    G, starts, shared, lens = H // kv, s["starts"].long(), s["shared"].long(), s["lens"].long()
    each = c["each"]                                                       # of a group, at most
    group = torch.bucketize(torch.arange(B, device=DEV), starts[1:], right=True)
    place = torch.arange(B, device=DEV) - starts[group]
    member = (starts[:-1, None] + torch.arange(each, device=DEV)).clamp(max=B - 1)         # behind a group's last: any row
    j = torch.arange(c["prefix"], device=DEV).expand(P, -1)
    row = _rows(s, starts[:-1], j)
    q = s["q"] / math.sqrt(hd)
    qg = q[member].view(P, each, kv, G, hd).permute(0, 1, 3, 2, 4).reshape(P, each * G, kv, hd)
    sp = _products(qg, _values(s["kq"][row], s["ks"][row])).view(P, kv, each, G, -1)
    sp = sp.permute(0, 2, 1, 3, 4)[group, place]                           # [B, kv, G, prefix]
    sp = sp.masked_fill((j[:1] >= torch.minimum(shared[group], lens)[:, None])[:, None, None], -math.inf)
    jo = shared[group][:, None] + torch.arange(c["tail"], device=DEV)
    ro = _rows(s, torch.arange(B, device=DEV), jo)
    so = _products(q.view(B, kv, G, hd).permute(0, 2, 1, 3), _values(s["kq"][ro], s["ks"][ro]))
    so = so.masked_fill((jo >= lens[:, None])[:, None, None], -math.inf)
    m = torch.maximum(sp.amax(-1, keepdim=True), so.amax(-1, keepdim=True))
    ep, eo = torch.exp(sp - m), torch.exp(so - m)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    wg = torch.zeros(P, each, kv, G, ep.shape[-1], device=DEV)
    wg[group, place] = ep / total
    og = _mix(wg.permute(0, 2, 1, 3, 4).reshape(P, kv, each * G, -1), _values(s["vq"][row], s["vs"][row])).reshape(P, each, G, kv, hd)
    oo = _mix(eo / total, _values(s["vq"][ro], s["vs"][ro]))
    s["out"].copy_((og[group, place] + oo).permute(0, 2, 1, 3).reshape(B, H, hd))
    return s["out"]


def _plain_lora(s):
    """All adapters' products, those of other requests set to zero."""
    n, r, K = s["a"].shape
    mine = s["idx"][:, None] == torch.arange(n, device=DEV)
    h = (s["x"] @ s["a"].float().view(n * r, K).T).view(-1, n, r)
    h = torch.where(mine[..., None], h * s["scale"][:, None], 0.0)
    s["y"].add_(h.view(-1, n * r) @ s["b"].float().permute(0, 2, 1).reshape(n * r, -1))
    return s["y"]


def _plain_logprobs(s):
    c, x = s["c"], s["x"]
    there = (s["ids"] >= 0) & (s["ids"] < c["N"])
    xi = x.gather(1, s["ids"].long().clamp(0, c["N"] - 1)[:, None])
    m = x.amax(1, keepdim=True)
    z = x - m
    e = z.exp()
    total = e.sum(1, dtype=torch.float64)
    turned = torch.where(e > 0, e * z, 0.0).sum(1, dtype=torch.float64)
    out = dict(lp=torch.where(there, ((xi - m).double()[:, 0] - total.log()).float(), -math.inf), ent=(total.log() - turned / total).float(),
               rank=torch.where(there, (x > xi).sum(1) + 1, 0).int())
    if c["top"]:
        # one whole number a value: larger values first, equal ones by the lower index
        b = torch.where(x == 0, 0.0, x).view(torch.int32).long()
        key = torch.where(b < 0, -(b & 0x7FFFFFFF), b) * (1 << 24) - torch.arange(c["N"], device=DEV)
        top = torch.topk(key, c["top"], dim=1).indices
        out.update(top_ids=top.int(), top_lp=(z.gather(1, top).double() - total.log()[:, None]).float())
    return out


def run(state):
    if own:
        return _own(state)
    return dict(append=_plain_append, shared=_plain_shared, lora=_plain_lora, logprobs=_plain_logprobs)[state["c"]["kind"]](state)


# ---- 64 bits --------------------------------------------------------------------------------------
def _deq64(codes, scales):
    return codes.double() * (scales.double() / 127).repeat_interleave(32, -1)


def _codes64(x):
    """The values that the codes of f32 rows x stand for."""
    g = x.reshape(-1, 32)
    top = np.maximum(np.abs(g).max(1), np.float32(1e-12))[:, None]
    part = np.clip((g / top).astype(np.float32), -1, 1)
    return (np.floor(0.5 + 127 * part.astype(np.float64)) * top.astype(np.float64) / 127).reshape(x.shape)


def _turn64(x, w, at):
    """Norm and rotation of x [T, heads, hd] in 64 bits."""
    hd = x.shape[-1]
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + float(np.float32(EPS))) * w
    z = (y[..., :hd // 2] + 1j * y[..., hd // 2:]) * np.exp(1j * _angles(hd, at))
    return np.concatenate([z.real, z.imag], -1)


def _angles(hd, at):
    return at.astype(np.float64)[:, None, None] * np.float64(np.float32(THETA)) ** (np.arange(hd // 2) * (-2.0 / hd))


def _turn32(x, w, at):
    """The same as the cache's format defines it: every operation rounded to f32, squares added up as a tree of halves of 128."""
    f, hd = np.float32, x.shape[-1]
    t = np.zeros(x.shape[:-1] + (128,), f)
    t[..., :hd] = x * x
    while t.shape[-1] > 1:
        t = t[..., :t.shape[-1] // 2] + t[..., t.shape[-1] // 2:]
    y = x * (f(1) / np.sqrt(t / f(hd) + f(EPS))) * w.astype(f)
    ang = _angles(hd, at)
    co, si = np.cos(ang).astype(f), np.sin(ang).astype(f)
    lo, hi = y[..., :hd // 2], y[..., hd // 2:]
    return np.concatenate([lo * co - hi * si, hi * co + lo * si], -1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    host = lambda t: t.cpu().numpy()  # noqa: E731
    if c["kind"] == "append":
        at = host(s["pos"] if s["rot"] is None else s["rot"])
        q = _turn64(host(s["q"]).astype(np.float64), host(s["qw"]).astype(np.float64), at)
        return dict(q=q, k=_codes64(_turn32(host(s["k"]), host(s["kw"]), at)), v=_codes64(np.ascontiguousarray(host(s["v"]))))
    if c["kind"] == "shared":
        out = torch.zeros(s["B"], c["heads"], c["hd"], dtype=torch.float64, device=DEV)
        table, (sizes, shared, lens), G = host(s["table"]), _groups(c), c["heads"] // c["kv_heads"]
        of = [p for p, m in enumerate(sizes) for _ in range(m)]
        for b, n in enumerate(lens):
            p = of[b]
            j = np.arange(n)
            first = sum(sizes[:p])
            ids = np.where(j < shared[p], table[first, j // c["page"]], table[b, j // c["page"]]).astype(np.int64)
            rows = torch.from_numpy(ids * c["page"] + j % c["page"]).to(DEV)
            k, v = _deq64(s["kq"][rows], s["ks"][rows]), _deq64(s["vq"][rows], s["vs"][rows])
            for hq in range(c["heads"]):
                z = k[:, hq // G] @ s["q"][b, hq].double() * c["hd"] ** -0.5
                w = (z - z.max()).exp()
                out[b, hq] = w @ v[:, hq // G] / w.sum()
        return out
    if c["kind"] == "lora":
        y = s["y"].double()
        for a in range(c["n"]):
            t = (s["idx"] == a).nonzero()[:, 0]
            if len(t):
                y[t] += s["scale"][a].double() * (s["x"][t].double() @ s["a"][a].double().T @ s["b"][a].double().T)
        return y
    res = dict(lp=np.full(c["T"], -np.inf), ent=np.zeros(c["T"]), rank=np.zeros(c["T"], np.int32))
    if c["top"]:
        res.update(top_ids=np.zeros((c["T"], c["top"]), np.int32), top_lp=np.zeros((c["T"], c["top"])))
    x, ids = host(s["x"]), host(s["ids"])
    for t in range(c["T"]):
        r = x[t].astype(np.float64)
        live = r[np.isfinite(r)]
        lse = live.max() + np.log(np.exp(live - live.max()).sum())
        res["ent"][t] = -(np.exp(live - lse) * (live - lse)).sum()
        if 0 <= ids[t] < c["N"]:
            res["lp"][t], res["rank"][t] = r[ids[t]] - lse, 1 + (r > r[ids[t]]).sum()
        if c["top"]:
            near = np.flatnonzero(r >= np.partition(r, c["N"] - c["top"])[c["N"] - c["top"]])
            first = near[np.lexsort((near, -r[near]))][:c["top"]]
            res["top_ids"][t], res["top_lp"][t] = first, r[first] - lse
    return res


# ---- what a pass cannot do without -------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "append":                        # Q, K and V in, Q and the cache's rows out; those in again, values out
        q, kv = 4 * c["heads"] * c["hd"], 8 * c["kv_heads"] * c["hd"]
        return dict(bytes=c["T"] * (2 * q + 2 * kv + 2 * _row(c) + 12), flops=0)
    if c["kind"] == "shared":                        # the groups' shared positions once, every sequence's own
        sizes, shared, lens = _groups(c)
        keys = sum(shared) + sum(lens) - sum(m * n for m, n in zip(sizes, shared))
        return dict(bytes=keys * _row(c) + 8 * len(lens) * c["heads"] * c["hd"] + 4 * (keys // c["page"] + len(lens)), flops=4 * sum(lens) * c["heads"] * c["hd"])
    if c["kind"] == "lora":                          # rows in, the output in and out, the adapters in use
        used = min(c["n"], c["turns"])
        return dict(bytes=4 * c["T"] * (c["K"] + 2 * c["N"] + 1) + 2 * used * c["r"] * (c["K"] + c["N"]), flops=2 * c["T"] * c["r"] * (c["K"] + c["N"]))
    return dict(bytes=c["T"] * (4 * c["N"] + 16 + 8 * c["top"]), flops=4 * c["T"] * c["N"])
