"""The attention operators around the KV cache, as cases that can be timed and compared.

  rope   norms of queries and keys for each head and the position rotation in one pass
         (either layout, part of the head, scaled for long contexts), on views of a fused
         projection: a prompt's tokens, or one token for each request;
  attn   attention of a tree of drafted tokens (one token and a chain are trees too) over a
         cache in one piece or in pages, grouped query heads, with the attention weight that
         each cached position received added to the cache's running sums;
  evict  eviction from such a cache: the first positions, the newest ones and the ones with the
         largest accumulated weight stay, and keys, values and sums are compacted.

Where `own` is false `run` is the plain form: elementary torch operations in 32 bits, rounded
once at the end.  Where it is true `run` calls the framework.  `exact` is the definition in 64 bits.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ---------------------------------------------------------------- the cases

def rope_case(name, **kw):
    c = dict(op="rope", T=1, hq=32, hk=8, d=128, rot=128, layout="half", scaling="none", factor=1.0, theta=10000.0,
             norm=True, zero=False, pos="run", pos0=0, dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def attn_case(name, **kw):
    c = dict(op="attn", B=1, n=1, hq=32, hk=8, d=128, L=1024, ragged=False, page=0, tree="chain", weights=False,
             dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def evict_case(name, **kw):
    c = dict(op="evict", B=1, hk=8, d=128, L=4096, ragged=False, page=0, budget=2048, sinks=4, recent=256, dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of the small model (9 query and 3 key heads of 64), no norms: latency alone
        rope_case("rope token", T=1, hq=9, hk=3, d=64, rot=64, norm=False, pos0=517),
        # a long prompt with normed heads of 128, the frequencies stretched for a long context
        rope_case("rope prompt", T=16384, hq=32, hk=8, theta=1e6, scaling="yarn", factor=4.0, pos0=0),
        # heads of 256 with a quarter rotated in pairs, weights around zero, an odd chunk far into a context
        rope_case("rope partial chunk", T=4099, hq=16, hk=2, d=256, rot=64, layout="interleaved", theta=1e7, zero=True,
                  pos0=120011, dtype="fp16"),
        # one token of the small model over a short cache: latency alone
        attn_case("attn token short", hq=9, hk=3, d=64, L=511),
        # one token over a very long cache, the sums that eviction reads kept
        attn_case("attn token long", L=131072, weights=True),
        # a serving batch: one token each, lengths all different, pages of 16 positions
        attn_case("attn batch pages16", B=32, L=16000, ragged=True, page=16),
        # a drafted tree of 26 tokens for one request, sums kept
        attn_case("attn tree one", n=26, L=8191, tree="random", weights=True),
        # drafted trees of 64 tokens for eight requests over pages of 256: arithmetic counts
        attn_case("attn tree batch", B=8, n=64, L=16384, ragged=True, page=256, tree="random"),
        # a chunk of a prompt over what is cached, heads of 256, eight query heads to a key head
        attn_case("attn chunk", n=1023, hq=16, hk=2, d=256, L=6145, dtype="fp16"),
        # a short cache of the small model halved
        evict_case("evict short", hk=3, d=64, L=1025, budget=512, recent=64),
        # one very long cache cut to a quarter
        evict_case("evict long", L=131071, budget=32768, recent=1024),
        # a serving batch in pages of 16, each request cut to its budget if it is over it
        evict_case("evict batch pages16", B=16, L=16384, ragged=True, page=16, budget=4096, sinks=1, recent=333),
    ]


def _log(rng, lo, hi):
    v = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    return v + 1 if v == 3072 else v


def draw(rng):
    op = rng.choice(("rope", "attn", "attn", "evict"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    d = rng.choice((64, 128, 128, 256))
    hk = rng.choice((1, 2, 3, 4, 8))
    if op == "rope":
        dtype = rng.choice(("bf16", "fp16", "fp32"))
        scaling = rng.choice(("none", "linear", "yarn"))
        hq = hk * rng.choice((1, 3, 4))
        return rope_case(None, T=_log(rng, 1, min(8192, (1 << 25) // ((hq + hk) * d))), hq=hq, hk=hk, d=d,
                         rot=d if rng.random() < 0.5 else rng.choice((d // 4, d // 2)),
                         layout=rng.choice(("half", "interleaved")), scaling=scaling,
                         factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)), theta=rng.choice((1e4, 1e6)),
                         norm=rng.random() < 0.7, zero=rng.random() < 0.3, pos=rng.choice(("run", "batch")),
                         pos0=_log(rng, 1, 120000), dtype=dtype)
    page = rng.choice((0, 16, 48, 256))
    if op == "evict":
        B = _log(rng, 1, 16)
        L = _log(rng, 64, 131072 // B)
        budget = max(8, int(L * rng.uniform(0.1, 0.9)))
        return evict_case(None, B=B, hk=hk, d=d, L=L, ragged=rng.random() < 0.5, page=page, budget=budget,
                          sinks=rng.randrange(0, 5), recent=int(budget * rng.uniform(0, 0.5)), dtype=dtype)
    # the score matrix of the plain form, n * heads * length, stays within what the listed cases have
    B = _log(rng, 1, 32)
    tree = rng.choice(("chain", "random", "random"))
    n = 1 if rng.random() < 0.35 else (_log(rng, 2, 64) if tree == "random" else _log(rng, 2, 512))
    g = rng.choice((1, 3, 4, 8))
    L = max(1, min(_log(rng, 16, 131072 // B), (1 << 27) // (B * n * hk * g)))
    return attn_case(None, B=B, n=n, hq=hk * g, hk=hk, d=d, L=L, ragged=rng.random() < 0.5, page=page, tree=tree,
                     weights=rng.random() < 0.4, dtype=dtype)


# ------------------------------------------------- what a case says of itself

def lengths_of(case):
    """Cached positions of each request: all L, or spread from about L / 16 up to L."""
    B, L = case["B"], case["L"]
    if not case["ragged"]:
        return [L] * B
    r = random.Random(1000003 * B + L)
    out = [max(1, int(L * r.uniform(0.06, 1.0))) for _ in range(B)]
    out[r.randrange(B)] = L
    return out


def frequencies(case):
    """Radians per position of each rotated pair, and the factor on the rotated part, in 64 bits."""
    r, theta = case["rot"], case["theta"]
    f = [theta ** (-2.0 * i / r) for i in range(r // 2)]
    if case["scaling"] == "linear":
        return [x / case["factor"] for x in f], 1.0
    if case["scaling"] == "yarn":
        def at(turns):
            return r * math.log(8192 / (turns * 2 * math.pi)) / (2 * math.log(theta))

        lo, hi = max(math.floor(at(32.0)), 0), min(math.ceil(at(1.0)), r - 1)
        ramp = [min(max((i - lo) / max(hi - lo, 0.001), 0.0), 1.0) for i in range(r // 2)]
        return [x / case["factor"] * t + x * (1 - t) for x, t in zip(f, ramp)], 0.1 * math.log(case["factor"]) + 1.0
    return f, 1.0


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "rope":
        n = case["T"] * (case["hq"] + case["hk"]) * case["d"]
        return {"bytes": 2 * n * e + 8 * case["T"], "flops": 8 * n}
    lens, d, hk = lengths_of(case), case["d"], case["hk"]
    if case["op"] == "attn":
        n, hq = case["n"], case["hq"]
        seen = sum(n * x + (n * (n + 1) // 2 if case["tree"] == "chain" else n) for x in lens)
        b = sum(2 * x * hk * d * e for x in lens) + case["B"] * n * (2 * hq + 2 * hk) * d * e
        if case["weights"]:
            b += sum(2 * 4 * hk * (x + n) for x in lens)
        return {"bytes": b + 4 * case["B"] * n * hq, "flops": 4 * d * hq * seen}
    kept = [min(x, case["budget"]) for x in lens]
    return {"bytes": hk * sum(4 * x + k * (2 * 2 * d * e + 2 * 4) for x, k in zip(lens, kept)), "flops": 4 * hk * sum(lens)}


# ------------------------------------------------------------------ the inputs

def _tree(B, n, kind, seed):
    """parents[b][i] < i, or -1: a chain, or drafts that branch off one of the last few tokens."""
    if kind == "chain":
        return [[i - 1 for i in range(n)] for _ in range(B)]
    r = random.Random(seed)
    return [[-1 if i == 0 else r.randrange(max(-1, i - 9), i) for i in range(n)] for _ in range(B)]


def _cache(case, g, scale):
    """Keys and values of the requests, in one piece (B, heads, L, d), or in pages (N, heads, page, d) that a table names."""
    B, hk, d, L, page = case["B"], case["hk"], case["d"], case["L"], case["page"]
    t = DTYPES[case["dtype"]]
    if not page:
        shape, table = (B, hk, L, d), None
    else:
        per = -(-L // page)
        shape = (B * per, hk, page, d)
        table = torch.randperm(B * per, device="cuda", generator=g).reshape(B, per).to(torch.int32)
    k = (torch.randn(shape, device="cuda", generator=g) * scale[:, None, None]).to(t)
    v = torch.randn(shape, device="cuda", generator=g).to(t)
    return k, v, table


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = DTYPES[case["dtype"]]
    hk, d = case["hk"], case["d"]
    s = {"case": case}
    if case["op"] == "rope":
        T, hq, r = case["T"], case["hq"], case["rot"]
        qkv = torch.randn((T, hq + 2 * hk, d), device="cuda", generator=g).to(t)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hk]
        s["qw"] = s["kw"] = None
        if case["norm"]:
            one = 0.0 if case["zero"] else 1.0
            s["qw"], s["kw"] = ((one + 0.2 * torch.randn(d, device="cuda", generator=g)).to(t) for _ in range(2))
        if case["pos"] == "run":
            s["pos"] = torch.arange(case["pos0"], case["pos0"] + T, device="cuda")
        else:
            s["pos"] = torch.randint(0, case["pos0"] + 1, (T,), device="cuda", generator=g)
        f, s["factor"] = frequencies(case)
        s["f"] = torch.tensor(f, dtype=torch.float64, device="cuda")
        # turns per position, as the whole number of 2^-64ths: position times this wraps to the angle's fraction
        turns = [round(x / (2 * math.pi) * 2 ** 64) % 2 ** 64 for x in f]
        s["turns"] = torch.tensor([x - 2 ** 64 if x >= 2 ** 63 else x for x in turns], dtype=torch.int64, device="cuda")
        if own:
            from voom_b200.runtime import rotary

            scaling = {"none": None, "linear": {"rope_type": "linear", "factor": case["factor"]},
                       "yarn": {"rope_type": "yarn", "factor": case["factor"],
                                "original_max_position_embeddings": 8192}}[case["scaling"]]
            s["rotary"] = rotary.Rotary(d, rot_dim=r, theta=case["theta"], layout=case["layout"], scaling=scaling,
                                        device="cuda")
        return s
    scale = 0.5 + 2.0 * torch.rand(hk, device="cuda", generator=g)
    s["k"], s["v"], s["table"] = _cache(case, g, scale)
    s["host_lengths"] = lengths_of(case)
    s["len"] = torch.tensor(s["host_lengths"], dtype=torch.int32, device="cuda")
    B, L = case["B"], case["L"]
    if case["op"] == "attn":
        n, hq = case["n"], case["hq"]
        qkv = torch.randn((B, n, hq + 2 * hk, d), device="cuda", generator=g)
        qkv[:, :, hq:hq + hk] *= scale[:, None]
        qkv = qkv.to(t)
        s["q"], s["kn"], s["vn"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk], qkv[:, :, hq + hk:]
        s["parents"] = torch.tensor(_tree(B, n, case["tree"], seed), dtype=torch.int32, device="cuda")
        s["sums"] = torch.rand((B, hk, L + n), device="cuda", generator=g) if case["weights"] else None
    else:
        # sums of attention weight: heavy-tailed, some positions never attended, equal values among them
        w = torch.exp(2.0 * torch.randn((B, hk, L), device="cuda", generator=g))
        w = torch.round(w * 1024.0) / 1024.0
        s["sums"] = torch.where(torch.rand((B, hk, L), device="cuda", generator=g) < 0.1, torch.zeros_like(w), w)
    if own:
        from voom_b200.runtime import kv_attention as kva

        if s["table"] is None:
            s["view"] = kva.KVView.contiguous(s["k"], s["v"], s["len"], max_len=max(s["host_lengths"]))
        else:
            s["view"] = kva.KVView.pool(s["k"], s["v"], s["table"], s["len"], max_len=max(s["host_lengths"]))
        if case["op"] == "attn":
            s["tree"] = kva.DraftTree.chain(B, n, "cuda") if case["tree"] == "chain" else kva.DraftTree(s["parents"])
    return s


# -------------------------------------------------------------- the plain form

def _plain_rope(s):
    c = s["case"]
    r = c["rot"]
    h = r // 2
    # the low bits of the product are the fraction of a turn
    angle = (s["pos"][:, None] * s["turns"]).to(torch.float32) * (2.0 * math.pi / 2.0 ** 64)
    cos, sin = (torch.cos(angle) * s["factor"])[:, None], (torch.sin(angle) * s["factor"])[:, None]

    def one(x, w):
        x = x.to(torch.float32)
        if w is not None:
            w = w.to(torch.float32)
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + w if c["zero"] else w)
        a, b = (x[..., :h], x[..., h:r]) if c["layout"] == "half" else (x[..., 0:r:2], x[..., 1:r:2])
        a, b = a * cos - b * sin, a * sin + b * cos
        turned = torch.cat((a, b), -1) if c["layout"] == "half" else torch.stack((a, b), -1).flatten(-2)
        return torch.cat((turned, x[..., r:]), -1).to(DTYPES[c["dtype"]])

    return {"q": one(s["q"], s["qw"]), "k": one(s["k"], s["kw"])}


def _whole(x, table):
    """The cache in one piece: (B, heads, positions, d)."""
    if table is None:
        return x
    B, per = table.shape
    N, hk, page, d = x.shape
    return x[table.reshape(-1).long()].reshape(B, per, hk, page, d).transpose(1, 2).reshape(B, hk, per * page, d)


def _ancestors(parents):
    """seen[b, i, j]: token j is token i or one of its ancestors; the parents' steps are doubled until all are in."""
    B, n = parents.shape
    step = torch.zeros((B, n, n + 1), device=parents.device)
    step.scatter_(2, torch.where(parents < 0, n, parents).long()[..., None], 1.0)
    step = step[..., :n]
    seen = torch.eye(n, device=parents.device) + step
    for _ in range(max(1, n - 1).bit_length()):
        seen = ((seen @ seen) > 0).to(torch.float32)
    return seen > 0


def _plain_attn(s):
    c = s["case"]
    B, n, hq, hk, d = c["B"], c["n"], c["hq"], c["hk"], c["d"]
    g = hq // hk
    t = DTYPES[c["dtype"]]
    k = torch.cat((_whole(s["k"], s["table"])[:, :, :c["L"]], s["kn"].transpose(1, 2)), 2).to(torch.float32)
    v = torch.cat((_whole(s["v"], s["table"])[:, :, :c["L"]], s["vn"].transpose(1, 2)), 2).to(torch.float32)
    q = s["q"].to(torch.float32).reshape(B, n, hk, g, d).permute(0, 2, 1, 3, 4).reshape(B, hk, n * g, d)
    x = (q @ k.transpose(2, 3)).reshape(B, hk, n, g, -1) * (1.0 / math.sqrt(d))
    cached = torch.arange(c["L"], device=x.device) < s["len"][:, None]
    if c["tree"] == "chain":
        tree = torch.ones((n, n), dtype=torch.bool, device=x.device).tril().expand(B, n, n)
    else:
        tree = _ancestors(s["parents"])
    see = torch.cat((cached[:, None].expand(B, n, c["L"]), tree), 2)[:, None, :, None]
    x = torch.where(see, x, torch.full_like(x[..., :1], -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    p = p / total
    out = (p.reshape(B, hk, n * g, -1) @ v).reshape(B, hk, n, g, d).permute(0, 2, 1, 3, 4).reshape(B, n, hq, d).to(t)
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(B, n, hq)
    if s["sums"] is None:
        return {"out": out, "lse": lse}
    # the new tokens' sums stand right behind each request's cached positions
    got = p.sum((2, 3))
    at = torch.arange(c["L"] + n, device=x.device)
    at = torch.where(at < s["len"][:, None], at, at + (c["L"] - s["len"][:, None])).clamp(max=c["L"] + n - 1)
    inside = torch.arange(c["L"] + n, device=x.device) < s["len"][:, None] + n
    got = got.gather(2, at[:, None].expand(B, hk, -1))
    s["sums"] += torch.where(inside[:, None], got, torch.zeros_like(got))
    return {"out": out, "lse": lse, "sums": s["sums"]}


def _plain_evict(s):
    c = s["case"]
    B, hk, d, L = c["B"], c["hk"], c["d"], c["L"]
    keep = min(c["budget"], L)
    at = torch.arange(L, device="cuda")
    n = s["len"][:, None]
    forced = (at < c["sinks"]) | (at >= n - c["recent"])
    key = torch.where(forced[:, None], torch.full_like(s["sums"], math.inf), s["sums"])
    key = torch.where((at < n)[:, None], key, torch.full_like(key, -math.inf))
    index = torch.sort(key, dim=2, descending=True, stable=True)[1][..., :keep]
    lengths = torch.clamp(s["len"], max=c["budget"])
    unused = (torch.arange(keep, device="cuda") >= lengths[:, None])[:, None]
    index = torch.sort(torch.where(unused, L, index), dim=2)[0]
    unused = index >= L
    row = torch.where(unused, 0, index)

    def pick(x):
        x = _whole(x, s["table"]).gather(2, row[..., None].expand(B, hk, keep, d))
        return torch.where(unused[..., None], torch.zeros_like(x), x)

    sums = torch.where(unused, torch.zeros_like(s["sums"][..., :keep]), s["sums"].gather(2, row))
    pad = c["budget"] - keep
    index = torch.where(unused, -1, index).to(torch.int32)
    f = torch.nn.functional.pad
    return {"k": f(pick(s["k"]), (0, 0, 0, pad)), "v": f(pick(s["v"]), (0, 0, 0, pad)), "sums": f(sums, (0, pad)),
            "index": f(index, (0, pad), value=-1), "lengths": lengths}


# ------------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    if not own:
        return {"rope": _plain_rope, "attn": _plain_attn, "evict": _plain_evict}[c["op"]](s)
    if c["op"] == "rope":
        from voom_b200.runtime import rotary

        q, k = rotary.qk_norm_rope(s["q"], s["k"], s["pos"], s["rotary"], q_weight=s["qw"], k_weight=s["kw"], eps=EPS,
                                   zero_centered=c["zero"])
        return {"q": q, "k": k}
    from voom_b200.runtime import kv_attention as kva

    if c["op"] == "attn":
        out, lse = kva.tree_attention(s["q"], s["kn"], s["vn"], s["tree"], s["view"], weights=s["sums"], return_lse=True)
        return {"out": out, "lse": lse} if s["sums"] is None else {"out": out, "lse": lse, "sums": s["sums"]}
    e = kva.kv_evict(s["view"], s["sums"], budget=c["budget"], sinks=c["sinks"], recent=c["recent"])
    return {"k": e.k, "v": e.v, "sums": e.weights, "index": e.index, "lengths": e.lengths}


# ------------------------------------------------------ the definition, 64 bits

def _exact_rope(c, s):
    T, r = c["T"], c["rot"]
    pos = s["pos"].double()
    out = {}
    for name, w in (("q", s["qw"]), ("k", s["kw"])):
        x = s[name].double()
        if w is not None:
            gain = w.double() + (1.0 if c["zero"] else 0.0)
            x = x / torch.sqrt(x.pow(2).sum(-1, keepdim=True) / c["d"] + EPS) * gain
        y = x.clone()
        for i in range(r // 2):  # the pairs, as complex numbers, one at a time
            a, b = (i, i + r // 2) if c["layout"] == "half" else (2 * i, 2 * i + 1)
            z = torch.complex(x[..., a], x[..., b]) * torch.polar(torch.full_like(pos, s["factor"]), pos * s["f"][i])[:, None]
            y[..., a], y[..., b] = z.real, z.imag
        out[name] = y
    return out


def _exact_attn(c, s):
    B, n, hq, hk, d, L = c["B"], c["n"], c["hq"], c["hk"], c["d"], c["L"]
    g = hq // hk
    out = torch.zeros((B, n, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((B, n, hq), dtype=torch.float64, device="cuda")
    sums = None if s["sums"] is None else s["sums"].double()
    parents = _tree(B, n, c["tree"], s["seed"])
    for b, x in enumerate(s["host_lengths"]):
        see = torch.zeros((n, x + n), dtype=torch.bool)
        see[:, :x] = True
        for i in range(n):  # a token sees what its parent sees, and itself
            if parents[b][i] >= 0:
                see[i, x:] = see[parents[b][i], x:]
            see[i, x + i] = True
        see = see.cuda()
        for h in range(hk):
            if s["table"] is None:
                k, v = s["k"][b, h, :x], s["v"][b, h, :x]
            else:
                pages = s["table"][b].long()
                k, v = (y[pages, h].reshape(-1, d)[:x] for y in (s["k"], s["v"]))
            k, v = torch.cat((k, s["kn"][b, :, h])).double(), torch.cat((v, s["vn"][b, :, h])).double()
            for j in range(h * g, h * g + g):
                z = (s["q"][b, :, j].double() @ k.T / math.sqrt(d)).masked_fill(~see, -math.inf)
                lse[b, :, j] = torch.logsumexp(z, 1)
                p = torch.exp(z - lse[b, :, j, None])
                out[b, :, j] = p @ v
                if sums is not None:
                    sums[b, h, :x + n] += p.sum(0)
    return {"out": out, "lse": lse} if sums is None else {"out": out, "lse": lse, "sums": sums}


def exact(case, seed):
    s = prepare(case, seed)
    s["seed"] = seed
    if case["op"] == "rope":
        return _exact_rope(case, s)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    return None  # what stays is copied, not computed
