"""Decoding several continuations over a paged KV cache, as cases that can be timed and compared.

  attn     attention over the cache with scores that are capped by a tanh, biased by the distance
           between query and key, and limited to a window of the newest positions;
  beam     the choice of the best continuations of each request over its beams and the vocabulary;
  append   new tokens' keys and values written to their places in the cache;
  fork     rows of a page table become continuations of others: pages are shared, an open page that
           several would write to is copied, fresh pages are handed out, ended rows' pages are freed;
  compact  the pages in use move to the front of the pool.

Where `own` is false `run` is the plain form: elementary torch operations in 32 bits (beam scores in
64: candidates of different beams lie close), rounded once at the end.  Where it is true `run` calls the
framework.  `exact` is the definition in 64 bits.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------- the cases

def attn_case(name, **kw):
    c = dict(op="attn", B=1, n=1, hq=32, hk=8, d=128, L=1024, ragged=False, page=0, tree="chain", cap=0.0, bias=False,
             window=0, dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def beam_case(name, **kw):
    c = dict(op="beam", B=1, beams=4, width=4, V=32000, first=False, dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def append_case(name, **kw):
    c = dict(op="append", B=1, n=1, hk=8, d=128, L=1024, page=16, accept=False, dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def fork_case(name, **kw):
    c = dict(op="fork", B=1, beams=4, hk=8, d=128, L=512, page=16, layers=1, grow=1, dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def compact_case(name, **kw):
    c = dict(op="compact", B=4, hk=8, d=128, L=512, page=16, layers=1, pages=512, dtype="bf16")
    c.update(kw)
    return dict(c, name=name) if name else c


def listed():
    return [
        # one new token of the small model (9 query and 3 key heads of 64) in a layer with a window: latency alone
        attn_case("attn token window", hq=9, hk=3, d=64, L=8191, window=1000, cap=50.0),
        # a serving batch, capped scores, lengths all different, pages of 16 positions: the cache's bytes
        attn_case("attn batch capped pages16", B=32, L=16000, ragged=True, page=16, cap=30.0),
        # a chunk of a prompt over a long cache, biased by distance, capped, windowed: arithmetic counts
        attn_case("attn chunk biased", n=1000, L=8192, cap=50.0, bias=True, window=6000, dtype="fp16"),
        # four beams of one request: latency alone
        beam_case("beam one request", B=1, beams=4, V=49152),
        # a prompt's first choice: one beam alive, twice as many continuations as beams
        beam_case("beam first step", B=8, beams=5, width=10, V=131072, first=True, dtype="fp32"),
        # a serving batch of eight beams, an odd vocabulary
        beam_case("beam batch", B=32, beams=8, width=16, V=200019, dtype="fp16"),
        # one token of one request
        append_case("append token", hk=3, d=64, L=700),
        # prompts' chunks of eight requests
        append_case("append chunks", B=8, n=2047, L=6001, page=64),
        # four beams over a short cache
        fork_case("fork one request", hk=3, d=64, L=701, page=16, layers=4),
        # a serving batch of beams: tables of long rows, open pages of several layers copied
        fork_case("fork batch", B=32, beams=8, L=1999, page=64, layers=2),
        # a small pool with holes
        compact_case("compact small", hk=3, d=64, layers=4),
        # a pool of 1.6 GB that lost half its requests
        compact_case("compact large", B=24, L=6000, page=64, layers=2, pages=3001),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("attn", "attn", "beam", "append", "fork", "compact"))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    d = rng.choice((64, 128, 128, 256))
    hk = rng.choice((1, 2, 3, 4, 8))
    page = rng.choice((16, 48, 64, 256))
    if op == "beam":
        beams = rng.randrange(1, 13)
        B = _log(rng, 1, max(1, 256 // beams))
        V = _log(rng, 500, min(200000, (1 << 25) // (B * beams)))
        return beam_case(None, B=B, beams=beams, width=min(V, rng.randrange(1, 2 * beams + 1)), V=V, first=rng.random() < 0.2,
                         dtype=rng.choice(("bf16", "fp16", "fp32")))
    if op == "append":
        B = _log(rng, 1, 32)
        n = _log(rng, 1, 8192 // B)
        return append_case(None, B=B, n=n, hk=hk, d=d, L=_log(rng, 1, 4000), page=rng.choice((0, page)),
                           accept=rng.random() < 0.4, dtype=dtype)
    if op == "fork":
        beams = rng.randrange(1, 9)
        L, grow = _log(rng, 10, 4000), rng.choice((1, 1, 7, 70))
        B = _log(rng, 1, max(1, min(32, (1 << 26) // ((L + 2 * page + grow) * beams * hk * d))))
        return fork_case(None, B=B, beams=beams, hk=hk, d=d, L=L, page=page, layers=rng.randrange(1, 5), grow=grow, dtype=dtype)
    if op == "compact":
        L = _log(rng, 10, 4000)
        B = _log(rng, 1, max(1, min(32, (1 << 26) // (L * hk * d))))
        return compact_case(None, B=B, hk=hk, d=d, L=L, page=page, layers=rng.randrange(1, 4),
                            pages=int(B * -(-L // page) * rng.uniform(1.0, 2.0)) + 1, dtype=dtype)
    # the score matrix of the plain form, n * heads * length, stays within what the listed cases have
    B = _log(rng, 1, 32)
    tree = rng.choice(("chain", "random"))
    n = 1 if rng.random() < 0.4 else (_log(rng, 2, 64) if tree == "random" else _log(rng, 2, 512))
    g = rng.choice((1, 3, 4, 8))
    L = max(1, min(_log(rng, 16, 131072 // B), (1 << 27) // (B * n * hk * g)))
    kind = rng.randrange(1, 8)  # which of the three, one at least
    return attn_case(None, B=B, n=n, hq=hk * g, hk=hk, d=d, L=L, ragged=rng.random() < 0.5, page=rng.choice((0, page)),
                     tree=tree, cap=rng.choice((15.0, 30.0, 50.0)) if kind & 1 else 0.0, bias=bool(kind & 2),
                     window=_log(rng, 1, 8192) if kind & 4 else 0, dtype=dtype)


# ------------------------------------------------- what a case says of itself

def lengths_of(case):
    """Cached positions of each request: all L, or spread from about L / 16 up to L."""
    B, L = case["B"], case["L"]
    if not case.get("ragged", case["op"] in ("append", "compact")):
        return [L] * B
    r = random.Random(1000003 * B + L)
    out = [max(1, int(L * r.uniform(0.06, 1.0))) for _ in range(B)]
    out[r.randrange(B)] = L
    return out


def accepted(case, seed):
    """The accepted path of each request's new tokens: some of them, in order."""
    r = random.Random(seed)
    return [sorted(r.sample(range(case["n"]), r.randrange(1, case["n"] + 1))) for _ in range(case["B"])]


def slopes_of(case):
    """A head's bias per position of distance: 2^(-8 (h + 1) / heads), in 32 bits."""
    return torch.tensor([2.0 ** (-8.0 * (h + 1) / case["hq"]) for h in range(case["hq"])], dtype=torch.float32)


def work(case):
    e = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "beam":
        n = case["B"] * (1 if case["first"] else case["beams"]) * case["V"]
        return {"bytes": n * e + case["B"] * (4 * case["beams"] + 12 * case["width"]), "flops": 3 * n}
    hk, d = case["hk"], case["d"]
    if op == "append":
        n = sum(map(len, accepted(case, 0))) if case["accept"] else case["B"] * case["n"]
        return {"bytes": 2 * 2 * n * hk * d * e, "flops": n}
    if op == "fork":
        p = fork_plan(case, 0)
        P, row = case["page"], 2 * 2 * case["layers"] * hk * d * e  # bytes that a copied position reads and writes
        used = [-(-x // P) for x in p["lengths"]]
        moved = 0  # positions of open pages that several rows would write to, but for the one that keeps the page
        for r0 in range(0, len(used), case["beams"]):
            rows = range(r0, r0 + case["beams"])
            moved += sum(p["lengths"][r0] % P for r in set(p["parents"][r] for r in rows) - {-1}
                         for _ in range(sum(p["parents"][x] == r for x in rows) - 1))
        return {"bytes": 2 * 4 * sum(used) + 4 * p["pages"] + moved * row, "flops": sum(used)}
    if op == "compact":
        used, B = [-(-x // case["page"]) for x in lengths_of(case)], case["B"]
        moved = sum(used) * (1.0 - sum(used) / case["pages"])  # of as many pages anywhere in the pool
        return {"bytes": int(2 * 2 * moved * case["layers"] * hk * case["page"] * d * e) + 2 * 4 * sum(used) + 4 * case["pages"],
                "flops": case["pages"] + B}
    lens, n, hq, w = lengths_of(case), case["n"], case["hq"], case["window"] or 1 << 62
    read = seen = 0
    for x in lens:
        read += min(x, w - 1)
        if case["tree"] == "chain":
            seen += sum(min(x + i + 1, w) for i in range(n))
        else:
            seen += n * min(x + 1, w)
    b = 2 * read * hk * d * e + case["B"] * n * (2 * hq + 2 * hk) * d * e
    return {"bytes": b + 4 * case["B"] * n * hq, "flops": 4 * d * hq * seen}


# ------------------------------------------------------------------ the inputs

def _tree(B, n, kind, seed):
    """parents[b][i] < i, or -1: a chain, or drafts that branch off one of the last few tokens."""
    if kind == "chain":
        return [[i - 1 for i in range(n)] for _ in range(B)]
    r = random.Random(seed)
    return [[-1 if i == 0 else r.randrange(max(-1, i - 9), i) for i in range(n)] for _ in range(B)]


def fork_plan(case, seed):
    """Tables, lengths and parents of a batch of beams: a request's rows share its prompt's full pages and what
    followed up to where they parted; each parent is drawn, the better beams more often; a few requests have ended."""
    B, beams, P = case["B"], case["beams"], case["page"]
    r, q = random.Random(7 * seed + 3), random.Random(1000003 * B + case["L"])  # q: sizes, the same for every seed
    per = -(-(case["L"] + case["grow"]) // P)
    table, lengths, parents, pages = [], [], [], 0
    for b in range(B):
        n = case["L"] if b == 0 else max(1, int(case["L"] * q.uniform(0.3, 1.0)))
        used = -(-n // P)
        shared = min(used - 1, int(used * q.uniform(0.5, 0.9)))
        common = list(range(pages, pages + shared))
        pages += shared
        for _ in range(beams):
            table.append(common + list(range(pages, pages + used - shared)))
            pages += used - shared
            lengths.append(n)
        ended = b > 0 and r.random() < 0.05
        parents += [-1 if ended else b * beams + min(r.randrange(beams), r.randrange(beams)) for _ in range(beams)]
    pages += B * beams * (2 + case["grow"] // P)
    place = list(range(pages))
    r.shuffle(place)
    return {"table": [[place[x] for x in t] + [-1] * (per - len(t)) for t in table], "lengths": lengths,
            "parents": parents, "pages": pages}


def _pool(case, layers, pages, g):
    t = DTYPES[case["dtype"]]
    shape = (layers, pages, case["hk"], case["page"], case["d"])
    return tuple(torch.randn(shape, device="cuda", generator=g, dtype=t) for _ in range(2))


def _i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(int(seed))
    t = DTYPES[case["dtype"]]
    s = {"case": case}
    if case["op"] == "beam":
        B, beams, V = case["B"], case["beams"], case["V"]
        s["logits"] = (3.0 * torch.randn((B, beams, V), device="cuda", generator=g)).to(t)
        s["scores"] = -5.0 * torch.rand((B, beams), device="cuda", generator=g)
        if case["first"]:
            s["scores"][:, 1:] = -math.inf
        return s
    hk, d, page = case["hk"], case["d"], case["page"]
    if case["op"] == "fork":
        p = fork_plan(case, int(seed))
        s["k"], s["v"] = _pool(case, case["layers"], p["pages"], g)
        s["table"], s["len"], s["parents"] = _i32(p["table"]), _i32(p["lengths"]), _i32(p["parents"])
        return s
    s["host_lengths"] = lens = lengths_of(case)
    s["len"] = _i32(lens)
    B, L = case["B"], case["L"]
    if case["op"] == "compact":
        per, N = -(-L // page), case["pages"]
        s["k"], s["v"] = _pool(case, case["layers"], N, g)
        order = torch.randperm(N, device="cuda", generator=g)[:B * per].to(torch.int32).reshape(B, per)
        used = (s["len"] + page - 1) // page
        s["table"] = torch.where(torch.arange(per, device="cuda") < used[:, None], order, -1)
        return s
    n = case["n"]
    room = L + n if case["op"] == "append" else L
    if page:
        per = -(-room // page)
        shape = (B * per, hk, page, d)
        s["table"] = torch.randperm(B * per, device="cuda", generator=g).reshape(B, per).to(torch.int32)
    else:
        shape, s["table"] = (B, hk, room, d), None
    if case["op"] == "append":
        s["k"], s["v"] = (torch.randn(shape, device="cuda", generator=g, dtype=t) for _ in range(2))
        kv = torch.randn((B, n, 2 * hk, d), device="cuda", generator=g, dtype=t)
        s["kn"], s["vn"] = kv[:, :, :hk], kv[:, :, hk:]
        s["index"] = None
        if case["accept"]:
            s["index"] = _i32([x + [-1] * (n - len(x)) for x in accepted(case, seed)])
    else:
        hq = case["hq"]
        # keys of growing size head by head: flat and sharp softmax, scores well into the cap
        scale = 0.5 + 3.0 * torch.rand(hk, device="cuda", generator=g)
        s["k"] = (torch.randn(shape, device="cuda", generator=g) * scale[:, None, None]).to(t)
        s["v"] = torch.randn(shape, device="cuda", generator=g).to(t)
        qkv = torch.randn((B, n, hq + 2 * hk, d), device="cuda", generator=g)
        qkv[:, :, :hq] *= 2.0
        qkv[:, :, hq:hq + hk] *= scale[:, None]
        qkv = qkv.to(t)
        s["q"], s["kn"], s["vn"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk], qkv[:, :, hq + hk:]
        s["parents"] = _i32(_tree(B, n, case["tree"], seed))
        s["slopes"] = slopes_of(case).cuda() if case["bias"] else None
    if own:
        from voom_b200.runtime import kv_attention as kva

        if s["table"] is None:
            s["view"] = kva.KVView.contiguous(s["k"], s["v"], s["len"], max_len=max(lens))
        else:
            s["view"] = kva.KVView.pool(s["k"], s["v"], s["table"], s["len"], max_len=max(lens))
        if case["op"] == "attn":
            s["tree"] = kva.DraftTree.chain(B, n, "cuda") if case["tree"] == "chain" else kva.DraftTree(s["parents"])
    return s


# -------------------------------------------------------------- the plain form

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
    B, n, hq, hk, d, L = c["B"], c["n"], c["hq"], c["hk"], c["d"], c["L"]
    g = hq // hk
    t = DTYPES[c["dtype"]]
    k = torch.cat((_whole(s["k"], s["table"])[:, :, :L], s["kn"].transpose(1, 2)), 2).to(torch.float32)
    v = torch.cat((_whole(s["v"], s["table"])[:, :, :L], s["vn"].transpose(1, 2)), 2).to(torch.float32)
    q = s["q"].to(torch.float32).reshape(B, n, hk, g, d).permute(0, 2, 1, 3, 4).reshape(B, hk, n * g, d)
    x = (q @ k.transpose(2, 3)).reshape(B, hk, n, g, -1) * (1.0 / math.sqrt(d))
    if c["cap"]:
        x = c["cap"] * torch.tanh(x / c["cap"])
    at = torch.arange(L, device=x.device)
    if c["tree"] == "chain":
        tree = torch.ones((n, n), dtype=torch.bool, device=x.device).tril().expand(B, n, n)
    else:
        tree = _ancestors(s["parents"])
    mine = s["len"][:, None] + tree.sum(2) - 1  # the new tokens' positions: behind the cache, their depth in the tree
    there = torch.cat((at.expand(B, L), mine), 1)
    ahead = there[:, None, :] - mine[:, :, None]  # a key's position less the query's, (B, n, L + n)
    see = torch.cat(((at < s["len"][:, None])[:, None].expand(B, n, L), tree), 2)
    if c["window"]:
        see = see & (ahead > -c["window"])
    if c["bias"]:
        x = x + s["slopes"].reshape(1, hk, 1, g, 1) * ahead[:, None, :, None].to(torch.float32)
    x = torch.where(see[:, None, :, None], x, torch.full_like(x[..., :1], -math.inf))
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    p = p / total
    out = (p.reshape(B, hk, n * g, -1) @ v).reshape(B, hk, n, g, d).permute(0, 2, 1, 3, 4).reshape(B, n, hq, d).to(t)
    lse = (top + torch.log(total))[..., 0].permute(0, 2, 1, 3).reshape(B, n, hq)
    return {"out": out, "lse": lse}


def _plain_beam(s):
    c = s["case"]
    B, beams, V, width = c["B"], c["beams"], c["V"], c["width"]
    x = s["logits"].to(torch.float64)
    top = x.amax(2, keepdim=True)
    z = s["scores"].to(torch.float64)[..., None] + (x - (top + torch.log(torch.exp(x - top).sum(2, keepdim=True))))
    z = torch.where(torch.isnan(z), torch.full_like(z[..., :1], -math.inf), z).reshape(B, beams * V)
    score, at = torch.sort(z, dim=1, descending=True, stable=True)
    score, at = score[:, :width].to(torch.float32), at[:, :width]
    none = score == -math.inf
    row = torch.arange(B, device=at.device)[:, None] * beams + at // V
    return {"scores": score, "parents": torch.where(none, -1, row).to(torch.int32),
            "tokens": torch.where(none, -1, at % V).to(torch.int32)}


def _plain_append(s):
    c = s["case"]
    B, n, P = c["B"], c["n"], c["page"]
    k, v = s["kn"], s["vn"]
    at = s["len"][:, None].long() + torch.arange(n, device="cuda")
    row = torch.arange(B, device="cuda")[:, None].expand(B, n)
    if s["index"] is not None:
        on = s["index"] >= 0
        k, v, at, row = k[row[on], s["index"][on].long()], v[row[on], s["index"][on].long()], at[on], row[on]
    if s["table"] is None:
        s["k"][row, :, at], s["v"][row, :, at] = k, v
    else:
        page = s["table"][row, at // P].long()
        s["k"][page, :, at % P], s["v"][page, :, at % P] = k, v
    return {"k": s["k"], "v": s["v"]}


def _plain_fork(s):
    c = s["case"]
    P, N = c["page"], s["k"].shape[1]
    R, per = s["table"].shape
    live, at, rows = s["parents"] >= 0, torch.arange(per, device="cuda"), torch.arange(R, device="cuda")
    parent = s["parents"].clamp(min=0).long()
    n = torch.where(live, s["len"][parent], 0).long()
    used, fill = (n + P - 1) // P, n % P
    table = torch.where(at < used[:, None], s["table"][parent].long(), -1)
    last = table.gather(1, (used - 1).clamp(min=0)[:, None])[:, 0]
    open_ = fill > 0
    # who may write on in an open page: no row that has it full, and of the others the longest, then the first
    held = torch.zeros(N + 1, dtype=torch.long, device="cuda")
    held.scatter_add_(0, torch.where(at < (n // P)[:, None], table, N).reshape(-1), torch.ones(R * per, dtype=torch.long, device="cuda"))
    claim = fill * R + (R - 1 - rows)
    best = torch.full((N + 1,), -1, dtype=torch.long, device="cuda")
    best.scatter_reduce_(0, torch.where(open_, last, N), claim, "amax")
    copy = live & open_ & ((held[last] > 0) | (best[last] != claim))
    want = torch.where(live, (n + c["grow"] + P - 1) // P, 0)
    need = ((at >= used[:, None]) & (at < want[:, None])) | (copy[:, None] & (at == (used - 1)[:, None]))
    count = torch.zeros(N + 1, dtype=torch.long, device="cuda")
    count.scatter_add_(0, torch.where(table >= 0, table, N).reshape(-1), torch.ones(R * per, dtype=torch.long, device="cuda"))
    free = torch.sort(count[:N] > 0, stable=True)[1]
    have = (count[:N] == 0).sum()
    rank = torch.cumsum(need.reshape(-1).long(), 0).reshape(R, per) - 1
    fresh = torch.where(rank < have, free[rank.clamp(0, N - 1)], -1)
    table = torch.where(need, fresh, table)
    count = torch.zeros(N + 1, dtype=torch.long, device="cuda")
    count.scatter_add_(0, torch.where(table >= 0, table, N).reshape(-1), torch.ones(R * per, dtype=torch.long, device="cuda"))
    to, src, m = table[copy, used[copy] - 1], last[copy], fill[copy]
    in_ = (torch.arange(P, device="cuda") < m[:, None])[None, :, None, :, None]
    for x in (s["k"], s["v"]):
        x[:, to] = torch.where(in_, x[:, src], x[:, to])
    missing = (need & (rank >= have)).sum().reshape(1)
    return {"table": table.to(torch.int32), "lengths": n.to(torch.int32), "refs": count[:N].to(torch.int32),
            "missing": missing.to(torch.int32), "k": s["k"], "v": s["v"]}


def _plain_compact(s):
    c = s["case"]
    N, per = s["k"].shape[1], s["table"].shape[1]
    used = (s["len"] + c["page"] - 1) // c["page"]
    table = torch.where(torch.arange(per, device="cuda") < used[:, None], s["table"], -1).long()
    live = torch.zeros(N + 1, dtype=torch.bool, device="cuda")
    live[torch.where(table >= 0, table, N)] = True
    live = live[:N]
    count = live.sum()
    at = torch.arange(N, device="cuda")
    src, to = at[live & (at >= count)], at[~live & (at < count)]
    moved = at.clone()
    moved[src] = to
    for x in (s["k"], s["v"]):
        x[:, to] = x[:, src]
    table = torch.where(table >= 0, moved[table.clamp(min=0)], -1)
    return {"table": table.to(torch.int32), "live": count.reshape(1).to(torch.int32), "k": s["k"], "v": s["v"]}


# ------------------------------------------------------------------- one pass

def run(state):
    s, c = state, state["case"]
    if not own:
        return {"attn": _plain_attn, "beam": _plain_beam, "append": _plain_append, "fork": _plain_fork,
                "compact": _plain_compact}[c["op"]](s)
    if c["op"] == "attn":
        from voom_b200.runtime import kv_attention as kva

        out, lse = kva.tree_attention(s["q"], s["kn"], s["vn"], s["tree"], s["view"], cap=c["cap"] or None,
                                      slopes=s["slopes"], window=c["window"] or None, return_lse=True)
        return {"out": out, "lse": lse}
    if c["op"] == "beam":
        from voom_b200.runtime import beam

        r = beam.beam_select(s["logits"], s["scores"], c["width"])
        return {"scores": r.scores, "parents": r.parents, "tokens": r.tokens}
    from voom_b200.runtime import kv_pool

    if c["op"] == "append":
        kv_pool.kv_append(s["view"], s["kn"], s["vn"], index=s["index"])
        return {"k": s["k"], "v": s["v"]}
    if c["op"] == "fork":
        r = kv_pool.fork_pages(s["k"], s["v"], s["table"], s["len"], s["parents"], grow=c["grow"])
        return {"table": r.table, "lengths": r.lengths, "refs": r.refs, "missing": r.missing, "k": s["k"], "v": s["v"]}
    r = kv_pool.compact_pages(s["k"], s["v"], s["table"], s["len"])
    return {"table": r.table, "live": r.live, "k": s["k"], "v": s["v"]}


# ------------------------------------------------------ the definition, 64 bits

def _exact_attn(c, s):
    B, n, hq, hk, d = c["B"], c["n"], c["hq"], c["hk"], c["d"]
    g = hq // hk
    out = torch.zeros((B, n, hq, d), dtype=torch.float64, device="cuda")
    lse = torch.zeros((B, n, hq), dtype=torch.float64, device="cuda")
    parents = _tree(B, n, c["tree"], s["seed"])
    for b, x in enumerate(s["host_lengths"]):
        see = torch.zeros((n, x + n), dtype=torch.bool)
        see[:, :x] = True
        place = list(range(x)) + [0] * n
        for i in range(n):  # a token sees what its parent sees, and itself, one place further
            if parents[b][i] >= 0:
                see[i, x:] = see[parents[b][i], x:]
            see[i, x + i] = True
            place[x + i] = x if parents[b][i] < 0 else place[x + parents[b][i]] + 1
        place = torch.tensor(place, dtype=torch.float64, device="cuda")
        behind = place[x:, None] - place[None, :]
        see = see.cuda()
        if c["window"]:
            see &= behind < c["window"]
        for h in range(hk):
            if s["table"] is None:
                k, v = s["k"][b, h, :x], s["v"][b, h, :x]
            else:
                pages = s["table"][b].long()
                k, v = (y[pages, h].reshape(-1, d)[:x] for y in (s["k"], s["v"]))
            k, v = torch.cat((k, s["kn"][b, :, h])).double(), torch.cat((v, s["vn"][b, :, h])).double()
            for j in range(h * g, h * g + g):
                z = s["q"][b, :, j].double() @ k.T / math.sqrt(d)
                if c["cap"]:
                    z = torch.tanh(z / c["cap"]) * c["cap"]
                if c["bias"]:
                    z = z - s["slopes"][j].double() * behind
                z = z.masked_fill(~see, -math.inf)
                lse[b, :, j] = torch.logsumexp(z, 1)
                out[b, :, j] = torch.exp(z - lse[b, :, j, None]) @ v
    return {"out": out, "lse": lse}


def exact(case, seed):
    s = prepare(case, seed)
    s["seed"] = seed
    if case["op"] == "attn":
        return _exact_attn(case, s)
    if case["op"] == "beam":
        best = []
        for b in range(case["B"]):
            z = [s["scores"][b, i].double() + torch.log_softmax(s["logits"][b, i].double(), 0) for i in range(case["beams"])]
            best.append(torch.topk(torch.cat(z).nan_to_num(-math.inf, math.inf, -math.inf), case["width"])[0])
        return {"scores": torch.stack(best), "parents": None, "tokens": None}
    return None  # what the others give is copied or counted, not computed
