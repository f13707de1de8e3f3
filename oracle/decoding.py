"""Oracle of decoding over a paged cache: scored attention, beam selection, the
writing, forking and compacting of pages, from their definitions (torch CPU, 64
bits, loops)."""

from __future__ import annotations

import math

import torch


def scored_attention(q, kn, vn, sees, depth, k, v, scale, *, cap=0.0, slopes=None, window=0, token_weight=None):
    """One request: q (n, Hq, D), kn / vn (n, H, D) new, k / v (H, L, D) cached, sees
    (n, n), depth (n).  Returns out (n, Hq, D), lse (n, Hq), weight sums (H, L + n)."""
    n, hq, D = q.shape
    H, L, _ = k.shape
    g = hq // H
    out = torch.zeros((n, hq, D), dtype=torch.float64)
    lse = torch.full((n, hq), -math.inf, dtype=torch.float64)
    sums = torch.zeros((H, L + n), dtype=torch.float64)
    place = torch.tensor(list(range(L)) + [L + int(d) for d in depth], dtype=torch.float64)
    for i in range(n):
        if not sees[i, i]:
            continue
        behind = place[L + i] - place
        at = torch.cat((torch.ones(L, dtype=torch.bool), sees[i]))
        if window:
            at &= behind < window
        for h in range(hq):
            kk = torch.cat((k[h // g], kn[:, h // g])).double()[at]
            vv = torch.cat((v[h // g], vn[:, h // g])).double()[at]
            z = kk @ q[i, h].double() * scale
            if cap:
                z = torch.tanh(z / cap) * cap
            if slopes is not None:
                z = z - float(slopes[h]) * behind[at]
            lse[i, h] = torch.logsumexp(z, 0)
            p = torch.exp(z - lse[i, h])
            out[i, h] = p @ vv
            sums[h // g, at] += p * (1.0 if token_weight is None else float(token_weight[i]))
    return out, lse, sums


def beam_select(logits, scores, width):
    """(B, beams, V) logits, (B, beams) scores: scores (B, width) in 64 bits, parents, tokens."""
    B, beams, V = logits.shape
    best = torch.full((B, width), -math.inf, dtype=torch.float64)
    parents, tokens = (torch.full((B, width), -1, dtype=torch.int32) for _ in range(2))
    for b in range(B):
        z = []
        for i in range(beams):
            x = logits[b, i].double()
            top = x.max()
            z.append(scores[b, i].double() + (x - (top + torch.log(torch.exp(x - top).sum()))))
        z = torch.cat(z)
        z[torch.isnan(z)] = -math.inf
        order = torch.sort(z, descending=True, stable=True)[1][:width]
        for j, at in enumerate(order.tolist()):
            if z[at] == -math.inf:
                break
            best[b, j], parents[b, j], tokens[b, j] = z[at], b * beams + at // V, at % V
    return best, parents, tokens


def page_in(x, n_pages):
    """The page that an entry names; as page - 2^31 its row holds it, but cannot use it.  -1: none."""
    x &= 2 ** 31 - 1
    return x if x < n_pages else -1


def held(table, lengths, page, n_pages):
    """Each row's pages: the first ceil(length / page) entries, -1 where an entry is no page."""
    rows = []
    for t, n in zip(table, lengths):
        n = max(0, min(n, len(t) * page))
        rows.append([page_in(x, n_pages) for x in t[:-(-n // page)]])
    return rows


def fork(table, lengths, parents, grow, page, n_pages):
    """Lists in, lists out: table, lengths, refs, missing, and the open pages copied
    as (from, to, positions)."""
    R, per = len(table), len(table[0])
    had = held(table, lengths, page, n_pages)
    new_len, rows = [], []
    for r in range(R):
        p = parents[r]
        ok = 0 <= p < R
        new_len.append(max(0, min(lengths[p], per * page)) if ok else 0)
        rows.append(list(had[p]) if ok else [])
    refs = [0] * n_pages
    for t in rows:
        for x in t:
            if x >= 0:
                refs[x] += 1
    wanted, copies, missing = [], [], 0
    for r in range(R):
        n, g = new_len[r], grow[r] if 0 <= parents[r] < R else 0
        if g <= 0:
            continue
        used, want = -(-n // page), -(-(n + g) // page)
        missing += max(0, want - per)
        want = min(want, per)
        last = rows[r][used - 1] if n % page else -1
        if last >= 0:
            holders = [(min(new_len[x] - (used - 1) * page, page), -x) for x in range(R) if last in rows[x]]
            most = max(holders)
            if most[0] == page or most[1] != -r:
                wanted.append((r, used - 1))
                copies.append([last, None, n % page, len(wanted) - 1])
        wanted += [(r, j) for j in range(used, want)]
    free = [x for x in range(n_pages) if refs[x] == 0]
    given = [free[i] if i < len(free) else -1 for i in range(len(wanted))]
    missing += sum(x < 0 for x in given)
    out = [t + [-1] * (per - len(t)) for t in rows]
    for (r, j), x in zip(wanted, given):
        out[r][j] = x if x >= 0 or out[r][j] < 0 else out[r][j] - 2 ** 31  # (an open page that found no copy)
    refs = [0] * n_pages
    for t in out:
        for x in t:
            if page_in(x, n_pages) >= 0:
                refs[page_in(x, n_pages)] += 1
    return out, new_len, refs, missing, [(a, given[i], m) for a, _, m, i in copies if given[i] >= 0]


def compact(table, lengths, page, n_pages):
    """table, live, and the moves as (from, to)."""
    per = len(table[0])
    rows = held(table, lengths, page, n_pages)
    live = sorted({x for t in rows for x in t if x >= 0})
    count = len(live)
    moves = dict(zip([x for x in live if x >= count], [x for x in range(count) if x not in set(live)]))
    new = [[moves.get(x, x) - (2 ** 31 if x >= 0 and was < 0 else 0) for x, was in zip(t, old)] + [-1] * (per - len(t))
           for t, old in zip(rows, table)]
    return new, count, sorted(moves.items())
