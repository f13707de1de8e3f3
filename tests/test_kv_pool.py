"""Pages written, forked and compacted, against the rules in plain Python; then
decoding with several beams over a pool.  What is copied or counted has to be equal."""

from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

from oracle import attention as oa
from oracle import decoding as od


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def bits(x):
    return x.view(torch.int16)


# --------------------------------------------------------------------- append

def cache(kind, B, H, D, cap, page, dtype, seed=1):
    """A view over numbered values, its request-wise reader, and the number of positions it can hold."""
    from voom_b200.runtime.kv_attention import KVView

    g = torch.Generator(device="cuda").manual_seed(seed)
    length = i32([0] * B)
    if kind == "whole":
        k, v = (torch.randn((B, H, cap, D), device="cuda", generator=g).to(dtype) for _ in range(2))
        return KVView.contiguous(k, v, length), lambda x, b: (k if x == 0 else v)[b], cap
    if kind == "strided":  # keys and values of a position side by side, positions first
        kv = torch.randn((B, cap, 2, H, D + 8), device="cuda", generator=g).to(dtype)
        k, v = (kv[:, :, i, :, :D].transpose(1, 2) for i in range(2))
        return KVView.contiguous(k, v, length), lambda x, b: (k if x == 0 else v)[b], cap
    per = -(-cap // page)
    if kind == "pool":
        k, v = (torch.randn((B * per + 3, H, page, D), device="cuda", generator=g).to(dtype) for _ in range(2))
        table = torch.randperm(B * per + 3, generator=torch.Generator().manual_seed(seed))[:B * per].reshape(B, per)
        t = table.to(torch.int32).cuda()

        def read(x, b):
            return (k if x == 0 else v)[t[b].long()].transpose(0, 1).reshape(H, per * page, D)

        return KVView.pool(k, v, t, length), read, per * page
    pages = [[tuple(torch.randn((1, H, page, D), device="cuda", generator=g).to(dtype) for _ in range(2)) for _ in range(per)]
             for _ in range(B)]
    return (KVView.pages(pages, length), lambda x, b: torch.cat([p[x][0] for p in pages[b]], 1), per * page)


@pytest.mark.gpu
@pytest.mark.parametrize("kind,page", [("whole", 0), ("strided", 0), ("pool", 16), ("pool", 5), ("pages", 7)])
@pytest.mark.parametrize("H,D,dtype", [(1, 64, torch.bfloat16), (3, 128, torch.float16), (5, 40, torch.bfloat16),
                                       (9, 256, torch.float16)])
@pytest.mark.parametrize("n", [1, 6, 33])
def test_append(kind, page, H, D, dtype, n):
    from voom_b200.runtime.kv_pool import kv_append

    B, cap = 4, 60
    lens = [0, 17, 31, 44]  # the last one runs past the cache's end with 33
    view, read, room = cache(kind, B, H, D, cap, page, dtype)
    view.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    g = torch.Generator(device="cuda").manual_seed(3)
    kv = torch.randn((B, n, 2 * H + 1, D), device="cuda", generator=g).to(dtype)
    new = kv[:, :, :H], kv[:, :, H:2 * H]
    r = random.Random(n)
    m = n + 2
    index = [[r.randrange(-2, n + 2) for _ in range(m)] for _ in range(B)]
    for path in (None, index):
        want = [[read(x, b).clone() for b in range(B)] for x in range(2)]
        for b in range(B):
            for j in range(n if path is None else m):
                i = j if path is None else path[b][j]
                if 0 <= i < n and lens[b] + j < room:
                    for x in range(2):
                        want[x][b][:, lens[b] + j] = new[x][b, i]
        kv_append(view, *new, index=None if path is None else i32(path))
        for x in range(2):
            for b in range(B):
                assert torch.equal(bits(read(x, b).contiguous()), bits(want[x][b].contiguous())), (x, b)
    assert view.lengths.tolist() == lens


@pytest.mark.gpu
def test_append_past_pages_and_bad_entries():
    """Entries outside the pool take nothing, lengths outside the cache are clamped as the attention clamps them."""
    from voom_b200.runtime.kv_attention import KVView
    from voom_b200.runtime.kv_pool import kv_append

    k, v = (torch.zeros((4, 2, 8, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    view = KVView.pool(k, v, i32([[0, -1], [1, 99], [2, 3], [-5, 4]]), i32([7, 6, 1000, -4]))
    x = torch.ones((4, 4, 2, 64), dtype=torch.bfloat16, device="cuda")
    kv_append(view, x, 2 * x)
    want = torch.zeros_like(k)
    want[0, :, 7] = want[1, :, 6:] = 1
    assert torch.equal(k, want) and torch.equal(v, 2 * want)
    kv_append(view, x[:, :0], x[:, :0])
    kv_append(view, x, x, index=i32([[]] * 4))
    assert torch.equal(k, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["whole", "pool"])
def test_append_behind_a_view_s_bound(kind):
    """lengths[b] + j is where a token goes, whatever the view's max_len: what is cached already stays."""
    from voom_b200.runtime.kv_attention import KVView
    from voom_b200.runtime.kv_pool import kv_append

    k, v = (torch.zeros((2, 2, 40, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    if kind == "whole":
        view = KVView.contiguous(k, v, i32([10, 25]), max_len=10)
    else:
        k, v = (x.view(10, 2, 8, 64) for x in (k, v))
        view = KVView.pool(k, v, i32([[0, 1, 2, 3, 4], [5, 6, 7, 8, 9]]), i32([10, 25]), max_len=10)

    def rows():
        y = k if kind == "whole" else k.view(2, 5, 2, 8, 64).transpose(1, 2).reshape(2, 2, 40, 64)
        return y[:, 0, :, 0].float().cpu()

    want = torch.zeros(2, 40)
    for step in range(5):
        x = torch.full((2, 4, 2, 64), step + 1.0, dtype=torch.bfloat16, device="cuda")
        kv_append(view, x, x)
        for b, at in ((0, 10 + 4 * step), (1, 25 + 4 * step)):
            want[b, at:at + 4] = step + 1.0
        assert torch.equal(rows(), want), step
        view.lengths.add_(4)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("n,cap", [(1, None), (1, 9.0), (8, 9.0), (12, None), (20, 9.0), (60, None), (60, 9.0), (150, None), (150, 9.0)])
def test_entries_that_are_no_pages_read_as_zeros(n, cap, D):
    """By every kernel, however far outside the pool, an open page without a copy among them."""
    from voom_b200.runtime.kv_attention import DraftTree, KVView, tree_attention

    B, H, P, per = 2, 2, 64, 40  # tiles that TMA reads, requests that several blocks share
    g = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.randn((B * per, H, P, D), device="cuda", generator=g).bfloat16() for _ in range(2))
    table = torch.randperm(B * per, generator=torch.Generator().manual_seed(1)).reshape(B, per)
    k2, v2 = (x[table.reshape(-1).cuda()].reshape(B, per, H, P, D).clone() for x in (k, v))
    for b, j, x in ((0, 0, -1), (0, 3, B * per), (0, 4, 2 ** 31 - 1), (0, 39, 3 - 2 ** 31), (1, 1, -2 ** 31), (1, 2, 10 ** 6), (1, 38, -7)):
        table[b, j] = x
        k2[b, j], v2[b, j] = 0, 0
    k2, v2 = (x.transpose(1, 2).reshape(B, H, per * P, D).contiguous() for x in (k2, v2))
    lengths = i32([per * P - 3, per * P - 70])
    x = torch.randn((B, n, 3 * H, D), device="cuda", generator=g).bfloat16()
    args = (x[:, :, :H], x[:, :, H:2 * H], x[:, :, 2 * H:], DraftTree.chain(B, n, "cuda"))
    got = []
    for view in (KVView.pool(k, v, table.to(torch.int32).cuda(), lengths), KVView.contiguous(k2, v2, lengths)):
        w = torch.zeros((B, H, per * P + n), device="cuda")
        out, lse = tree_attention(*args, view, cap=cap, return_lse=True, weights=w)
        view.check_status()
        got.append((out, lse, w, tree_attention(*args, view, cap=cap)))
    assert all(torch.equal(a, b) for a, b in zip(*got))


# ----------------------------------------------------------------------- fork

def state(seed, *, rows, page, per, n_pages, ended=True):
    """Tables as forks, growth, rollbacks and ends leave them (by the oracle)."""
    r = random.Random(seed)
    table, lengths = [[-1] * per for _ in range(rows)], [0] * rows
    for step in range(8):
        parents = [r.randrange(rows) if r.random() < 0.5 else i for i in range(rows)]
        if ended:
            parents = [-1 if r.random() < 0.05 else p for p in parents]
        grow = [r.choice((0, 1, 1, page - 1, page, 2 * page + 3)) for _ in range(rows)]
        t, n, _, missing, _ = od.fork(table, lengths, parents, grow, page, n_pages)
        if missing or any(a + b > per * page for a, b in zip(n, grow)):
            continue
        table, lengths = t, [a + (b if parents[i] >= 0 else 0) for i, (a, b) in enumerate(zip(n, grow))]
        if r.random() < 0.3:  # some drop what they had written last
            lengths = [max(0, x - r.randrange(0, 2 * page)) if r.random() < 0.3 else x for x in lengths]
    return table, lengths, r


def check_fork(table, lengths, parents, grow, page, n_pages, layers=2, H=2, D=16, in_place=False, tensor_grow=True, dtype=torch.bfloat16):
    from voom_b200.runtime import kv_pool

    g = torch.Generator(device="cuda").manual_seed(5)
    k, v = (torch.randn((layers, n_pages, H, page, D), device="cuda", generator=g).to(dtype) for _ in range(2))
    t, n, refs, missing, copies = od.fork(table, lengths, parents, grow, page, n_pages)
    wk, wv = k.clone(), v.clone()
    for a, b, m in copies:
        wk[:, b, :, :m], wv[:, b, :, :m] = k[:, a, :, :m], v[:, a, :, :m]
    dt, dl = i32(table), i32(lengths)
    out = None
    if in_place:
        out = kv_pool.Forked(dt, dl, i32([7] * n_pages), i32([100]))
    identity = parents == list(range(len(parents)))
    got = kv_pool.fork_pages(k, v, dt, dl, None if identity else i32(parents), grow=i32(grow) if tensor_grow else grow[0], out=out)
    assert got.table.tolist() == t
    assert got.lengths.tolist() == n
    assert got.refs.tolist() == refs
    assert got.missing.tolist() == [missing + (100 if in_place else 0)]
    assert torch.equal(bits(k), bits(wk)) and torch.equal(bits(v), bits(wv))
    if not in_place:
        assert dt.tolist() == table and dl.tolist() == lengths
    return t, n, missing, copies


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed", range(12))
def test_fork(seed, in_place):
    rows, page, per = ((4, 16, 6), (9, 5, 11), (33, 4, 9), (6, 1, 40))[seed % 4]
    n_pages = rows * per // (1 if seed < 8 else 3) + 1
    table, lengths, r = state(seed, rows=rows, page=page, per=per, n_pages=n_pages)
    parents = [r.randrange(-1, rows + 1) for _ in range(rows)]
    grow = [r.choice((0, 1, 1, 2, page, 3 * page, -2)) for _ in range(rows)]
    check_fork(table, lengths, parents, grow, page, n_pages, in_place=in_place)
    check_fork(table, lengths, list(range(rows)), [1] * rows, page, n_pages, in_place=in_place, tensor_grow=False)
    check_fork(table, lengths, parents, [0] * rows, page, n_pages, in_place=in_place, tensor_grow=False)


@pytest.mark.gpu
def test_fork_finds_every_case():
    """Shared open pages with equal and unequal holders, full holders, pages that ran out, rows that are full."""
    P, N = 4, 12
    # rows 0, 1 share page 3 (open, equal); row 2 is a longer holder of it; row 3 has it full
    two = [[3, -1, -1], [3, -1, -1], [5, -1, -1], [6, 7, -1]]
    t, n, missing, copies = check_fork(two, [2, 2, 1, 6], [0, 1, 2, 3], [1] * 4, P, N)
    assert t[0][0] == 3 and t[1][0] == 0 and copies == [(3, 0, 2)] and not missing
    longer = [[3, -1, -1], [3, -1, -1], [3, -1, -1]]
    t, _, _, copies = check_fork(longer, [1, 3, 2], [0, 1, 2], [1] * 3, P, N)
    assert t[1][0] == 3 and copies == [(3, 0, 1), (3, 1, 2)]
    full = [[3, 4, -1], [3, -1, -1]]
    t, _, _, copies = check_fork(full, [5, 3], [0, 1], [1] * 2, P, N)
    assert t[0] == [3, 4, -1] and copies == [(3, 0, 3)]
    # the last page is given to the first row that wants one; a table row of three pages holds 12 positions
    tight = [[0, -1, -1], [1, -1, -1]]
    t, _, missing, _ = check_fork(tight, [4, 4], [0, 1], [1, 1], P, 3)
    assert t == [[0, 2, -1], [1, -1, -1]] and missing == 1
    _, _, missing, _ = check_fork([[0, 1, 2]], [11], [0], [6], P, 8)
    assert missing == 2
    # a page that a row of the old table held alone is free in the new one
    t, _, _, copies = check_fork([[2, -1, -1], [0, -1, -1]], [3, 4], [0, 0], [2, 2], P, 4)
    assert t == [[2, 0, -1], [1, 3, -1]] and copies == [(2, 1, 3)]
    # entries that are no pages, lengths out of bounds
    check_fork([[9, 99, -7], [1, 2, 3]], [500, -3], [0, 1], [1, 1], P, N)


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
def test_an_open_page_that_finds_no_copy_is_kept(in_place):
    """Too few pages for the copies: the rows hold their open pages still, marked, until a fork has pages for them."""
    P, N = 4, 5
    shared = [[0, 1, -1]] * 4  # four rows with an open page, two pages left for three copies
    t, n, missing, copies = check_fork(shared, [6] * 4, [0, 1, 2, 3], [1] * 4, P, N, in_place=in_place)
    assert t == [[0, 1, -1], [0, 2, -1], [0, 3, -1], [0, 4, -1]] and not missing
    t, n, missing, copies = check_fork(shared, [6] * 4, [0, 1, 2, 3], [3] * 4, P, N, in_place=in_place)
    assert t == [[0, 1, 2], [0, 3, 4], [0, 1 - 2 ** 31, -1], [0, 1 - 2 ** 31, -1]] and missing == 4 and len(copies) == 1
    again, _, missing, copies = check_fork(t, n, [0, 1, 2, 3], [1] * 4, P, 8, in_place=in_place)  # three pages more
    assert again == [[0, 1, -1], [0, 3, -1], [0, 2, -1], [0, 4, -1]] and not missing and len(copies) == 2
    # the others end: the page is the row's own, nothing is copied
    again, _, missing, copies = check_fork(t, n, [-1, -1, -1, 3], [1] * 4, P, N, in_place=in_place)
    assert again[3] == [0, 1, -1] and not missing and not copies
    # no growth: it reads as the page that it is
    again, _, missing, copies = check_fork(t, n, [0, 1, 2, 3], [0] * 4, P, N, in_place=in_place)
    assert again[2] == again[3] == [0, 1, -1]
    check_fork([[0, -2 ** 31 + 9, 2], [-2 ** 31, 3, -1]], [9, 5], [0, 1], [1, 1], P, N, in_place=in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(6))
def test_forks_with_too_few_pages(seed):
    """Rows that all share and all grow over pools of a few pages, then forks and compactions of what that leaves."""
    from voom_b200.runtime import kv_pool

    rows, page, per = ((4, 16, 6), (9, 5, 11), (33, 4, 9))[seed % 3]
    table, lengths, r = state(seed, rows=rows, page=page, per=per, n_pages=rows * per)
    n_pages = max(max(x for t in table for x in t) + 1, 1)
    for again in range(4):
        parents = [r.randrange(-1, rows) for _ in range(rows)]
        grow = [r.choice((0, 1, 1, page)) for _ in range(rows)]
        table, lengths, _, _ = check_fork(table, lengths, parents, grow, page, n_pages, in_place=bool(seed & 1))
        k, v = (torch.zeros((1, n_pages, 1, page, 8), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        for room in (False, True):
            counted = [per * page] * rows if room else lengths
            want, live, _ = od.compact(table, counted, page, n_pages)
            got = kv_pool.compact_pages(k, v, i32(table), i32(lengths), room=room)
            assert got.table.tolist() == want and got.live.tolist() == [live]


@pytest.mark.gpu
def test_a_large_table_with_too_few_pages():
    """More entries than one block forks: rows in fives share two pages, and two copies of every three wanted are to be had."""
    rows, page, per = 1000, 4, 9
    table = [[2 * (i // 5), 2 * (i // 5) + 1] + [-1] * 7 for i in range(rows)]
    n_pages = 400 + 500
    t, n, missing, _ = check_fork(table, [6] * rows, list(range(rows)), [1] * rows, page, n_pages, layers=1, H=1, D=8)
    assert missing == 300 and sum(x < -1 for r in t for x in r) == 300
    check_fork(t, n, list(range(rows)), [1] * rows, page, n_pages + 300, layers=1, H=1, D=8, in_place=True)


@pytest.mark.gpu
@pytest.mark.parametrize("compact", [False, True])
def test_a_pool_that_ran_out_goes_on_after_a_resize(compact):
    from voom_b200.runtime.kv_pool import PagePool

    pool = PagePool(2, 1, 64, pages=4, rows=3, max_len=32, page=8)
    pool.fork(grow=i32([12, 0, 0]))
    x = torch.randn((1, 12, 1, 64), device="cuda").bfloat16().expand(3, -1, -1, -1)
    for layer in range(2):
        pool.append(layer, x, 2 * x)
    pool.advance(i32([12, 0, 0]))
    pool.fork(i32([0, 0, 0]))
    pool.fork(grow=6)  # the first row's next page, then two copies and two pages behind them: two are left
    with pytest.raises(RuntimeError, match="3 too few"):
        pool.check_status()
    held = pool.refs.tolist()
    assert held[:2] == [3, 2] and pool.lengths.tolist() == [12] * 3
    if compact:
        pool.compact()
    pool.resize(8)
    pool.fork(grow=6)
    y = torch.randn((3, 6, 1, 64), device="cuda").bfloat16()
    for layer in range(2):
        pool.append(layer, y, 2 * y)
    pool.advance(6)
    pool.check_status()
    for r in range(3):
        t = pool.table[r, :3].long()
        assert bool((t >= 0).all())
        for layer in range(2):
            k, v = (p[layer, t, 0].reshape(-1, 64)[:18] for p in (pool.k, pool.v))
            want = torch.cat((x[r, :, 0], y[r, :, 0]))
            assert torch.equal(k, want) and torch.equal(v, 2 * want)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,per,page,n_pages", [(1, 1, 32768, 3), (700, 3, 2, 2500), (5, 600, 16, 9000), (1500, 40, 16, 70001)])
def test_fork_large(rows, per, page, n_pages):
    r = random.Random(rows)
    place = list(range(n_pages))
    r.shuffle(place)
    used = [r.randrange(0, per + 1) for _ in range(rows)]
    while sum(used) > n_pages:
        used[r.randrange(rows)] = 0
    it = iter(place)
    table = [[next(it) for _ in range(u)] + [-1] * (per - u) for u in used]
    lengths = [max(0, u * page - r.randrange(page)) for u in used]
    parents = [r.randrange(max(0, i - 3), min(rows, i + 3)) for i in range(rows)]
    check_fork(table, lengths, parents, [1] * rows, page, n_pages, layers=1, H=1, D=8, tensor_grow=False)


@pytest.mark.gpu
@pytest.mark.parametrize("H,D,page,layers", [(1, 256, 16, 3), (8, 128, 64, 2), (3, 40, 48, 1)])
def test_fork_copies_every_layer_of_odd_layouts(H, D, page, layers):
    from voom_b200.runtime import kv_pool

    # keys and values interleaved, positions before heads, padded
    store = torch.randn((6, layers, page, 2, H, D + 8), device="cuda").to(torch.float16)
    k, v = (store[:, :, :, i, :, :D].permute(1, 0, 3, 2, 4) for i in range(2))
    before = store.clone()
    m = page - 3
    got = kv_pool.fork_pages(k, v, i32([[4, -1], [2, -1]]), i32([m, 5]), i32([0, 0]), grow=1)
    assert got.table.tolist() == [[4, -1], [0, -1]]
    want = before.clone()
    want[0, :, :m, :, :, :D] = before[4, :, :m, :, :, :D]
    assert torch.equal(bits(store), bits(want))


# -------------------------------------------------------------------- compact

@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("seed,rows,page,per,n_pages", [(0, 4, 16, 6, 30), (1, 9, 5, 11, 100), (2, 33, 4, 9, 700), (3, 5, 3, 8, 20000),
                                                        (4, 2, 8, 3, 6), (5, 6, 1, 40, 300)])
def test_compact(seed, rows, page, per, n_pages, in_place):
    from voom_b200.runtime import kv_pool

    table, lengths, r = state(seed, rows=rows, page=page, per=per, n_pages=n_pages)
    place = list(range(n_pages))
    r.shuffle(place)  # anywhere in the pool
    table = [[place[x] if x >= 0 else x for x in t] for t in table]
    k, v = (torch.randn((2, n_pages, 2, page, 16), device="cuda").to(torch.bfloat16) for _ in range(2))
    t, live, moves = od.compact(table, lengths, page, n_pages)
    wk, wv = k.clone(), v.clone()
    for a, b in moves:
        wk[:, b], wv[:, b] = k[:, a], v[:, a]
    dt = i32(table)
    out = kv_pool.Compacted(dt, i32([0])) if in_place else None
    got = kv_pool.compact_pages(k, v, dt, i32(lengths), out=out)
    assert got.live.tolist() == [live] and got.table.tolist() == t
    assert torch.equal(bits(k), bits(wk)) and torch.equal(bits(v), bits(wv))


# ---------------------------------------------------------- refusals, streams

@pytest.mark.gpu
def test_refusals():
    from voom_b200.runtime import kv_pool
    from voom_b200.runtime.kv_attention import KVView

    k, v = (torch.zeros((2, 6, 2, 8, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    t, n = i32([[0, 1], [2, -1]]), i32([9, 3])
    ok = kv_pool.fork_pages(k, v, t, n)
    for a in ((k[0], v[0], t, n), (k, v[:1], t, n), (k.float(), v.float(), t, n), (k, v.half(), t, n), (k[..., :12], v[..., :12], t, n),
              (k[..., 4:36], v[..., 4:36], t, n), (k, v, t.long(), n), (k, v, t[0], n), (k, v, t[:, ::2], n), (k, v, t, n[:1]),
              (k, v, t, n.long()), (k, v, t, n.cpu()), (k[:, :0], v[:, :0], t, n)):
        with pytest.raises(ValueError):
            kv_pool.fork_pages(*a)
        with pytest.raises(ValueError):
            kv_pool.compact_pages(*a)
    for a in ((k, k), (k[:, :1].expand(2, 6, 2, 8, 64), v), (k[:1].expand(2, 6, 2, 8, 64), v)):
        with pytest.raises(ValueError, match="share|overlap"):
            kv_pool.fork_pages(*a, t, n)
        with pytest.raises(ValueError, match="share|overlap"):
            kv_pool.compact_pages(*a, t, n)
    for p in (i32([0]), i32([0, 1]).long(), torch.zeros(2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="parents"):
            kv_pool.fork_pages(k, v, t, n, p)
        with pytest.raises(ValueError, match="grow"):
            kv_pool.fork_pages(k, v, t, n, grow=p)
    with pytest.raises(ValueError, match="grow"):
        kv_pool.fork_pages(k, v, t, n, grow=-1)
    p = i32([0, 0])
    for out in (ok._replace(table=t), ok._replace(lengths=n), ok._replace(table=t, lengths=n[:1]), ok._replace(missing=ok.refs[:1]),
                ok._replace(refs=p), ok._replace(lengths=p), ok._replace(table=ok.table.long())):
        with pytest.raises(ValueError):
            kv_pool.fork_pages(k, v, t, n, p, out=out)
    for out in (kv_pool.Compacted(t, n[:1]), kv_pool.Compacted(ok.table, ok.table[0, :1]), kv_pool.Compacted(t[:1], ok.missing)):
        with pytest.raises(ValueError):
            kv_pool.compact_pages(k, v, t, n, out=out)
    view = KVView.pool(k[0], v[0], t, n)
    x = torch.zeros((2, 1, 2, 64), dtype=torch.bfloat16, device="cuda")
    for a in ((x[:1], x[:1]), (x.half(), x.half()), (x, x[:, :, :1]), (x[0], x[0]), (x.cpu(), x.cpu()), (x[..., :32], x[..., :32])):
        with pytest.raises(ValueError):
            kv_pool.kv_append(view, *a)
    for index in (i32([0, 0]), i32([[0], [0]]).long(), i32([[0]]), torch.zeros((2, 1), dtype=torch.int32)):
        with pytest.raises(ValueError, match="index"):
            kv_pool.kv_append(view, x, x, index=index)
    with pytest.raises(ValueError, match="share"):  # the new tokens are positions of the cache
        kv_pool.kv_append(view, k[0, :2, :, :1].transpose(1, 2), x)
    with pytest.raises(ValueError, match="overlap"):
        kv_pool.kv_append(KVView.pool(k[0, :1].expand(6, 2, 8, 64), v[0], t, n), x, x)
    with pytest.raises(ValueError):
        kv_pool.PagePool(1, 2, 64, pages=0, rows=1, max_len=8)
    with pytest.raises(ValueError):
        kv_pool.PagePool(1, 2, 60, pages=2, rows=1, max_len=8)


@pytest.mark.gpu
def test_tables_without_rows_are_refused_in_words():
    from voom_b200.runtime import kv_pool

    k, v = (torch.zeros((1, 6, 2, 8, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    for shape in ((0, 3), (3, 0)):
        t = torch.zeros(shape, dtype=torch.int32, device="cuda")
        for call in (kv_pool.fork_pages, kv_pool.compact_pages):
            with pytest.raises(ValueError, match="table"):
                call(k, v, t, torch.zeros(shape[0], dtype=torch.int32, device="cuda"))


def test_c_entries_refuse(built_lib):
    from voom_b200._lib import (VOOM_E_CAPACITY, VOOM_E_INVALID_ARG, VOOM_E_OVERLAP, VOOM_E_UNSUPPORTED, KvAppendArgs,
                                KvCompactArgs, KvForkArgs, KvViewStruct)

    def pool(a, kw):
        a.k, a.v, a.table, a.lengths, a.table_out = (1 << x for x in range(28, 33))
        a.layers, a.n_pages, a.hk, a.page, a.D, a.rows, a.per = 2, 6, 2, 8, 64, 3, 4
        a.k_pos = a.v_pos = 64
        a.k_head = a.v_head = 8 * 64
        a.k_page = a.v_page = 2 * 8 * 64
        a.k_layer = a.v_layer = 6 * 2 * 8 * 64
        for x, y in kw.items():
            setattr(a, x, y)
        return a

    def fork(scratch=1 << 40, **kw):
        a = KvForkArgs()
        a.lengths_out, a.refs, a.missing = 1 << 33, 1 << 34, 1 << 35
        return built_lib.voom_kv_fork(ctypes.byref(pool(a, kw)), scratch, 0, None)

    def compact(scratch=1 << 40, **kw):
        a = KvCompactArgs()
        a.live = 1 << 33
        return built_lib.voom_kv_compact(ctypes.byref(pool(a, kw)), scratch, 0, None)

    for call in (fork, compact):
        assert call() == VOOM_E_CAPACITY
        for bad in (dict(k=None), dict(table=None), dict(table_out=None), dict(layers=0), dict(n_pages=0), dict(D=0), dict(D=60),
                    dict(per=0), dict(k=(1 << 28) + 8), dict(v_page=2 * 8 * 64 + 4), dict(scratch=None), dict(scratch=24)):
            assert call(**bad) == VOOM_E_INVALID_ARG, bad
        for bad in (dict(page=32769), dict(rows=65536), dict(D=264), dict(per=1 << 29), dict(rows=60000, per=1 << 17, page=8)):
            assert call(**bad) == VOOM_E_UNSUPPORTED, bad
        for bad in (dict(k_layer=0), dict(v_page=0), dict(k_head=256), dict(v_pos=32), dict(v=1 << 28), dict(v=(1 << 28) + 128)):
            assert call(**bad) == VOOM_E_OVERLAP, bad
    for bad in (dict(lengths_out=None), dict(refs=None), dict(missing=None), dict(table_out=1 << 30), dict(lengths_out=1 << 31),
                dict(grow=1 << 31)):
        assert fork(**bad) == VOOM_E_INVALID_ARG, bad
    assert compact(live=None) == VOOM_E_INVALID_ARG

    c = KvViewStruct()
    c.k, c.v, c.len = 1 << 30, 1 << 31, 1 << 20
    c.k_page = c.k_head = c.v_page = c.v_head = 64 * 64
    c.k_page = c.v_page = 2 * 64 * 64
    c.k_pos = c.v_pos = 64
    c.B, c.hk, c.D, c.page, c.max_len = 2, 2, 64, 64, 64

    def append(view=c, **kw):
        a = KvAppendArgs()
        a.kn, a.vn = 1 << 21, 1 << 22
        a.n = a.m = 3
        a.kn_h = a.vn_h = 64
        a.kn_t = a.vn_t = 128
        a.kn_b = a.vn_b = 3 * 128
        for x, y in kw.items():
            setattr(a, x, y)
        return built_lib.voom_kv_append(ctypes.byref(view), ctypes.byref(a), None)

    assert append(n=0, m=0) == 0
    for bad in (dict(kn=None), dict(vn=None), dict(m=4), dict(kn=(1 << 21) + 8), dict(vn_t=4)):
        assert append(**bad) == VOOM_E_INVALID_ARG, bad
    assert append(kn=1 << 30) == VOOM_E_OVERLAP and append(vn=(1 << 31) + 256) == VOOM_E_OVERLAP
    same = KvViewStruct.from_buffer_copy(c)
    same.v = c.k
    assert append(view=same) == VOOM_E_OVERLAP


@pytest.mark.gpu
def test_a_pool_in_a_captured_step():
    """fork, append and attention of a step in one graph: replays see the table, lengths and parents of their time."""
    from voom_b200.runtime.kv_attention import DraftTree, tree_attention
    from voom_b200.runtime.kv_pool import PagePool

    def make():
        pool = PagePool(2, 2, 64, pages=40, rows=4, max_len=100, page=8)
        pool.k.zero_()
        pool.v.zero_()
        return pool

    g = torch.Generator().manual_seed(2)
    steps = [(torch.randn((4, 1, 8, 64), generator=g).to(torch.bfloat16).cuda(),
              i32([random.Random(s).randrange(4) if s else i for i in range(4)])) for s in range(20)]
    tree = DraftTree.chain(4, 1, "cuda")

    def step(pool, x, parents):
        pool.fork(parents, grow=1)
        out = []
        for layer in range(2):
            out.append(tree_attention(x[:, :, :4], x[:, :, 4:6], x[:, :, 6:], tree, pool.view(layer), window=50))
            pool.append(layer, x[:, :, 4:6], x[:, :, 6:])
        pool.advance(1)
        return out

    eager, want = make(), []
    for x, p in steps:
        want.append([y.clone() for y in step(eager, x, p)])
    pool = make()
    x, p = steps[0][0].clone(), steps[0][1].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(make(), x, p)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step(pool, x, p)
    for (nx, np_), w in zip(steps, want):
        x.copy_(nx)
        p.copy_(np_)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, w))
    assert torch.equal(pool.table, eager.table) and torch.equal(pool.lengths, eager.lengths) and torch.equal(pool.k, eager.k)
    pool.check_status()


@pytest.mark.gpu
def test_other_streams():
    from voom_b200.runtime import kv_pool

    table, lengths, _ = state(3, rows=9, page=5, per=11, n_pages=100)
    k, v = (torch.randn((2, 100, 2, 5, 16), device="cuda").to(torch.bfloat16) for _ in range(2))
    t, n = i32(table), i32(lengths)
    k2, v2 = k.clone(), v.clone()
    want = kv_pool.fork_pages(k2, v2, t, n, grow=3)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = kv_pool.fork_pages(k, v, t, n, grow=3, stream=side)
    packed = kv_pool.compact_pages(k, v, got.table, got.lengths, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    again = kv_pool.compact_pages(k2, v2, want.table, want.lengths)
    torch.cuda.synchronize()
    assert torch.equal(packed.table, again.table) and torch.equal(k, k2) and torch.equal(v, v2)


# -------------------------------------------------------------- used together

@pytest.mark.gpu
@pytest.mark.parametrize("B,beams,page,dtype", [(1, 4, 4, torch.bfloat16), (3, 3, 16, torch.float16)])
def test_beams_over_a_pool(B, beams, page, dtype):
    """A prompt, then steps of beams: attention over the pool equals attention over each beam's own history, the
    choices are those of the definition, and the pool holds no page that no beam needs."""
    from voom_b200.runtime.beam import beam_select
    from voom_b200.runtime.kv_attention import DraftTree, tree_attention
    from voom_b200.runtime.kv_pool import PagePool

    layers, hq, hk, D, V, prompt, steps = 2, 4, 2, 64, 500, 11, 14
    rows = B * beams
    g = torch.Generator().manual_seed(9)
    embed = torch.randn((V, hq + 2 * hk, D), generator=g).to(dtype)
    head = (torch.randn((hq * D, V), generator=g) * 0.2).to(dtype).cuda()
    slopes = torch.tensor([2.0 ** -(h + 1) for h in range(hq)])
    pool = PagePool(layers, hk, D, pages=rows * 12, rows=rows, max_len=prompt + steps, page=page, dtype=dtype)
    history = [[] for _ in range(rows)]  # tokens of each row
    kw = dict(cap=20.0, slopes=slopes.cuda(), window=9)

    def attend(new, n):
        """Appends n tokens a row; the last layer's attention of each row's last token."""
        x = torch.stack([embed[t] for t in new]).cuda()  # (rows, n, heads, D)
        for layer in range(layers):
            q, k, v = (x * (layer + 1)).split((hq, hk, hk), 2)
            o = tree_attention(q, k, v, DraftTree.chain(rows, n, "cuda"), pool.view(layer), **kw)
            pool.append(layer, k, v)
        pool.advance(n)
        for r in range(rows):
            history[r] = history[r] + list(new[r])
        for r in range(rows):  # the row's whole history in one piece
            y = embed[torch.tensor(history[r])] * layers
            q, k, v = y.split((hq, hk, hk), 1)
            m = len(history[r])
            sees = oa.tree_sees(list(range(-1, m - 1)))
            want, _, _ = od.scored_attention(q, k, v, sees, list(range(m)), k.new_zeros((hk, 0, D)), k.new_zeros((hk, 0, D)),
                                             D ** -0.5, cap=20.0, slopes=slopes, window=9)
            big = float(v.abs().max())
            step = 2.0 ** (-8 if dtype == torch.bfloat16 else -11)
            err = (o[r, -1].double().cpu() - want[-1]).abs().max()
            assert float(err) <= (2 * step + 1e-4) * big, (r, m)
        return o[:, -1].reshape(rows, -1)

    # the prompt goes into the first row of each request, the others fork from it
    r = random.Random(4)
    prompts = [[r.randrange(V) for _ in range(prompt)] for _ in range(B)]
    pool.fork(grow=prompt)
    out = attend([prompts[i // beams] for i in range(rows)], prompt)
    firsts = [b * beams for b in range(B) for _ in range(beams)]
    pool.fork(i32(firsts))
    scores = torch.full((B, beams), -math.inf, device="cuda")
    scores[:, 0] = 0.0
    for step in range(steps):
        logits = (out @ head).view(B, beams, V)
        choice = beam_select(logits, scores, beams)
        want, parents, tokens = od.beam_select(logits.cpu(), scores.cpu(), beams)
        assert torch.equal(choice.parents.cpu(), parents) and torch.equal(choice.tokens.cpu(), tokens)
        scores = choice.scores
        history = [history[p] for p in choice.parents.flatten().tolist()]
        if step + 1 == steps:
            break
        pool.fork(choice.parents.flatten(), grow=1)
        out = attend([[t] for t in choice.tokens.flatten().tolist()], 1)
        if step == 6:
            pool.resize(max(int(pool.compact().item()), 1) + 3 * rows)
    pool.check_status()
    held = {x for t, n in zip(pool.table.tolist(), pool.lengths.tolist()) for x in t[:-(-n // page)]}
    assert -1 not in held and len(held) <= int((pool.refs > 0).sum())
    pool.fork(i32([-1] * rows))
    assert int(pool.refs.sum()) == 0 and pool.lengths.tolist() == [0] * rows and int(pool.compact().item()) == 0


@pytest.mark.gpu
def test_a_pool_that_runs_out_says_so():
    from voom_b200.runtime.kv_pool import PagePool

    pool = PagePool(1, 1, 64, pages=3, rows=2, max_len=32, page=8)
    pool.fork(grow=8)
    pool.check_status()
    pool.advance(8)
    pool.fork(grow=1)
    assert pool.table.tolist()[0][1] == 2 and pool.table.tolist()[1][1] == -1
    with pytest.raises(RuntimeError, match="1 too few"):
        pool.check_status()
    pool.check_status()
    with pytest.raises(ValueError, match="in use"):
        pool.resize(1)


@pytest.mark.gpu
def test_a_row_that_is_full_says_so():
    """max_len counts whole pages; what a row has no room for is reported, not written past its end."""
    from voom_b200.runtime.kv_pool import PagePool

    pool = PagePool(1, 1, 64, pages=8, rows=2, max_len=10, page=4)
    assert pool.max_len == 12
    pool.fork(grow=i32([12, 5]))
    x = torch.ones((2, 13, 1, 64), dtype=torch.bfloat16, device="cuda")
    pool.k.zero_()
    pool.append(0, x, x)
    pool.check_status()
    pool.advance(i32([12, 5]))
    pool.fork(grow=1)
    assert pool.lengths.tolist() == [12, 5]
    with pytest.raises(RuntimeError, match="1 too few"):
        pool.check_status()
    assert int(pool.k.sum()) == (12 + 8) * 64  # the rows' five pages and no other


@pytest.mark.gpu
@pytest.mark.parametrize("pages,fail_at", [(40, 0), (40, 1), (40, 2), (9, 0), (9, 1), (9, 2)])
def test_a_resize_that_runs_out_leaves_the_pool_usable(pages, fail_at, monkeypatch):
    from voom_b200.runtime.kv_pool import PagePool

    def fill(pool, n, x):
        pool.fork(grow=n)
        for layer in range(2):
            pool.append(layer, x, 2 * x)
        pool.advance(n)

    def read(pool):
        t = pool.table[:, :2].long()
        return [y[:, t].transpose(2, 3).reshape(2, 2, 2, 16, 64)[..., :11, :].clone() for y in (pool.k, pool.v)]

    g = torch.Generator(device="cuda").manual_seed(1)
    pool = PagePool(2, 2, 64, pages=20, rows=2, max_len=32, page=8)
    fill(pool, 11, torch.randn((2, 11, 2, 64), device="cuda", generator=g).bfloat16())
    want = read(pool)
    plain, calls = torch.Tensor.new_empty, []

    def new_empty(self, size, *a, **kw):  # only what resize asks for
        if isinstance(size, tuple) and len(size) == 5:
            calls.append(tuple(size))
            if len(calls) == fail_at + 1:
                raise torch.OutOfMemoryError("no memory for a test")
        return plain(self, size, *a, **kw)

    monkeypatch.setattr(torch.Tensor, "new_empty", new_empty)
    if fail_at < 2:
        with pytest.raises(torch.OutOfMemoryError):
            pool.resize(pages)
    else:
        pool.resize(pages)
    monkeypatch.undo()
    assert pool.k.shape == pool.v.shape and pool.refs.shape == (pool.pages,) and pool.pages >= 4
    assert all(pool.view(i).k.data_ptr() == pool.k[i].data_ptr() and pool.view(i).v.data_ptr() == pool.v[i].data_ptr() for i in range(2))
    assert all(torch.equal(a, b) for a, b in zip(read(pool), want))
    x = torch.randn((2, 3, 2, 64), device="cuda", generator=g).bfloat16()
    fill(pool, 3, x)
    pool.check_status()
    assert pool.lengths.tolist() == [14, 14]
    assert all(torch.equal(a, b) for a, b in zip(read(pool), want))
    pool.resize(12)
    assert pool.pages == 12 and all(torch.equal(a, b) for a, b in zip(read(pool), want))


@pytest.mark.gpu
def test_resize_holds_one_old_and_one_new_piece_at_a_time():
    from voom_b200.runtime.kv_pool import PagePool

    pool = PagePool(1, 8, 128, pages=4000, rows=2, max_len=128, page=64)  # 524 MB of keys, as much of values
    pool.fork(grow=70)
    one = pool.k.numel() * 2
    torch.cuda.synchronize()
    was = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    pool.resize(3600)
    assert torch.cuda.max_memory_allocated() - was < one
    assert torch.cuda.memory_allocated() - was < -0.15 * one


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["compact", "resize"])
def test_room_outlasts_compaction(how):
    """Room that a fork made and nothing has filled yet is still there afterwards: what is appended then is written."""
    from voom_b200.runtime.kv_pool import PagePool

    pool = PagePool(2, 1, 64, pages=30, rows=4, max_len=64, page=8)
    pool.fork(grow=i32([20, 3, 9, 8]))
    x = torch.randn((4, 20, 1, 64), device="cuda").bfloat16()
    for layer in range(2):
        pool.append(layer, x, x)
    pool.advance(i32([20, 3, 9, 8]))
    pool.fork(i32([-1, 1, 2, 3]), grow=13)  # row 0's pages are free: there are holes
    live = -(-16 // 8) + -(-22 // 8) + -(-21 // 8)
    if how == "compact":
        assert pool.compact().tolist() == [live]
    else:
        with pytest.raises(ValueError, match="in use"):
            pool.resize(live - 1)
        pool.resize(live)
    y = torch.randn((4, 13, 1, 64), device="cuda").bfloat16()
    for layer in range(2):
        pool.append(layer, y, 2 * y)
    pool.advance(i32([0, 13, 13, 13]))
    pool.check_status()
    for r, n in ((1, 3), (2, 9), (3, 8)):
        t = pool.table[r, :-(-(n + 13) // 8)].long()
        assert bool((t >= 0).all()) and bool((t < live).all())
        for layer in range(2):
            k, v = (p[layer, t, 0].reshape(-1, 64)[:n + 13] for p in (pool.k, pool.v))
            assert torch.equal(k[:n], x[r, :n, 0]) and torch.equal(k[n:], y[r, :, 0]) and torch.equal(v[n:], 2 * y[r, :, 0])


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(40))
def test_lives_of_a_pool(seed):
    """Forks, ends, growth, rollbacks, compactions, resizes and shortages in any order: every row holds its own history."""
    from voom_b200.runtime.kv_pool import PagePool

    r = random.Random(seed)
    rows, page, layers = r.choice((1, 2, 5, 9, 40)), r.choice((1, 2, 4, 8, 16)), 2
    pool = PagePool(layers, 1, 8, pages=r.choice((1, 3, rows, 3 * rows)), rows=rows, max_len=r.choice((10, 40, 100)), page=page)
    history, token = [[] for _ in range(rows)], 0
    for step in range(20):
        parents = [-1 if r.random() < 0.1 else r.choice((i, i, r.randrange(rows))) for i in range(rows)]
        history = [list(history[p]) if p >= 0 else [] for p in parents]
        grow = [min(r.choice((0, 1, 1, 2, page, 2 * page + 1)), pool.max_len - len(h)) for h in history]
        pool.fork(i32(parents), grow=i32(grow))
        grow = [g if p >= 0 else 0 for g, p in zip(grow, parents)]
        for _ in range(100):
            try:
                pool.check_status()
                break
            except RuntimeError:
                pool.resize(int(pool.compact().item()) + r.choice((1, 5, 2 * rows)))
                pool.fork(grow=i32(grow))
        if r.random() < 0.3:
            live = int(pool.compact().item())
            if r.random() < 0.5:
                pool.resize(max(1, live + r.choice((0, 1, 4))))
        n = max(grow + [1])
        ids, index = torch.zeros((rows, n)), torch.full((rows, n), -1, dtype=torch.int32)
        new = [r.randrange(g + 1) for g in grow]
        for i, m in enumerate(new):
            for j in range(m):
                token = token % 200 + 1
                ids[i, j], index[i, j] = token, j
                history[i].append(token)
        x = ids[:, :, None, None].expand(rows, n, 1, 8).to(torch.bfloat16).cuda()
        for layer in range(layers):
            pool.append(layer, x * (layer + 1), -x, index=index.cuda())
        pool.advance(i32(new))
        if r.random() < 0.2:
            back = [min(r.randrange(page + 2), len(h)) if r.random() < 0.4 else 0 for h in history]
            pool.advance(i32([-b for b in back]))
            history = [h[:len(h) - b] for h, b in zip(history, back)]
        assert pool.lengths.tolist() == [len(h) for h in history], step
        table = pool.table.cpu().long()
        for layer in range(layers):
            k, v = pool.k[layer, :, 0, :, 0].float().cpu(), pool.v[layer, :, 0, :, 7].float().cpu()
            for i, h in enumerate(history):
                at = table[i, :-(-len(h) // page)]
                assert bool(((at >= 0) & (at < pool.pages)).all()), (step, i)
                assert k[at].reshape(-1)[:len(h)].tolist() == [float(y * (layer + 1)) for y in h], (step, i)
                assert v[at].reshape(-1)[:len(h)].tolist() == [-float(y) for y in h], (step, i)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 9])
def test_pages_past_32_bits(n):
    """A pool of more than 2^32 bytes and 2^31 values: its last pages are written, forked, read and moved as its first are."""
    from voom_b200.runtime import kv_attention as kva
    from voom_b200.runtime.kv_pool import compact_pages, fork_pages, kv_append

    N, H, P, D, L = 34000, 8, 64, 128, 130
    k, v = (torch.zeros((1, N, H, P, D), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    assert (N - 3) * H * P * D > 2 ** 31
    g = torch.Generator(device="cuda").manual_seed(3)
    new = [torch.randn((1, L, H, D), generator=g, device="cuda").bfloat16() for _ in range(2)]
    q, kn, vn = (torch.randn((2, n, h, D), generator=g, device="cuda").bfloat16() for h in (2 * H, H, H))
    tables = [torch.tensor([[a, a + 1, a + 2, -1]], dtype=torch.int32, device="cuda") for a in (0, N - 3)]
    empty, full = (torch.full((1,), x, dtype=torch.int32, device="cuda") for x in (0, L))
    for t in tables:
        kv_append(kva.KVView.pool(k[0], v[0], t, empty, max_len=4 * P), *new)
    assert torch.equal(k[0, N - 3:], k[0, :3]) and torch.equal(v[0, N - 3:], v[0, :3]) and bool(k[0, N - 1, :, 0].any())
    both = torch.cat(tables)
    view = kva.KVView.pool(k[0], v[0], both, torch.cat([full, full]), max_len=4 * P)
    qs, ks, vs = (x[:1].expand(2, -1, -1, -1).contiguous() for x in (q, kn, vn))
    out = kva.tree_attention(qs, ks, vs, kva.DraftTree.chain(2, n, "cuda"), view, cap=20.0, window=100)
    view.check_status()
    assert torch.equal(out[0], out[1]) and bool(out[0].any())
    # the last row twice, both growing: its open page is copied for one of them
    f = fork_pages(k, v, both, torch.cat([full, full]), torch.tensor([1, 1], dtype=torch.int32, device="cuda"), grow=1)
    assert f.table.tolist() == [[N - 3, N - 2, N - 1, -1], [N - 3, N - 2, 0, -1]] and int(f.missing) == 0
    assert torch.equal(k[0, 0, :, :L % P], k[0, N - 1, :, :L % P])
    was = k[0, N - 3:].clone()
    c = compact_pages(k, v, f.table, f.lengths)
    assert c.table.tolist() == [[1, 2, 3, -1], [1, 2, 0, -1]] and int(c.live) == 4
    assert torch.equal(k[0, 1:4], was) and torch.equal(v[0, 1:4], v[0, N - 3:])
