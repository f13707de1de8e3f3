"""Tree attention over a KV cache, its weight sums, and eviction, against the
definitions in 64 bits.

Tolerances.  Scores are sums of D products of 16-bit values in fp32: with the
inputs here (|q| ~ 1, |k| ~ 1) they are off by at most about 1e-5, so lse and a
row's weights are good to 3e-5 and 5e-5 relative.  The output is a convex sum of
values: rounding its probabilities and itself to 16 bits costs at most one unit
each, 2 * 2^-8 (BF16) or 2 * 2^-11 (FP16) of the largest value a row could take,
relative to max |v|."""

from __future__ import annotations

import ctypes
import math
import random

import pytest
import torch

from oracle import attention as oa

STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def parents_of(kind, n, seed=0):
    r = random.Random(seed)
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return [-1] + [0] * (n - 1)
    if kind == "roots":
        return [-1] * n
    if kind == "padded":  # the last third are no tokens, one hole before them
        p = [-1 if i == 0 else r.randrange(-1, i) for i in range(n)]
        return [-2 if i >= n - n // 3 or (i == 2 and n > 4) else x for i, x in enumerate(p)]
    return [-1 if i == 0 else r.randrange(max(-1, i - 5), i) for i in range(n)]


def inputs(B, n, hq, hk, D, lens, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    cap = max(max(lens), 1)
    qkv = torch.randn((B, n, hq + 2 * hk, D), generator=g).to(dtype)
    k = torch.randn((B, hk, cap, D), generator=g).to(dtype)
    v = torch.randn((B, hk, cap, D), generator=g).to(dtype)
    return qkv, k, v


def place(k, v, lens, layout, page, seed=3):
    """The cache on the device in one of the layouts; everything past a request's length is NaN."""
    from voom_b200.runtime.kv_attention import KVView

    B, H, cap, D = k.shape
    k, v = k.clone(), v.clone()
    for b, x in enumerate(lens):
        k[b, :, x:] = math.nan
        v[b, :, x:] = math.nan
    length = torch.tensor(lens, dtype=torch.int32, device="cuda")
    if layout == "whole":
        return KVView.contiguous(k.cuda(), v.cuda(), length, max_len=max(lens))
    if layout == "strided":  # (B, cap, H, D + 8) storage
        def put(x):
            big = torch.full((B, cap, H, D + 8), math.nan, dtype=x.dtype, device="cuda")
            big[..., :D] = x.transpose(1, 2).cuda()
            return big[..., :D].transpose(1, 2)

        return KVView.contiguous(put(k), put(v), length)
    per = -(-cap // page)

    def pages(x):
        pad = torch.full((B, H, per * page, D), math.nan, dtype=x.dtype)
        pad[:, :, :cap] = x
        return pad.reshape(B, H, per, page, D).transpose(1, 2)

    kp, vp = pages(k), pages(v)
    if layout == "pool":
        perm = torch.randperm(B * per + 2, generator=torch.Generator().manual_seed(seed))[: B * per]
        kk, vv = (torch.full((B * per + 2, H, page, D), math.nan, dtype=k.dtype) for _ in range(2))
        kk[perm], vv[perm] = kp.reshape(-1, H, page, D), vp.reshape(-1, H, page, D)
        table = perm.reshape(B, per).to(torch.int32)
        for b, x in enumerate(lens):
            table[b, -(-x // page):] = -1
        return KVView.pool(kk.cuda(), vv.cuda(), table.cuda(), length)
    return KVView.pages([[(kp[b, p].contiguous().cuda()[None], vp[b, p].contiguous().cuda()[None])
                          for p in range(per)] for b in range(B)], length)


def check(got, want, tol, what):
    got, want = got.double().cpu(), want.double()
    assert torch.equal(torch.isneginf(got), torch.isneginf(want)), what
    fine = torch.isfinite(want)
    assert bool(torch.isfinite(got[fine]).all()), what
    err = (got[fine] - want[fine]).abs()
    assert err.numel() == 0 or float(err.max()) <= tol, (what, float(err.max()), tol)


def run_case(B, n, hq, hk, D, lens, dtype, layout="whole", page=16, kind="tree", weights=True, tw=False, scale=None,
             seed=0, sharp=1.0):
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(B, n, hq, hk, D, lens, dtype, seed)
    qkv[:, :, :hq] *= sharp
    par = [parents_of(kind, n, seed + b) for b in range(B)]
    d = qkv.cuda()
    view = place(k, v, lens, layout, page)
    tree = kva.DraftTree.chain(B, n, "cuda") if kind == "chain" else kva.DraftTree(
        torch.tensor(par, dtype=torch.int32, device="cuda").reshape(B, n))
    w0 = torch.rand((B, hk, view.max_len + n + 3), generator=torch.Generator().manual_seed(9))
    w = w0.cuda() if weights else None
    t = torch.rand((B, n), generator=torch.Generator().manual_seed(8)) if tw else None
    for b in range(B):  # what no row may see, none may feel
        for j in range(n):
            if par[b][j] == -2:
                d[b, j] = math.nan
    out, lse = kva.tree_attention(d[:, :, :hq], d[:, :, hq:hq + hk], d[:, :, hq + hk:], tree, view, scale=scale,
                                  weights=w, token_weight=None if t is None else t.cuda(), return_lse=True)
    bare, bare_lse = kva.tree_attention(d[:, :, :hq], d[:, :, hq:hq + hk], d[:, :, hq + hk:], tree, view, scale=scale,
                                        return_lse=True)
    torch.cuda.synchronize()
    view.check_status()
    f = D ** -0.5 if scale is None else scale
    for b, x in enumerate(lens):
        o, l, s = oa.attention(qkv[b, :, :hq], qkv[b, :, hq:hq + hk], qkv[b, :, hq + hk:], oa.tree_sees(par[b]),
                               k[b, :, :x], v[b, :, :x], f, None if t is None else t[b])
        big = max(float(v[b].abs().max()), float(qkv[b, :, hq + hk:].abs().max()))
        check(out[b], o, 2 * STEP[dtype] * big, ("out", b))
        check(lse[b], l, 3e-5 * max(1.0, sharp), ("lse", b))
        check(bare[b], o, 2 * STEP[dtype] * big, ("out without weights", b))
        check(bare_lse[b], l, 3e-5 * max(1.0, sharp), ("lse without weights", b))
        if weights:
            want = w0[b].double()
            want[:, :x + n] += s
            check(w[b], want, 5e-5 * max(1.0, sharp) * (n * hq // hk) ** 0.5 + 1e-6, ("weights", b))
    return out, lse, w


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("layout,page", [("whole", 0), ("strided", 0), ("pool", 16), ("pool", 5), ("pages", 48)])
@pytest.mark.parametrize("n,hq,hk,D", [(1, 9, 3, 64), (1, 8, 1, 128), (7, 4, 2, 128), (5, 6, 2, 256), (33, 4, 2, 64),
                                       (20, 8, 1, 128), (48, 8, 2, 256)])
def test_layouts_heads_and_types(dtype, layout, page, n, hq, hk, D):
    run_case(3, n, hq, hk, D, [77, 0, 130], dtype, layout, page)


@pytest.mark.gpu
@pytest.mark.parametrize("length", [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 255, 257, 511])
@pytest.mark.parametrize("n,hq,D", [(1, 4, 64), (1, 4, 128), (1, 2, 256), (40, 4, 128), (9, 8, 256)])
def test_lengths_around_tiles(length, n, hq, D):
    run_case(1, n, hq, 1, D, [length], torch.bfloat16, kind="chain" if n == 9 else "tree")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["chain", "star", "roots", "padded", "tree"])
@pytest.mark.parametrize("n,g", [(2, 1), (17, 3), (32, 1), (64, 4), (65, 2), (100, 8), (129, 1)])
def test_trees(kind, n, g):
    run_case(2, n, 2 * g, 2, 64, [70, 3], torch.bfloat16, kind=kind, tw=True)


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 40, 72, 80, 96, 112, 192, 200])
@pytest.mark.parametrize("n", [1, 21])
def test_head_sizes(D, n):
    run_case(2, n, 6, 2, D, [50, 133], torch.float16)


@pytest.mark.gpu
def test_many_split_and_ragged():
    # long enough to be split over many blocks; ragged, with empty requests among them
    run_case(4, 1, 4, 1, 64, [20000, 0, 777, 5], torch.bfloat16, "pool", 16)
    run_case(2, 36, 2, 1, 64, [9000, 1234], torch.bfloat16, "pool", 16)


@pytest.mark.gpu
def test_long_chain_over_cache():
    run_case(1, 300, 2, 1, 64, [200], torch.bfloat16, kind="chain")
    run_case(1, 150, 2, 1, 256, [70], torch.float16, kind="chain", layout="pool", page=32)
    run_case(2, 200, 1, 1, 128, [0, 130], torch.bfloat16, kind="chain")


@pytest.mark.gpu
@pytest.mark.parametrize("n,g,D", [(1, 4, 128), (40, 4, 128), (40, 2, 256), (12, 1, 64)])
def test_sharp_softmax(n, g, D):
    # rows dominated by one position, the maximum moving along the keys
    run_case(1, n, g, 1, D, [700], torch.bfloat16, sharp=8.0)


@pytest.mark.gpu
def test_growing_scores():
    """Keys that grow along the cache: every tile raises the running maximum."""
    from voom_b200.runtime import kv_attention as kva

    for n, g, D in ((1, 4, 128), (40, 4, 64), (24, 2, 256)):
        qkv, k, v = inputs(1, n, g, 1, D, [900], torch.bfloat16)
        qkv[:, :, :g] = qkv[:, :, :g].abs()
        k = (k.abs() * torch.linspace(0.0, 1.0, 900)[:, None]).to(torch.bfloat16)
        d = qkv.cuda()
        view = place(k, v, [900], "whole", 0)
        out, lse = kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], kva.DraftTree.chain(1, n, "cuda"),
                                      view, return_lse=True)
        o, l, _ = oa.attention(qkv[0, :, :g], qkv[0, :, g:g + 1], qkv[0, :, g + 1:],
                               oa.tree_sees(list(range(-1, n - 1))), k[0], v[0], D ** -0.5)
        check(out[0], o, 2 * STEP[torch.bfloat16] * float(v.abs().max()), "out")
        check(lse[0], l, 1e-4, "lse")


@pytest.mark.gpu
@pytest.mark.parametrize("n,g,D", [(6, 2, 64), (40, 4, 128), (20, 4, 256)])
def test_nan_and_inf_stay_in_their_branch(n, g, D):
    """Two branches from a root: values of one that are not finite reach its own rows only."""
    from voom_b200.runtime import kv_attention as kva

    par = [-1] + [0 if i < 3 else i - 2 for i in range(1, n)]
    qkv, k, v = inputs(1, n, g, 1, D, [37], torch.bfloat16)
    sees = oa.tree_sees(par)
    d = qkv.cuda()
    bad = 3  # in the odd branch
    d[0, bad, g + 1, 0] = math.nan
    d[0, bad, g + 1, 1] = math.inf
    d[0, bad + 1, g] = math.nan  # a key of the even branch
    view = place(k, v, [37], "whole", 0)
    tree = kva.DraftTree(torch.tensor([par], dtype=torch.int32, device="cuda"))
    out = kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], tree, view)[0].float().cpu()
    o, _, _ = oa.attention(qkv[0, :, :g], qkv[0, :, g:g + 1], qkv[0, :, g + 1:], sees, k[0], v[0], D ** -0.5)
    for i in range(n):
        if sees[i, bad + 1]:
            assert bool(out[i].isnan().all()), i
        elif sees[i, bad]:
            assert bool(out[i, :, 0].isnan().all()) and bool((out[i, :, 1] == math.inf).all()), i
            check(out[i, :, 2:], o[i, :, 2:], 2 * STEP[torch.bfloat16] * float(v.abs().max() + 1), i)
        else:
            check(out[i], o[i], 2 * STEP[torch.bfloat16] * float(v.abs().max() + 1), i)


@pytest.mark.gpu
def test_masks_and_depths():
    from voom_b200.runtime import kv_attention as kva

    for n in (1, 31, 32, 33, 64, 200, 1024):
        par = [parents_of("tree", n, 5), parents_of("padded", n, 6), parents_of("chain", n)]
        t = kva.DraftTree(torch.tensor(par, dtype=torch.int32, device="cuda"))
        bits = t.mask.cpu().to(torch.int64) & 0xFFFFFFFF
        for b in range(3):
            sees = oa.tree_sees(par[b])
            got = (bits[b][:, :, None] >> torch.arange(32) & 1).reshape(n, -1)[:, :n].bool()
            assert torch.equal(got, sees)
            assert t.depth[b].tolist() == oa.tree_depth(par[b])
    t = kva.DraftTree(torch.tensor([[5, 7, 0, -9]], dtype=torch.int32, device="cuda"))  # not parents: roots
    assert t.depth[0].tolist() == [0, 0, 1, 0]
    lens = torch.tensor([10], dtype=torch.int32, device="cuda")
    assert t.positions(lens)[0].tolist() == [10, 10, 11, 10]


@pytest.mark.gpu
def test_same_bits_again_streams_and_graph():
    from voom_b200.runtime import kv_attention as kva

    for n, hq in ((1, 8), (40, 8)):
        qkv, k, v = inputs(2, n, hq, 2, 128, [5000, 3000], torch.bfloat16)
        d = qkv.cuda()
        view = place(k, v, [5000, 3000], "pool", 16)
        tree = kva.DraftTree.chain(2, n, "cuda")
        args = (d[:, :, :hq], d[:, :, hq:hq + 2], d[:, :, hq + 2:], tree, view)

        def once(stream=None):
            w = torch.zeros((2, 2, view.max_len + n), device="cuda")
            torch.cuda.synchronize()
            o, l = kva.tree_attention(*args, weights=w, return_lse=True, stream=stream)
            torch.cuda.synchronize()
            return o, l, w

        first = once()
        bare = kva.tree_attention(*args)
        for _ in range(3):
            assert torch.equal(kva.tree_attention(*args), bare)
        for s in (None, torch.cuda.Stream(), None):
            for x, y in zip(once(s), first):
                assert torch.equal(x, y)
        w = torch.zeros((2, 2, view.max_len + n), device="cuda")
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            kva.tree_attention(*args, weights=w)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = kva.tree_attention(*args, weights=w)
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first[0]) and torch.equal(w, first[2])
        view.lengths.copy_(torch.tensor([100, 2000], dtype=torch.int32))  # the graph sees the new lengths
        w.zero_()
        graph.replay()
        torch.cuda.synchronize()
        again = once()
        assert torch.equal(out, again[0]) and torch.equal(w, again[2])


@pytest.mark.gpu
def test_lengths_out_of_bounds_are_clamped():
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(2, 1, 2, 1, 64, [64, 64], torch.bfloat16)
    d = qkv.cuda()
    view = place(k, v, [64, 64], "whole", 0)
    args = (d[:, :, :2], d[:, :, 2:3], d[:, :, 3:], kva.DraftTree.chain(2, 1, "cuda"), view)
    full = kva.tree_attention(*args)
    view.lengths.copy_(torch.tensor([1000, -7], dtype=torch.int32))
    got = kva.tree_attention(*args)
    assert torch.equal(got[0], full[0])
    assert torch.equal(got[1, 0], d[1, 0, 3:].expand(2, 64))  # its own value alone


# ------------------------------------------------------------------- eviction

def evict_case(B, H, D, lens, budget, sinks, recent, layout="whole", page=16, weights=None, dtype=torch.bfloat16):
    from voom_b200.runtime import kv_attention as kva

    _, k, v = inputs(B, 1, H, H, D, lens, dtype)
    cap = max(max(lens), 1)
    if weights is None:
        weights = torch.round(torch.rand((B, H, cap), generator=torch.Generator().manual_seed(4)) * 50) / 8
    view = place(k, v, lens, layout, page)
    sums = torch.nn.functional.pad(weights, (0, max(0, view.max_len - cap)), value=9.0)
    e = kva.kv_evict(view, sums.cuda(), budget=budget, sinks=sinks, recent=recent)
    assert e.lengths.tolist() == [min(x, budget) for x in lens]
    for b, x in enumerate(lens):
        for h in range(H):
            want = oa.kept(weights[b, h].tolist(), x, budget, sinks, recent)
            m = len(want)
            assert e.index[b, h].tolist() == want + [-1] * (budget - m)
            assert torch.equal(e.k[b, h, :m].cpu(), k[b, h, want]) and torch.equal(e.v[b, h, :m].cpu(), v[b, h, want])
            got, ref = e.weights[b, h].cpu(), weights[b, h, want]
            assert torch.equal(got[:m].nan_to_num(nan=-7.0), ref.nan_to_num(nan=-7.0))
            assert not e.k[b, h, m:].any() and not e.v[b, h, m:].any() and not e.weights[b, h, m:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("layout,page", [("whole", 0), ("strided", 0), ("pool", 16), ("pool", 7), ("pages", 48)])
def test_evict_layouts(layout, page):
    evict_case(3, 2, 64, [300, 0, 90], 100, 4, 17, layout, page)
    evict_case(2, 3, 80, [257, 129], 128, 0, 0, layout, page, dtype=torch.float16)


@pytest.mark.gpu
@pytest.mark.parametrize("length,budget,sinks,recent", [
    (1, 1, 0, 0), (2, 1, 1, 0), (2, 1, 0, 1), (5, 4, 2, 2), (1024, 1023, 0, 0), (1025, 1, 0, 0), (1025, 1024, 4, 1020),
    (2047, 513, 0, 512), (4096, 4096, 4, 64), (4097, 4096, 4, 64), (40000, 3000, 4, 100), (140000, 70001, 1, 0)])
def test_evict_sizes(length, budget, sinks, recent):
    evict_case(1, 2, 16, [length], budget, sinks, recent)


@pytest.mark.gpu
def test_evict_ties_and_odd_weights():
    for w in (torch.zeros(1, 1, 3000), torch.full((1, 1, 3000), -1.5),
              torch.arange(3000.0).flip(0).view(1, 1, -1), -torch.arange(3000.0).view(1, 1, -1)):
        evict_case(1, 1, 8, [3000], 1000, 3, 10, weights=w)
    g = torch.Generator().manual_seed(6)
    w = torch.randn((1, 1, 5000), generator=g)
    w[0, 0, ::7] = -0.0
    w[0, 0, ::11] = 0.0
    w[0, 0, ::501] = math.nan
    w[0, 0, 5::502] = math.inf
    w[0, 0, 6::503] = -math.inf
    w[0, 0, 7::97] = 1e-42
    for budget in (5, 20, 2500, 4999):
        evict_case(1, 1, 8, [5000], budget, 1, 1, weights=w)


# ------------------------------------------------------------------- refusals

def test_c_entries_refuse_bad_arguments(built_lib):
    from voom_b200._lib import KvEvictArgs, KvViewStruct, TreeAttentionArgs

    def view(**kw):
        c = KvViewStruct()
        c.k = c.v = c.len = 4096
        c.k_page = c.k_head = c.v_page = c.v_head = 64 * 64
        c.k_pos = c.v_pos = 64
        c.B, c.hk, c.D, c.page, c.max_len = 1, 1, 64, 64, 64
        for a, b in kw.items():
            setattr(c, a, b)
        return c

    def attn(c, **kw):
        a = TreeAttentionArgs()
        a.q = a.kn = a.vn = a.out = 4096
        a.n, a.hq, a.scale = 0, 1, 0.125
        for x, y in kw.items():
            setattr(a, x, y)
        return built_lib.voom_tree_attention(ctypes.byref(c), ctypes.byref(a), None, 0, None)

    assert attn(view()) == 0  # no new tokens: nothing to do
    assert built_lib.voom_tree_attention(None, None, None, 0, None) == -1
    assert attn(view(k=None)) == -1 and attn(view(len=None)) == -1 and attn(view(B=0)) == -1
    assert attn(view(k=4104)) == -1 and attn(view(k_pos=60)) == -1  # rows off 16 bytes
    assert attn(view(D=60)) == -4 and attn(view(D=264)) == -4
    assert attn(view(type=2)) == -1
    assert attn(view(max_len=65)) == -1  # more than the cache holds
    assert attn(view(table=4096, offsets=4096)) == -1
    assert attn(view(), q=None) == -1 and attn(view(), q=4100) == -1 and attn(view(), q_t=12) == -1
    assert attn(view(hk=2), hq=3) == -1
    assert attn(view(), scale=0.0) == -1 and attn(view(), scale=-1.0) == -1 and attn(view(), scale=math.nan) == -1
    assert attn(view(), n=2000, mask=4096) == -3
    assert built_lib.voom_tree_mask(None, 1, 1, None, None, None) == -1
    assert built_lib.voom_tree_mask(4096, 1, 1025, 4096, 4096, None) == -3
    assert built_lib.voom_tree_mask(4096, 0, 5, 4096, 4096, None) == 0

    def evict(c, **kw):
        a = KvEvictArgs()
        a.weights = a.k_out = a.v_out = a.w_out = a.index = a.len_out = 4096
        a.budget = 4
        for x, y in kw.items():
            setattr(a, x, y)
        return built_lib.voom_kv_evict(ctypes.byref(c), ctypes.byref(a), None)

    assert evict(view(), weights=None) == -1 and evict(view(), k_out=4100) == -1
    assert evict(view(), budget=0) == -1 and evict(view(), sinks=3, recent=2) == -1
    assert evict(view(D=7)) == -4


@pytest.mark.gpu
def test_refusals():
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(1, 3, 4, 2, 64, [20], torch.bfloat16)
    d, k, v = qkv.cuda(), k.cuda(), v.cuda()
    length = torch.tensor([20], dtype=torch.int32, device="cuda")
    view = kva.KVView.contiguous(k, v, length)
    tree = kva.DraftTree.chain(1, 3, "cuda")
    q, kn, vn = d[:, :, :4], d[:, :, 4:6], d[:, :, 6:]
    with pytest.raises(ValueError, match="BF16 or FP16"):
        kva.KVView.contiguous(k.float(), v.float(), length)
    with pytest.raises(ValueError, match="head size"):
        kva.KVView.contiguous(k[..., :1].repeat(1, 1, 1, 264), v[..., :1].repeat(1, 1, 1, 264), length)
    with pytest.raises(ValueError, match="lengths"):
        kva.KVView.contiguous(k, v, length.long())
    with pytest.raises(ValueError, match="max_len"):
        kva.KVView.contiguous(k, v, length, max_len=21)
    with pytest.raises(ValueError, match="16 bytes"):
        kva.KVView.contiguous(k[..., 4:36], v[..., 4:36], length)
    with pytest.raises(ValueError, match="table"):
        kva.KVView.pool(k, v, torch.zeros((1, 1), device="cuda"), length)
    with pytest.raises(ValueError, match="one shape"):
        kva.KVView.pages([[(k, v), (k[:, :, :8], v[:, :, :8])]], length)
    with pytest.raises(ValueError, match="new tokens in q"):
        kva.tree_attention(q, kn, vn, kva.DraftTree.chain(1, 2, "cuda"), view)
    with pytest.raises(ValueError, match="do not divide"):
        kva.tree_attention(q[:, :, :3], kn, vn, tree, view)
    with pytest.raises(ValueError, match="scale"):
        kva.tree_attention(q, kn, vn, tree, view, scale=-1.0)
    with pytest.raises(ValueError, match="k: "):
        kva.tree_attention(q, kn[:, :, :1], vn, tree, view)
    with pytest.raises(ValueError, match="v: "):
        kva.tree_attention(q, kn, vn.half(), tree, view)
    with pytest.raises(ValueError, match="weights"):
        kva.tree_attention(q, kn, vn, tree, view, weights=torch.zeros((1, 2, 22), device="cuda"))
    with pytest.raises(ValueError, match="token_weight"):
        kva.tree_attention(q, kn, vn, tree, view, token_weight=torch.zeros((1, 3), device="cuda"))
    with pytest.raises(ValueError, match="parents"):
        kva.DraftTree(torch.zeros((1, 3), device="cuda"))
    with pytest.raises(ValueError, match="at most 1024"):
        kva.DraftTree(torch.zeros((1, 1025), dtype=torch.int32, device="cuda"))
    with pytest.raises(ValueError, match="budget"):
        kva.kv_evict(view, torch.zeros((1, 2, 20), device="cuda"), budget=4, sinks=3, recent=2)
    with pytest.raises(ValueError, match="weights"):
        kva.kv_evict(view, torch.zeros((1, 2, 19), device="cuda"), budget=4, sinks=1)
