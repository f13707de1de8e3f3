"""Cache attention and eviction where lengths, pages, masks and workspaces are at
their edges, against the definitions in 64 bits.  Tolerances as in
test_kv_attention.py; those that are tighter or exact say why."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import attention as oa
from tests.test_kv_attention import STEP, check, inputs, place


def poison(view):
    """The view's workspaces filled with NaN: whatever a call does not write, it must not read."""
    for t in view._scratch.values():
        t.fill_(255)


@pytest.mark.gpu
@pytest.mark.parametrize("lens", [[100], [1], [0], [33, 0, 5], [700, 64]])
@pytest.mark.parametrize("n,g,D", [(1, 1, 64), (1, 4, 128), (2, 2, 256), (12, 2, 64), (40, 4, 128), (20, 2, 256), (300, 1, 64)])
def test_lengths_far_below_the_bound(lens, n, g, D):
    """The blocks are laid out for max_len; with fewer steps than blocks, those without one leave nothing to join."""
    from voom_b200.runtime import kv_attention as kva

    cap = 24000
    B = len(lens)
    qkv, _, _ = inputs(B, n, g, 1, D, [1], torch.bfloat16)
    gen = torch.Generator(device="cuda").manual_seed(7)
    k, v = (torch.randn((B, 1, cap, D), device="cuda", generator=gen).to(torch.bfloat16) for _ in range(2))
    view = kva.KVView.contiguous(k, v, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    tree = kva.DraftTree.chain(B, n, "cuda")
    d = qkv.cuda()
    for call in range(2):
        w = torch.zeros((B, 1, cap + n), device="cuda")
        poison(view)  # the second call's workspace
        out, lse = kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], tree, view, weights=w,
                                      return_lse=True)
    sees = oa.tree_sees(list(range(-1, n - 1)))
    for b, x in enumerate(lens):
        o, l, s = oa.attention(qkv[b, :, :g], qkv[b, :, g:g + 1], qkv[b, :, g + 1:], sees, k[b, :, :x].cpu(),
                               v[b, :, :x].cpu(), D ** -0.5)
        big = max(float(qkv[b, :, g + 1:].abs().max()), float(v[b, :, :max(x, 1)].abs().max()))
        check(out[b], o, 2 * STEP[torch.bfloat16] * big, ("out", b))
        check(lse[b], l, 3e-5, ("lse", b))
        check(w[b, :, :x + n], s, 5e-5 * (n * g) ** 0.5 + 1e-6, ("weights", b))
        assert not w[b, :, x + n:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("n,g", [(1, 2), (40, 4)])
def test_a_captured_graph_keeps_its_workspace(n, g):
    """A larger call on the same stream and view must not give a captured call's workspace to other tensors."""
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(1, 90, g, 1, 128, [6000], torch.bfloat16)
    d = qkv.cuda()
    view = place(k, v, [6000], "whole", 0)

    def call(m, **kw):
        x = d[:, :m]
        return kva.tree_attention(x[:, :, :g], x[:, :, g:g + 1], x[:, :, g + 1:], kva.DraftTree.chain(1, m, "cuda"), view,
                                  **kw)

    want = call(n)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(n)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = call(n)
    with torch.cuda.stream(side):
        w = torch.zeros((1, 1, view.max_len + 90), device="cuda")
        call(90, weights=w)
        call(3, weights=w)
        others = [torch.full((size,), 7, dtype=torch.uint8, device="cuda")
                  for size in (1 << 12, 1 << 16, 1 << 18, 1 << 20, 1 << 21, 1 << 22, 1 << 23, 1 << 24, 1 << 25) for _ in range(4)]
    torch.cuda.synchronize()
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    for t in others:
        assert bool((t == 7).all())


@pytest.mark.gpu
def test_threads_on_one_stream_do_not_mix_their_calls():
    """Two host threads, one stream, one view: the launches of a call stay together."""
    import threading

    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(1, 2, 8, 2, 128, [9000], torch.bfloat16)
    d = qkv.cuda()
    view = place(k, v, [9000], "whole", 0)
    tree = kva.DraftTree.chain(1, 1, "cuda")
    stream = torch.cuda.current_stream()

    def call(i):
        x = d[:, i:i + 1]
        return kva.tree_attention(x[:, :, :8], x[:, :, 8:10], x[:, :, 10:], tree, view)

    want = [call(0), call(1)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(stream):
            got = [call(i) for _ in range(300)]
            torch.cuda.synchronize()
            wrong.extend(i for x in got if not torch.equal(x, want[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.gpu
@pytest.mark.parametrize("n,g,D", [(1, 4, 64), (40, 4, 128), (20, 2, 256)])
def test_a_length_past_a_requests_own_pages_reads_zeros(n, g, D):
    """Requests of unequal page lists: what a request has no page for is zero keys and values, never another's."""
    from voom_b200.runtime import kv_attention as kva

    page, lists = 16, [9, 2, 0]
    gen = torch.Generator().manual_seed(5)
    k, v = (torch.randn((3, 9 * page, D), generator=gen).to(torch.bfloat16) for _ in range(2))
    for b, m in enumerate(lists):
        k[b, m * page:] = 0
        v[b, m * page:] = 0

    def cut(x, b, p):
        return x[b, p * page:(p + 1) * page].cuda()[None, None]

    view = kva.KVView.pages([[(cut(k, b, p), cut(v, b, p)) for p in range(m)] for b, m in enumerate(lists)],
                            torch.tensor([140, 140, 20], dtype=torch.int32, device="cuda"))
    qkv, _, _ = inputs(3, n, g, 1, D, [1], torch.bfloat16)
    d = qkv.cuda()
    out, lse = kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], kva.DraftTree.chain(3, n, "cuda"), view,
                                  return_lse=True)
    sees = oa.tree_sees(list(range(-1, n - 1)))
    for b, x in enumerate([140, 140, 20]):
        o, l, _ = oa.attention(qkv[b, :, :g], qkv[b, :, g:g + 1], qkv[b, :, g + 1:], sees, k[b:b + 1, :x], v[b:b + 1, :x],
                               D ** -0.5)
        check(out[b], o, 2 * STEP[torch.bfloat16] * 6.0, ("out", b))
        check(lse[b], l, 3e-5, ("lse", b))
    w = torch.rand((3, 1, 9 * page), generator=gen)
    e = kva.kv_evict(view, w.cuda(), budget=50, sinks=2, recent=3)
    for b, x in enumerate([140, 140, 20]):
        want = oa.kept(w[b, 0].tolist(), x, 50, 2, 3)
        assert torch.equal(e.k[b, 0, :len(want)].cpu(), k[b, want]) and torch.equal(e.v[b, 0, :len(want)].cpu(), v[b, want])


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 5])  # through TMA, and gathered
@pytest.mark.parametrize("n,g", [(1, 4), (40, 4)])
def test_a_pool_entry_that_is_no_page_reads_zeros(page, n, g):
    from voom_b200.runtime import kv_attention as kva

    L, D = 400, 64
    per = L // page
    gen = torch.Generator().manual_seed(6)
    kp, vp = (torch.randn((per, 1, page, D), generator=gen).to(torch.bfloat16) for _ in range(2))
    table = torch.arange(per, dtype=torch.int32)
    for at, entry in ((1, -1), (per // 2, per), (per - 1, -7)):
        table[at] = entry
        kp[at] = 0
        vp[at] = 0
    kd, vd = kp.cuda(), vp.cuda()
    for at in (1, per // 2, per - 1):  # no entry names them
        kd[at] = math.nan
        vd[at] = math.nan
    view = kva.KVView.pool(kd, vd, table[None].cuda(), torch.tensor([L], dtype=torch.int32, device="cuda"))
    qkv, _, _ = inputs(1, n, g, 1, D, [1], torch.bfloat16)
    d = qkv.cuda()
    out = kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], kva.DraftTree.chain(1, n, "cuda"), view)
    o, _, _ = oa.attention(qkv[0, :, :g], qkv[0, :, g:g + 1], qkv[0, :, g + 1:], oa.tree_sees(list(range(-1, n - 1))),
                           kp.reshape(1, L, D), vp.reshape(1, L, D), D ** -0.5)
    check(out[0], o, 2 * STEP[torch.bfloat16] * 6.0, "out")
    e = kva.kv_evict(view, torch.zeros((1, 1, L), device="cuda"), budget=L - 1, sinks=0, recent=L - 1)
    assert torch.equal(e.k[0, 0].cpu(), kp.reshape(L, D)[1:]) and torch.equal(e.v[0, 0].cpu(), vp.reshape(L, D)[1:])


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,g,D", [(1, 1, 64), (1, 8, 128), (24, 1, 64), (40, 4, 64), (80, 4, 64), (20, 1, 256)])
def test_denominator_of_many_small_weights_beside_a_large_one(dtype, n, g, D):
    """Half a million positions of 2^-25 each of the row's largest, 2^-6 of the row together: added to it one by
    one in fp32 they would not count.  160 requests read one cache, so that a block has a whole unit."""
    from voom_b200.runtime import kv_attention as kva

    B, page, L = 160, 1 << 13, 1 << 19
    k, v = (torch.zeros((L // page, 1, page, D), dtype=dtype, device="cuda") for _ in range(2))
    k[0, 0, 0, 0] = 25.1 * math.log(2.0)
    table = torch.arange(L // page, dtype=torch.int32, device="cuda").expand(B, -1).contiguous()
    view = kva.KVView.pool(k, v, table, torch.full((B,), L, dtype=torch.int32, device="cuda"))
    q = torch.zeros((B, n, g, D), dtype=dtype, device="cuda")
    q[..., 0] = 1.0
    new = torch.zeros((B, n, 1, D), dtype=dtype, device="cuda")
    _, lse = kva.tree_attention(q, new, new, kva.DraftTree.chain(B, n, "cuda"), view, scale=1.0, return_lse=True)
    top = math.exp(float(k[0, 0, 0, 0]))
    for i in (0, n - 1):
        want = math.log(top + (L - 1) + (i + 1))
        assert float((lse[:, i].double() - want).abs().max()) <= 3e-5, i


@pytest.mark.gpu
@pytest.mark.parametrize("n,g,D,L", [(1, 1, 64, 1 << 19), (40, 4, 64, 1 << 17), (80, 4, 64, 1 << 17), (20, 1, 256, 1 << 17)])
def test_fp16_many_small_probabilities_beside_a_large_one(n, g, D, L):
    """One position takes nearly all of a row's weight, the others 2^-25 of it each: too small for FP16 by
    themselves, 2^-6 or 2^-8 of the row together.  160 requests read one cache, so that a block has a whole unit."""
    from voom_b200.runtime import kv_attention as kva

    B, page = 160, 1 << 13
    k, v = (torch.zeros((L // page, 1, page, D), dtype=torch.float16, device="cuda") for _ in range(2))
    v[..., 0] = 1.0
    k[0, 0, 0, 0], v[0, 0, 0, 0] = 25.1 * math.log(2.0), 0.0
    table = torch.arange(L // page, dtype=torch.int32, device="cuda").expand(B, -1).contiguous()
    view = kva.KVView.pool(k, v, table, torch.full((B,), L, dtype=torch.int32, device="cuda"))
    q = torch.zeros((B, n, g, D), dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    new = torch.zeros((B, n, 1, D), dtype=torch.float16, device="cuda")
    out, lse = kva.tree_attention(q, new, new, kva.DraftTree.chain(B, n, "cuda"), view, scale=1.0, return_lse=True)
    top = math.exp(float(k[0, 0, 0, 0]))
    for i in (0, n - 1):
        total = top + (L - 1) + (i + 1)
        err = (out[:, i, :, 0].double() - (L - 1) / total).abs().max()
        assert float(err) <= 2 * STEP[torch.float16], (i, float(err), (L - 1) / total)
        assert float((lse[:, i].double() - math.log(total)).abs().max()) <= 3e-5


@pytest.mark.gpu
@pytest.mark.parametrize("n,g", [(3, 2), (20, 2)])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_token_weight_of_no_token_counts_for_nothing(n, g, bad):
    from voom_b200.runtime import kv_attention as kva

    par = [-1] * n
    par[1] = -2
    qkv, k, v = inputs(1, n, g, 1, 64, [50], torch.bfloat16)
    d = qkv.cuda()
    view = place(k, v, [50], "whole", 0)
    tree = kva.DraftTree(torch.tensor([par], dtype=torch.int32, device="cuda"))
    sums = []
    for x in (0.0, bad):
        tw = torch.ones((1, n), device="cuda")
        tw[0, 1] = x
        w = torch.zeros((1, 1, 50 + n), device="cuda")
        kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], tree, view, weights=w, token_weight=tw)
        sums.append(w)
    assert bool(torch.isfinite(sums[0]).all()) and torch.equal(sums[0], sums[1])


@pytest.mark.gpu
def test_evict_more_positions_than_shared_memory_holds():
    """Past 8 x 40960 positions of a head, the weights are read again in every pass."""
    from voom_b200.runtime import kv_attention as kva

    L, budget, sinks, recent = 330001, 5000, 3, 77
    gen = torch.Generator().manual_seed(2)
    w = torch.round(torch.rand((1, 1, L), generator=gen) * 1000) / 8
    k = torch.arange(L).remainder(251).to(torch.bfloat16)[None, None, :, None].expand(1, 1, L, 8).contiguous()
    view = kva.KVView.contiguous(k.cuda(), (-k).cuda(), torch.tensor([L], dtype=torch.int32, device="cuda"))
    e = kva.kv_evict(view, w.cuda(), budget=budget, sinks=sinks, recent=recent)
    want = oa.kept(w[0, 0].tolist(), L, budget, sinks, recent)
    assert e.index[0, 0].tolist() == want
    assert torch.equal(e.k[0, 0].cpu(), k[0, 0, want]) and torch.equal(e.weights[0, 0].cpu(), w[0, 0, want])


@pytest.mark.gpu
def test_a_graph_follows_lengths_far_below_its_bound():
    """A captured call over a cache laid out for 20000 positions, replayed as its lengths change."""
    from voom_b200.runtime import kv_attention as kva

    for n, g in ((1, 4), (40, 4)):
        qkv, k, v = inputs(2, n, g, 1, 64, [20000, 20000], torch.bfloat16)
        d, kd, vd = qkv.cuda(), k.cuda(), v.cuda()
        length = torch.tensor([20000, 3], dtype=torch.int32, device="cuda")
        view = kva.KVView.contiguous(kd, vd, length)
        tree = kva.DraftTree.chain(2, n, "cuda")
        args = (d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], tree)
        kva.tree_attention(*args, view)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = kva.tree_attention(*args, view)
        for lens in ([20000, 3], [0, 0], [1, 70], [5, 20000]):
            length.copy_(torch.tensor(lens, dtype=torch.int32))
            graph.replay()
            tight = kva.KVView.contiguous(kd, vd, length.clone(), max_len=max(lens))
            want = kva.tree_attention(*args, tight).float()
            big = max(float(v.abs().max()), float(qkv.abs().max()))
            assert float((out.float() - want).abs().max()) <= 4 * STEP[torch.bfloat16] * big, lens  # two roundings


@pytest.mark.gpu
@pytest.mark.parametrize("n,g", [(3, 2), (20, 2), (37, 8)])
def test_weights_at_an_infinite_key(n, g):
    """A key whose score is -inf for every row gets no weight, and rows that are no token change nothing."""
    from voom_b200.runtime import kv_attention as kva

    qkv, k, v = inputs(2, n, g, 1, 64, [50, 50], torch.bfloat16)
    qkv[:, :, :g, 0] = qkv[:, :, :g, 0].abs() + 0.5
    k[:, 0, 7, 0] = -math.inf
    d = qkv.cuda()
    view = place(k, v, [50, 50], "whole", 0)
    tree = kva.DraftTree(torch.tensor([[-1] * n, [-2] * n], dtype=torch.int32, device="cuda"))  # the second: no tokens at all
    w = torch.ones((2, 1, 50 + n), device="cuda")
    out, lse = kva.tree_attention(d[:, :, :g], d[:, :, g:g + 1], d[:, :, g + 1:], tree, view, weights=w, return_lse=True)
    assert bool((w[1] == 1).all()) and not out[1].any() and bool(torch.isneginf(lse[1]).all())
    o, l, s = oa.attention(qkv[0, :, :g], qkv[0, :, g:g + 1], qkv[0, :, g + 1:], oa.tree_sees([-1] * n), k[0], v[0], 64 ** -0.5)
    assert float(w[0, 0, 7]) == 1.0
    check(out[0], o, 2 * STEP[torch.bfloat16] * float(v.abs().max() + 1), "out")
    check(lse[0], l, 3e-5, "lse")
    check(w[0], 1.0 + s, 5e-5 * (n * g) ** 0.5 + 1e-6, "weights")
