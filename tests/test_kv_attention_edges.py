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
