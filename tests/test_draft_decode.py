"""The operators together: drafted trees over a PagedKVCache, evicted.

A tree step must give each token what decoding its path token by token gives,
up to BF16 rounding of the layers' outputs (2^-8 of values of a few units, a few
layers deep: 0.1)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def _stack(layers=2):
    from examples.draft_decode import AttentionStack

    return AttentionStack(layers, 192, 6, 2, 64, "cuda", seed=3)


def _kv(tmp_path, name, **kw):
    from voom_b200.runtime.kv_paged import PagedKVCache

    return PagedKVCache(2, kw.pop("max_bytes", 1 << 40), tmp_path / name, page_positions=16, **kw)


def _feed(stack, kv, sums, x):
    from voom_b200.runtime.kv_attention import DraftTree

    y, new = stack.step(x, DraftTree.chain(1, x.shape[0], "cuda"), kv, sums)
    stack.commit(new, torch.arange(x.shape[0], device="cuda"), kv, sums)
    return y


def _sums():
    return [torch.zeros((2, 256), device="cuda") for _ in range(2)]


@pytest.mark.parametrize("compress", [False, True])
def test_tree_step_equals_paths_token_by_token(tmp_path, compress):
    from voom_b200.runtime.kv_attention import DraftTree

    stack = _stack()
    g = torch.Generator(device="cuda").manual_seed(5)
    prompt = torch.randn((53, 192), device="cuda", generator=g).to(torch.bfloat16)
    drafts = torch.randn((7, 192), device="cuda", generator=g).to(torch.bfloat16)
    parents = [-1, 0, 0, 1, 2, 2, 5]
    # a budget of a few pages: old pages are spilled, and reloaded for every view
    kv = _kv(tmp_path, "tree", max_bytes=40000, compress_spill=compress)
    sums = _sums()
    _feed(stack, kv, sums, prompt)
    assert kv.stats.spills > 0
    y, new = stack.step(drafts, DraftTree(torch.tensor([parents], dtype=torch.int32, device="cuda")), kv, sums)
    for leaf in (3, 4, 6):
        path = []
        j = leaf
        while j >= 0:
            path.append(j)
            j = parents[j]
        path = path[::-1]
        kv2, s2 = _kv(tmp_path, f"path{leaf}"), _sums()
        _feed(stack, kv2, s2, prompt)
        for t, i in enumerate(path):
            z = _feed(stack, kv2, s2, drafts[i:i + 1])
            assert float((z.float() - y[i:i + 1].float()).abs().max()) < 0.1, (leaf, t)
    # what commit stores is the path's, and its weight moves with it
    before = [s.clone() for s in sums]
    stack.commit(new, torch.tensor([0, 2, 5], device="cuda"), kv, sums)
    assert kv.length(0) == 56 and kv.offset == 56
    for s, b in zip(sums, before):
        assert torch.equal(s[:, 53:56], b[:, [53, 55, 58]]) and not s[:, 56:].any()


def test_views_equal_update(tmp_path):
    """The pages in place hold what update() puts together."""
    from voom_b200.runtime.kv_attention import DraftTree, KVView, tree_attention

    g = torch.Generator(device="cuda").manual_seed(1)
    kv = _kv(tmp_path, "a", max_bytes=20000, compress_spill=True)
    for n in (5, 30, 16, 1):
        k, v = (torch.randn((1, 2, n, 64), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
        for layer in range(2):
            K, V = kv.update(layer, k, v)
    q = torch.randn((1, 3, 4, 64), device="cuda", generator=g).to(torch.bfloat16)
    kn, vn = (torch.randn((1, 3, 2, 64), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    tree = DraftTree.chain(1, 3, "cuda")
    whole = KVView.contiguous(K, V, torch.tensor([52], dtype=torch.int32, device="cuda"))
    assert torch.equal(tree_attention(q, kn, vn, tree, kv.view(1)), tree_attention(q, kn, vn, tree, whole))
    w = torch.rand((1, 2, 60), device="cuda", generator=g)
    e = kv.evict(1, w, budget=20, sinks=2, recent=4)
    assert kv.length(1) == 20 and kv.offset == 52 and kv.length(0) == 52
    for h in range(2):
        at = e.index[0, h].long()
        assert torch.equal(e.k[0, h], K[0, h, at]) and torch.equal(e.v[0, h], V[0, h, at])
    K2, _ = kv.update(1, K[:, :, :3], V[:, :, :3])
    assert torch.equal(K2[:, :, :20], e.k) and torch.equal(K2[:, :, 20:], K[:, :, :3])
    kv.release()
    assert not list((tmp_path / "a").iterdir())


def test_example_runs():
    from examples.draft_decode import run

    r = run(layers=2, prompt=300, steps=6, budget=128, drafts=9, page_positions=16)
    assert r["offset"] == 300 + r["accepted"] and r["accepted"] >= 6
    assert all(128 <= n <= 128 + 9 for n in r["lengths"])
    assert bool(torch.isfinite(r["hidden"].float()).all())
    for s in r["sums"]:  # every token spread a weight of one per query head over some positions
        assert bool((s >= 0).all()) and float(s.sum()) > 0


def test_view_of_nothing_is_refused(tmp_path):
    with pytest.raises(ValueError, match="no positions"):
        _kv(tmp_path, "none").view(0)
