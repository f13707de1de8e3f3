"""PagedKVCache as the attention and the eviction read and write it: pages of
their own, one key head, spilled pages, evictions that leave many pages."""

from __future__ import annotations

import pytest
import torch


def _plain(t):
    return t.stride() == torch.empty(t.shape, device="meta").stride() and \
        t.untyped_storage().nbytes() == t.numel() * t.element_size()


@pytest.mark.parametrize("hk", [1, 2])
@pytest.mark.parametrize("sizes", [(53,), (16,), (5, 30, 16, 1), (15, 1, 64)])
def test_pages_are_pieces_of_their_own(tmp_path, hk, sizes):
    """Plain strides, and no page holds the bytes of its neighbours."""
    from voom_b200.runtime.kv_paged import PagedKVCache

    kv = PagedKVCache(1, 1 << 40, tmp_path, page_positions=16)
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn((1, hk, sum(sizes), 64), generator=g).to(torch.bfloat16) for _ in range(2))
    at = 0
    for n in sizes:
        K, V = kv.update(0, k[:, :, at:at + n].clone(), v[:, :, at:at + n].clone())
        at += n
        assert torch.equal(K, k[:, :, :at]) and torch.equal(V, v[:, :, :at])
        assert kv.length(0) == at == kv.offset and len(kv._pages[0]) == at // 16
    assert all(_plain(x) for p in kv._pages[0] for x in (p.k, p.v))


@pytest.mark.gpu
@pytest.mark.parametrize("compress", [False, True])
@pytest.mark.parametrize("hk,n", [(1, 53), (1, 16), (2, 160)])
def test_pages_of_one_key_head_in_place_and_evicted(tmp_path, compress, hk, n):
    """One key head, a prompt longer than a page, spilled pages, and an eviction that leaves many pages."""
    from voom_b200.runtime.kv_attention import DraftTree, KVView, tree_attention
    from voom_b200.runtime.kv_paged import PagedKVCache

    g = torch.Generator(device="cuda").manual_seed(1)
    kv = PagedKVCache(1, 20000, tmp_path / "a", page_positions=16, compress_spill=compress)
    k, v = (torch.randn((1, hk, n, 64), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    K, V = kv.update(0, k, v)
    assert torch.equal(K, k) and torch.equal(V, v)
    q = torch.randn((1, 3, 4, 64), device="cuda", generator=g).to(torch.bfloat16)
    kn, vn = (torch.randn((1, 3, hk, 64), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    tree = DraftTree.chain(1, 3, "cuda")
    whole = KVView.contiguous(K, V, torch.tensor([n], dtype=torch.int32, device="cuda"))
    assert torch.equal(tree_attention(q, kn, vn, tree, kv.view(0)), tree_attention(q, kn, vn, tree, whole))
    w = torch.rand((1, hk, n), device="cuda", generator=g)
    m = n - 5
    e = kv.evict(0, w, budget=m, sinks=2, recent=4)
    assert kv.length(0) == m
    K2, V2 = kv.update(0, k[:, :, :3], v[:, :, :3])
    assert torch.equal(K2[:, :, :m], e.k) and torch.equal(V2[:, :, :m], e.v) and torch.equal(K2[:, :, m:], k[:, :, :3])


@pytest.mark.gpu
@pytest.mark.parametrize("compress", [False, True])
def test_evict_keeps_the_byte_budget(tmp_path, compress):
    """Pages that were reloaded for the eviction do not stay beyond the budget."""
    from voom_b200.runtime.kv_paged import PagedKVCache

    g = torch.Generator(device="cuda").manual_seed(2)
    limit = 60000
    kv = PagedKVCache(2, limit, tmp_path / "a", page_positions=16, compress_spill=compress)
    k, v = (torch.randn((1, 2, 300, 64), device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    for layer in range(2):
        kv.append(layer, k, v)
    assert kv.nbytes() <= limit
    w = torch.rand((1, 2, 300), device="cuda", generator=g)
    kept = []
    for layer in range(2):
        kept.append(kv.evict(layer, w, budget=250, sinks=2, recent=4))
        assert kv.nbytes() <= limit, layer
    for layer in range(2):  # what was spilled again comes back, and later files are not the deleted ones
        K, V = kv.update(layer, k[:, :, :1], v[:, :, :1])
        assert torch.equal(K[:, :, :250], kept[layer].k) and torch.equal(V[:, :, :250], kept[layer].v)
        assert torch.equal(K[:, :, 250:], k[:, :, :1])
    kv.release()
    assert not list((tmp_path / "a").iterdir())


def test_evict_keeps_the_byte_budget_on_the_host(tmp_path, monkeypatch):
    """The same bookkeeping without a GPU: the eviction itself is a stand-in that keeps the first positions."""
    from voom_b200.runtime import kv_attention
    from voom_b200.runtime.kv_paged import PagedKVCache

    kv = PagedKVCache(1, 20000, tmp_path, page_positions=16)
    k = torch.randn((1, 2, 100, 64)).to(torch.bfloat16)
    kv.append(0, k, k)
    assert kv.nbytes() <= 20000

    def evict(view, weights, *, budget, sinks, recent):
        n = torch.arange(budget, dtype=torch.int32).expand(1, 2, -1)
        return kv_attention.Evicted(k[:, :, :budget], k[:, :, :budget], weights[..., :budget], n, torch.tensor([budget]))

    monkeypatch.setattr(kv_attention, "kv_evict", evict)
    monkeypatch.setattr(PagedKVCache, "view", lambda self, layer: None)
    kv.evict(0, torch.zeros((1, 2, 100)), budget=90)
    assert kv.length(0) == 90 and kv.nbytes() <= 20000
    K, _ = kv.update(0, k[:, :, :1], k[:, :, :1])
    assert torch.equal(K, torch.cat((k[:, :, :90], k[:, :, :1]), 2))


def test_a_wait_that_ran_out_is_reported_by_the_cache(tmp_path, monkeypatch):
    """All views share the cache's status word; a kernel's report (here: the test's) reaches check_status()."""
    from voom_b200.runtime import kv_attention
    from voom_b200.runtime.kv_paged import PagedKVCache

    words = []
    monkeypatch.setattr(kv_attention.KVView, "pages", classmethod(lambda cls, *a, status=None, **kw: words.append(status)))
    kv = PagedKVCache(2, 1 << 40, tmp_path, page_positions=16)
    kv.check_status()  # no view yet
    k = torch.zeros((1, 2, 20, 64), dtype=torch.bfloat16)
    for layer in range(2):
        kv.append(layer, k, k)
        kv.view(layer)
    kv.check_status()
    words[0].fill_(1)  # a view that is gone by now
    kv.view(1)
    assert all(w is words[0] for w in words)
    with pytest.raises(RuntimeError, match="ran out"):
        kv.check_status()
    kv.check_status()


@pytest.mark.gpu
def test_views_of_a_cache_report_to_one_word(tmp_path):
    from voom_b200.runtime.kv_paged import PagedKVCache

    kv = PagedKVCache(1, 1 << 40, tmp_path, page_positions=16)
    k = torch.zeros((1, 2, 20, 64), dtype=torch.bfloat16, device="cuda")
    kv.append(0, k, k)
    a, b = kv.view(0), kv.view(0)
    assert a.status_ptr == b.status_ptr == kv._status.data_ptr()
    assert a.struct.k is not None and a.status.dtype == torch.int32
    a.status.fill_(1)
    with pytest.raises(RuntimeError, match="ran out"):
        kv.check_status()
    b.check_status()


@pytest.mark.gpu
def test_view_of_resident_pages_does_not_wait(tmp_path):
    from voom_b200.runtime.kv_attention import DraftTree, tree_attention
    from voom_b200.runtime.kv_paged import PagedKVCache

    kv = PagedKVCache(1, 1 << 40, tmp_path / "a", page_positions=16)
    k = torch.randn((1, 2, 53, 64), device="cuda").to(torch.bfloat16)
    kv.append(0, k, k)
    q = torch.randn((1, 1, 4, 64), device="cuda").to(torch.bfloat16)
    tree = DraftTree.chain(1, 1, "cuda")
    tree_attention(q, k[:, :, :1].transpose(1, 2), k[:, :, :1].transpose(1, 2), tree, kv.view(0))
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        tree_attention(q, k[:, :, :1].transpose(1, 2), k[:, :, :1].transpose(1, 2), tree, kv.view(0))
    finally:
        torch.cuda.set_sync_debug_mode(mode)


@pytest.mark.gpu
def test_a_view_that_holds_copies_is_not_written_to(tmp_path):
    """kv_append to a cache's view would go into a copy of its open page: it is refused, and the cache stays as it is."""
    from voom_b200.runtime.kv_attention import KVView
    from voom_b200.runtime.kv_paged import PagedKVCache
    from voom_b200.runtime.kv_pool import kv_append

    k, v = (torch.randn((1, 2, 37, 64), device="cuda").bfloat16() for _ in range(2))
    x = torch.randn((1, 3, 2, 64), device="cuda").bfloat16()
    for n in (5, 32, 37):  # an open page alone, none, and both kinds
        kv = PagedKVCache(1, 1 << 40, tmp_path, page_positions=16)
        kv.append(0, k[:, :, :n], v[:, :, :n])
        with pytest.raises(ValueError, match="append"):
            kv_append(kv.view(0), x, x)
        K, V = kv.update(0, x.transpose(1, 2), x.transpose(1, 2))
        assert torch.equal(K[:, :, :n], k[:, :, :n]) and torch.equal(K[:, :, n:], x.transpose(1, 2))
    # pages of the caller's own are written to
    pages = [[(k[:, :, :16].clone(), v[:, :, :16].clone())]]
    view = KVView.pages(pages, torch.tensor([4], dtype=torch.int32, device="cuda"))
    kv_append(view, x, x)
    assert torch.equal(pages[0][0][0][:, :, 4:7], x.transpose(1, 2))


@pytest.mark.gpu
def test_slopes_and_windows_are_refused_after_an_eviction(tmp_path):
    """An index is no position any more, and its distance would be wrong in silence; a cap does not ask for it."""
    from voom_b200.runtime.kv_attention import DraftTree, KVView, kv_evict, tree_attention
    from voom_b200.runtime.kv_paged import PagedKVCache

    k, v = (torch.randn((1, 2, 40, 64), device="cuda").bfloat16() for _ in range(2))
    x = torch.randn((1, 3, 8, 64), device="cuda").bfloat16()
    args = (x[:, :, :4], x[:, :, 4:6], x[:, :, 6:])
    tree = DraftTree.chain(1, 3, "cuda")
    slopes = torch.rand(4, device="cuda")
    kv = PagedKVCache(2, 1 << 40, tmp_path, page_positions=16)
    for layer in range(2):
        kv.append(layer, k, v)
    w = torch.rand((1, 2, 40), device="cuda")
    kv.evict(0, w, budget=64)  # keeps all: nothing moves
    whole = KVView.contiguous(k, v, torch.tensor([40], dtype=torch.int32, device="cuda"))
    for layer in range(2):
        for kw in (dict(window=9), dict(slopes=slopes), dict(cap=9.0)):
            assert torch.equal(tree_attention(*args, tree, kv.view(layer), **kw), tree_attention(*args, tree, whole, **kw))
    kv.evict(0, w, budget=30, sinks=2, recent=4)
    e = kv_evict(whole, w, budget=30, sinks=2, recent=4)
    kept = KVView.contiguous(e.k, e.v, e.lengths, displaced=True)
    for view in (kv.view(0), kept):
        for kw in (dict(window=9), dict(slopes=slopes), dict(window=9, cap=5.0)):
            with pytest.raises(ValueError, match="eviction"):
                tree_attention(*args, tree, view, **kw)
    assert torch.equal(tree_attention(*args, tree, kv.view(0), cap=9.0), tree_attention(*args, tree, kept, cap=9.0))
    tree_attention(*args, tree, kv.view(1), window=9)  # the other layer has not been cut
    kv.append(0, k, v)
    with pytest.raises(ValueError, match="eviction"):
        tree_attention(*args, tree, kv.view(0), window=9)
    kv.release()
    kv.append(0, k, v)
    tree_attention(*args, tree, kv.view(0), window=9)
