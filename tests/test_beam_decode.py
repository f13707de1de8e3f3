"""The operators together: beams over a pool of shared pages.

What the pool's rows hold after forks, appends and attention must be each beam's own
history: feeding a beam's tokens to a fresh pool of one row gives the same hidden
states, up to the order of the attention's sums and BF16 rounding of the layers'
outputs (2^-8 of values of a few units, a few layers deep: 0.1)."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_beams_hold_their_own_histories():
    from examples import beam_decode as bd
    from examples.draft_decode import AttentionStack
    from voom_b200.runtime.kv_pool import PagePool

    stack = AttentionStack(3, 192, 6, 2, 64, "cuda", seed=3)
    g = torch.Generator(device="cuda").manual_seed(5)
    embed = torch.randn((100, 192), device="cuda", generator=g).to(torch.bfloat16)
    kw = dict(cap=30.0, window=10)
    prompt = torch.randint(0, 100, (21,), device="cuda", generator=g)
    pool = PagePool(3, 2, 64, pages=40, rows=3, max_len=64, page=8)
    pool.fork(grow=torch.tensor([21, 0, 0], dtype=torch.int32, device="cuda"))
    bd.step(stack, pool, embed[prompt].expand(3, -1, -1), **kw)
    pool.fork(torch.zeros(3, dtype=torch.int32, device="cuda"))
    history = [prompt.tolist()] * 3
    for i in range(12):
        parents = torch.randint(0, 3, (3,), device="cuda", generator=g).to(torch.int32)
        tokens = torch.randint(0, 100, (3,), device="cuda", generator=g)
        pool.fork(parents, grow=1)
        hidden = bd.step(stack, pool, embed[tokens][:, None], **kw)[:, -1]
        history = [history[p] + [t] for p, t in zip(parents.tolist(), tokens.tolist())]
    pool.check_status()
    for r in range(3):
        alone = PagePool(3, 2, 64, pages=8, rows=1, max_len=64, page=8)
        alone.fork(grow=len(history[r]))
        want = bd.step(stack, alone, embed[torch.tensor(history[r], device="cuda")][None], **kw)[0, -1]
        assert float((hidden[r] - want).float().abs().max()) < 0.1, r


def test_example_runs():
    from examples.beam_decode import run

    r = run(batch=2, beams=3, layers=2, prompt=70, steps=9, window=20)
    assert r["tokens"].shape == (2, 3, 9) and bool(torch.isfinite(r["scores"]).all())
    s = r["scores"]
    assert bool((s[:, :-1] >= s[:, 1:]).all())  # the best first
    assert len({tuple(x) for x in r["tokens"].view(6, 9).tolist()[:3]}) == 3  # a request's beams differ
    assert r["pages"] < r["unshared"]


def test_example_reads_a_prompt_once_and_leaves_empty_rows_empty(monkeypatch):
    """The pool's contract: only rows that were written to are advanced; a prompt is one row's work."""
    from examples import beam_decode as bd
    from voom_b200.runtime.kv_pool import PagePool

    asked, lengths = [], []
    attend, fork = bd.tree_attention, PagePool.fork
    monkeypatch.setattr(bd, "tree_attention", lambda q, *a, **kw: (asked.append(tuple(q.shape[:2])), attend(q, *a, **kw))[1])
    monkeypatch.setattr(PagePool, "fork", lambda self, *a, **kw: (lengths.append(self.lengths.tolist()), fork(self, *a, **kw))[1])
    r = bd.run(batch=2, beams=3, layers=2, prompt=37, steps=4, window=20)
    assert asked == [(2, 37)] * 2 + [(6, 1)] * 6
    assert lengths[1] == [37, 0, 0, 37, 0, 0] and r["pool"].lengths.tolist() == [40] * 6


@pytest.mark.parametrize("vocab,alive", [(1, 1), (2, 3)])
def test_example_with_fewer_candidates_than_beams(monkeypatch, vocab, alive):
    from examples import beam_decode as bd

    monkeypatch.setattr(bd, "SMOLLM2_135M", dict(bd.SMOLLM2_135M, vocab=vocab))
    r = bd.run(batch=2, beams=3, layers=2, prompt=9, steps=4, window=5)
    t, s = r["tokens"], r["scores"]
    assert bool((t[:, :alive] >= 0).all()) and bool((t[:, alive:] == -1).all())
    assert bool(torch.isfinite(s[:, :alive]).all()) and bool((s[:, alive:] == -float("inf")).all())
    assert r["pool"].lengths.tolist() == [12 if i % 3 < alive else 0 for i in range(6)]
