"""Decoding with beams over a pool of shared cache pages.

A stack of attention layers (random weights; by default SmolLM2-135M's shape: 9
query and 3 key heads of 64), every other one looking back over a window only, all
with capped scores, reads the prompts of a batch, then takes a token for each beam a
step: the cache's rows follow the beams they continue (PagePool.fork: pages are
shared, an open one is copied where two beams write on), each layer attends over the
pool's pages in place (tree_attention), the new keys and values are appended, and the
step's continuations are chosen over beams and vocabulary (beam_select).

    python examples/beam_decode.py [--batch 2] [--beams 4] [--prompt 300] [--steps 32]
"""

from __future__ import annotations

import argparse
import math
import sys
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from examples.draft_decode import AttentionStack  # noqa: E402
from voom_b200.runtime.beam import beam_select  # noqa: E402
from voom_b200.runtime.kv_attention import DraftTree, KVView, tree_attention  # noqa: E402
from voom_b200.runtime.kv_pool import PagePool, kv_append  # noqa: E402
from voom_b200.runtime.rotary import qk_norm_rope  # noqa: E402
from voom_b200.synthetic import SMOLLM2_135M  # noqa: E402


def step(stack: AttentionStack, pool: PagePool, x: torch.Tensor, *, cap: float, window: int, rows: torch.Tensor | None = None,
         live: torch.Tensor | None = None) -> torch.Tensor:
    """x: (rows, n, hidden), the tokens that follow each row's positions, for which the pool has room; of the pool's
    rows those that `rows` names (None: all), and those of them whose `live` is 1 (int32; None: all).
    Returns their hidden states; keys and values are in the pool."""
    B, n, hidden = x.shape
    tree = DraftTree.chain(B, n, x.device)
    grown = n if live is None else n * live  # a row that has ended stays empty
    if rows is None:
        lengths, views = pool.lengths, [pool.view(i) for i in range(len(stack))]
    else:
        table, lengths = pool.table[rows], pool.lengths[rows]
        views = [KVView.pool(pool.k[i], pool.v[i], table, lengths, max_len=pool.max_len) for i in range(len(stack))]
        grown = torch.zeros_like(pool.lengths).index_put_((rows,), torch.as_tensor(grown, dtype=torch.int32, device=x.device))
    pos = tree.positions(lengths).reshape(-1)
    for i, view in enumerate(views):
        h = torch.nn.functional.rms_norm(x, (hidden,))
        qkv = (h @ stack.qkv[i].T).view(B * n, stack.hq + 2 * stack.hk, stack.D)
        q, k, v = qkv.split((stack.hq, stack.hk, stack.hk), dim=1)
        qk_norm_rope(q, k, pos, stack.rotary, q_weight=stack.q_norm[i], k_weight=stack.k_norm[i], out_q=q, out_k=k)
        q, k, v = (t.unflatten(0, (B, n)) for t in (q, k, v))
        o = tree_attention(q, k, v, tree, view, cap=cap, window=window if i % 2 else None)
        x = x + o.reshape(B, n, -1) @ stack.out[i].T
        kv_append(view, k, v)
    pool.advance(grown)
    return x


def run(batch: int = 2, beams: int = 4, layers: int = 4, prompt: int = 300, steps: int = 32, window: int = 128,
        cap: float = 50.0, seed: int = 0, page: int = 16) -> dict:
    c = SMOLLM2_135M
    dev = torch.device("cuda", torch.cuda.current_device())
    stack = AttentionStack(layers, c["hidden"], c["heads"], c["kv_heads"], c["head_dim"], dev, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    embed = torch.randn((c["vocab"], stack.hidden), device=dev, generator=g).to(torch.bfloat16)
    rows = batch * beams
    per = -(-(prompt + steps) // page)
    # a prompt's pages are held once; what follows, and an open page more while forking, by each beam
    pages = batch * per + rows * (-(-steps // page) + 2)
    pool = PagePool(layers, stack.hk, stack.D, pages=pages, rows=rows, max_len=prompt + steps, page=page, device=dev)
    t0 = time.perf_counter()
    # the prompts go into each request's first row; then all its beams continue that one
    first = torch.arange(rows, device=dev, dtype=torch.int32) // beams * beams
    lead = torch.arange(0, rows, beams, device=dev)
    ids = torch.randint(0, c["vocab"], (batch, prompt), device=dev, generator=g)
    pool.fork(grow=torch.zeros_like(first).index_fill_(0, lead, prompt))
    hidden = step(stack, pool, embed[ids], cap=cap, window=window, rows=lead)[:, -1].repeat_interleave(beams, 0)
    pool.fork(first)
    scores = torch.full((batch, beams), -math.inf, device=dev)
    scores[:, 0] = 0.0
    tokens = torch.empty((rows, 0), dtype=torch.int32, device=dev)
    for i in range(steps):
        logits = (torch.nn.functional.rms_norm(hidden, (stack.hidden,)) @ embed.T) / math.sqrt(stack.hidden)
        best = beam_select(logits.view(batch, beams, -1), scores, beams)
        scores, parents = best.scores, best.parents.flatten()
        live = parents >= 0  # where there are fewer candidates than beams the others end
        tokens = torch.cat((tokens[parents.clamp(min=0).long()], best.tokens.view(rows, 1)), 1).where(live[:, None], -1)
        if i + 1 < steps:
            pool.fork(parents, grow=1)
            hidden = step(stack, pool, embed[tokens[:, -1:].clamp(min=0).long()], cap=cap, window=window,
                          live=live.to(torch.int32))[:, -1]
    torch.cuda.synchronize()
    pool.check_status()  # no page was missing, no wait inside a kernel ran out
    return {"tokens": tokens.view(batch, beams, steps), "scores": scores, "seconds": time.perf_counter() - t0, "prompt": ids,
            "pages": int((pool.refs > 0).sum()), "unshared": sum(-(-n // page) for n in pool.lengths.tolist()), "pool": pool}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    for name, value in (("batch", 2), ("beams", 4), ("layers", 4), ("prompt", 300), ("steps", 32), ("window", 128)):
        ap.add_argument(f"--{name}", type=int, default=value)
    a = vars(ap.parse_args())
    r = run(**a)
    print(f"{a['batch']} requests of {a['beams']} beams, {a['steps']} steps: {r['seconds'] / a['steps'] * 1e3:.2f} ms a step; "
          f"{r['pages']} pages held for {r['unshared']}; best scores {[round(x, 3) for x in r['scores'][:, 0].tolist()]}")


if __name__ == "__main__":
    main()
