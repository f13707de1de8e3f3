"""Decoding with drafted trees over a paged, evicted KV cache.

A stack of attention layers (random weights; by default SmolLM2-135M's shape: 9
query and 3 key heads of 64) reads a prompt in chunks, then takes one drafted
tree of tokens a step: per-head norms and rotation (qk_norm_rope), attention of
the whole tree over the PagedKVCache's pages in place (tree_attention), the
accepted path's keys and values appended, and, once a layer is over its budget,
its least attended positions evicted (PagedKVCache.evict).

    python examples/draft_decode.py [--layers 4] [--prompt 700] [--steps 20] [--budget 512]
"""

from __future__ import annotations

import argparse
import sys
import tempfile
import time
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1]))

from voom_b200.runtime.kv_attention import DraftTree, KVView, tree_attention  # noqa: E402
from voom_b200.runtime.kv_paged import PagedKVCache  # noqa: E402
from voom_b200.runtime.rotary import Rotary, qk_norm_rope  # noqa: E402
from voom_b200.synthetic import SMOLLM2_135M  # noqa: E402


class AttentionStack:
    """Pre-norm attention layers with residuals, one request."""

    def __init__(self, layers: int, hidden: int, heads: int, kv_heads: int, head_dim: int, device, seed: int = 0):
        g = torch.Generator(device=device).manual_seed(seed)

        def w(*shape, std):
            return (torch.randn(shape, device=device, generator=g) * std).to(torch.bfloat16)

        self.hq, self.hk, self.D, self.hidden, self.device = heads, kv_heads, head_dim, hidden, torch.device(device)
        self.qkv = [w((heads + 2 * kv_heads) * head_dim, hidden, std=hidden ** -0.5) for _ in range(layers)]
        self.out = [w(hidden, heads * head_dim, std=(heads * head_dim) ** -0.5) for _ in range(layers)]
        self.q_norm = [1 + w(head_dim, std=0.1) for _ in range(layers)]
        self.k_norm = [1 + w(head_dim, std=0.1) for _ in range(layers)]
        self.rotary = Rotary(head_dim, device=device)
        e = torch.zeros((1, kv_heads, 1, head_dim), dtype=torch.bfloat16, device=device)
        self.empty = KVView.contiguous(e, e, torch.zeros(1, dtype=torch.int32, device=device), max_len=0)

    def __len__(self) -> int:
        return len(self.qkv)

    def step(self, x: torch.Tensor, tree: DraftTree, kv: PagedKVCache, sums: list[torch.Tensor]):
        """x: (n, hidden) embeddings of the step's tokens.  Returns their hidden
        states and each layer's new keys and values (not yet in the cache)."""
        n = x.shape[0]
        pos = (kv.offset + tree.depth[0]).contiguous()  # `offset` counts evicted positions too
        new = []
        for i in range(len(self)):
            h = torch.nn.functional.rms_norm(x, (self.hidden,))
            qkv = (h @ self.qkv[i].T).view(n, self.hq + 2 * self.hk, self.D)
            q, k, v = qkv.split((self.hq, self.hk, self.hk), dim=1)
            qk_norm_rope(q, k, pos, self.rotary, q_weight=self.q_norm[i], k_weight=self.k_norm[i], out_q=q, out_k=k)
            view = kv.view(i) if kv.length(i) else self.empty
            o = tree_attention(q[None], k[None], v[None], tree, view, weights=sums[i][None])
            x = x + o.view(n, -1) @ self.out[i].T
            new.append((k, v))
        return x, new

    def commit(self, new, path: torch.Tensor, kv: PagedKVCache, sums: list[torch.Tensor]) -> None:
        """Appends the accepted tokens (indexes of the tree, root first) to every
        layer; their weight sums move right behind the cached positions'."""
        for i, (k, v) in enumerate(new):
            n = kv.length(i)
            sums[i][:, n:n + path.numel()] = sums[i][:, n + path]
            sums[i][:, n + path.numel():] = 0
            kv.append(i, k[path].transpose(0, 1)[None].contiguous(), v[path].transpose(0, 1)[None].contiguous())


def evict_over(kv: PagedKVCache, sums: list[torch.Tensor], budget: int, sinks: int = 4) -> None:
    for i, s in enumerate(sums):
        if kv.length(i) > budget:
            e = kv.evict(i, s[None], budget=budget, sinks=sinks, recent=budget // 4)
            s.zero_()
            s[:, :budget] = e.weights[0]


def run(layers: int = 4, prompt: int = 700, steps: int = 20, budget: int = 512, drafts: int = 12, seed: int = 0,
        page_positions: int = 64) -> dict:
    c = SMOLLM2_135M
    dev = torch.device("cuda", torch.cuda.current_device())
    stack = AttentionStack(layers, c["hidden"], c["heads"], c["kv_heads"], c["head_dim"], dev, seed)
    g = torch.Generator(device=dev).manual_seed(seed + 1)
    host = torch.Generator().manual_seed(seed + 2)
    with tempfile.TemporaryDirectory() as spill:
        kv = PagedKVCache(layers, max_bytes=1 << 40, spill_dir=spill, page_positions=page_positions)
        sums = [torch.zeros((stack.hk, prompt + budget + 2 * page_positions + 512), device=dev) for _ in range(layers)]

        def tokens(n):
            return torch.randn((n, stack.hidden), device=dev, generator=g).to(torch.bfloat16)

        for at in range(0, prompt, 256):  # the prompt, in chunks
            n = min(256, prompt - at)
            x, new = stack.step(tokens(n), DraftTree.chain(1, n, dev), kv, sums)
            stack.commit(new, torch.arange(n, device=dev), kv, sums)
        t0 = time.perf_counter()
        accepted = 0
        for _ in range(steps):
            evict_over(kv, sums, budget)
            # a drafted tree; the verifier (here: chance) accepts one path from its root
            parents = [-1] + [int(torch.randint(max(0, i - 4), i, (1,), generator=host)) for i in range(1, drafts)]
            tree = DraftTree(torch.tensor([parents], dtype=torch.int32, device=dev))
            x, new = stack.step(tokens(drafts), tree, kv, sums)
            j = int(torch.randint(0, drafts, (1,), generator=host))
            path = []
            while j >= 0:
                path.append(j)
                j = parents[j]
            stack.commit(new, torch.tensor(path[::-1], device=dev), kv, sums)
            accepted += len(path)
        torch.cuda.synchronize()
        stack.empty.check_status()
        kv.check_status()  # no wait inside a kernel ran out in any layer of any step
        return {"accepted": accepted, "steps": steps, "seconds": time.perf_counter() - t0, "offset": kv.offset,
                "lengths": [kv.length(i) for i in range(layers)], "hidden": x, "sums": sums}


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--prompt", type=int, default=700)
    ap.add_argument("--steps", type=int, default=20)
    ap.add_argument("--budget", type=int, default=512)
    r = run(**vars(ap.parse_args()))
    print(f"{r['accepted']} tokens accepted in {r['steps']} steps, {r['seconds'] / r['steps'] * 1e3:.2f} ms a step; "
          f"{r['offset']} positions seen, {r['lengths'][0]} kept in layer 0")


if __name__ == "__main__":
    main()
