"""Attention over a KV cache: drafted trees, prompts and single tokens, the
weight each cached position receives, and eviction by it.

  KVView          - where keys and values lie: one piece, pages of a pool, or
                    pages anywhere (PagedKVCache.view).
  DraftTree       - the new tokens of a step: a tree of drafts per request, or
                    a chain (a prompt's chunk; one token).
  tree_attention  - the new tokens' attention over the cache and one another
                    (csrc/kv_attn.cu).
  kv_evict        - keeps a cache's first, newest and most attended positions
                    (csrc/kv_evict.cu).

New tokens' keys and values are separate tensors, as they come from the
projection: a drafted token enters a cache only once it is accepted, so a
rejected one leaves nothing to undo.  Only check_status synchronises with the
host.  A view's own tensors belong to the stream that was current when it was
made: calls on another stream need it kept until they have run.

Counterpart in the reference: the attention around its caches
(runtime/layer_runner.py `_attention`, runtime/kv_paged.py:143-181).
"""

from __future__ import annotations

import ctypes
import struct
import threading
from typing import NamedTuple

import numpy as np
import torch

from .. import _device
from .._lib import VOOM_E_CAPACITY, VOOM_E_OVERLAP, ELEMENT_TYPES, KvEvictArgs, KvViewStruct, TreeAttentionArgs, check, load

MAX_HEAD_DIM = 256
MAX_TREE = 1024  # tokens of a tree that is not a chain
NO_PAGE = -2 ** 63  # VOOM_NO_PAGE
_NO_SCRATCH = (None, 0)
_CACHE_TYPES = (torch.bfloat16, torch.float16)


def _rows(x: torch.Tensor, name: str) -> None:
    """Checks what the kernels need of a tensor whose last dimension is a head's values."""
    if x.stride(-1) != 1 or x.data_ptr() % 16 or any(s % 8 for s in x.stride()[:-1]):
        raise ValueError(f"{name}: heads must be contiguous and every row must start on 16 bytes")


def _steps(x: torch.Tensor) -> tuple:
    """Strides of a (.., heads, positions, D) page; 0 where there is one of a kind and any stride will do."""
    return tuple(s if n > 1 else 0 for s, n in zip(x.stride()[-3:], x.shape[-3:]))


def check_wait_status(status: torch.Tensor) -> None:
    """Raises RuntimeError if an attention kernel has set the status word; clears it.  Synchronises."""
    if int(status.item()):
        status.zero_()
        raise RuntimeError("tree_attention: a wait inside the kernel ran out")


class KVView:
    """Keys and values of B requests as the attention reads them; holds the
    tensors.  `lengths` is an int32 device tensor of the B requests' cached
    positions, read by the kernels when they run (it may change between
    calls, and a captured graph sees the change); `max_len` bounds them."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, *, batch: int, heads: int,
                 head_dim: int, page: int, strides: tuple, max_len: int, table: torch.Tensor | None = None,
                 offsets: torch.Tensor | None = None, table_stride: int = 0, n_pages: int = 0, keep: object = None,
                 status: torch.Tensor | None = None):
        if k.dtype not in _CACHE_TYPES or v.dtype != k.dtype:
            raise ValueError(f"cached keys and values must both be BF16 or FP16, got {k.dtype} and {v.dtype}")
        if head_dim % 8 or not 0 < head_dim <= MAX_HEAD_DIM:
            raise ValueError(f"head size {head_dim}: a multiple of 8 up to {MAX_HEAD_DIM}")
        self.device = _device.require_cuda(k.device)
        if lengths.dtype != torch.int32 or lengths.shape != (batch,) or not lengths.is_contiguous():
            raise ValueError(f"lengths: {batch} contiguous int32 wanted, got {tuple(lengths.shape)} {lengths.dtype}")
        if not (v.device == lengths.device == self.device):
            raise ValueError("keys, values and lengths must be on one device")
        capacity = page * table_stride if (table is not None or offsets is not None) else page
        if not 0 <= max_len <= capacity:
            raise ValueError(f"max_len {max_len} of a cache that holds {capacity} positions")
        self.k, self.v, self.lengths, self.table, self.offsets, self.keep = k, v, lengths, table, offsets, keep
        self.batch, self.heads, self.head_dim, self.max_len = batch, heads, head_dim, max_len
        self.dtype = k.dtype
        self.struct = KvViewStruct(k.data_ptr(), v.data_ptr(), lengths.data_ptr(),
                                   None if table is None else table.data_ptr(),
                                   None if offsets is None else offsets.data_ptr(), *strides, batch, heads, head_dim,
                                   ELEMENT_TYPES[k.dtype], page, table_stride, n_pages, max_len)
        self.packed = bytes(self.struct)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device) if status is None else status
        self.status_ptr = self.status.data_ptr()
        self.scale = head_dim ** -0.5
        self.index = self.device.index
        self._scratch: dict[int, torch.Tensor] = {}
        self.scratch: dict[int, tuple[int, int]] = {}  # stream -> address, bytes
        self.lock = threading.Lock()  # a call's launches share the stream's workspace: they stay together

    @classmethod
    def contiguous(cls, k: torch.Tensor, v: torch.Tensor, lengths: torch.Tensor, max_len: int | None = None) -> "KVView":
        """k, v: (B, heads, capacity, D), any strides that keep rows on 16 bytes."""
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"k and v: (B, heads, capacity, D) wanted, got {tuple(k.shape)} and {tuple(v.shape)}")
        _rows(k, "k")
        _rows(v, "v")
        B, H, cap, D = k.shape
        return cls(k, v, lengths, batch=B, heads=H, head_dim=D, page=cap, max_len=cap if max_len is None else max_len,
                   strides=(*k.stride()[:3], *v.stride()[:3]))

    @classmethod
    def pool(cls, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
             max_len: int | None = None) -> "KVView":
        """k, v: (pages, heads, positions, D); table: (B, pages per request)
        int32, the pool page of each run of positions.  A table entry outside
        the pool reads as zero keys and values."""
        if k.dim() != 4 or v.shape != k.shape:
            raise ValueError(f"k and v: (pages, heads, positions, D) wanted, got {tuple(k.shape)} and {tuple(v.shape)}")
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() or table.device != k.device:
            raise ValueError("table: a contiguous int32 (B, pages) tensor on the pool's device wanted")
        _rows(k, "k")
        _rows(v, "v")
        N, H, P, D = k.shape
        B, per = table.shape
        return cls(k, v, lengths, batch=B, heads=H, head_dim=D, page=P, table=table, table_stride=per, n_pages=N,
                   max_len=P * per if max_len is None else max_len, strides=(*k.stride()[:3], *v.stride()[:3]))

    @classmethod
    def pages(cls, pages: list[list[tuple[torch.Tensor, torch.Tensor]]], lengths: torch.Tensor,
              max_len: int | None = None, status: torch.Tensor | None = None) -> "KVView":
        """One list of (k, v) pages per request, each (1, heads, positions, D)
        or (heads, positions, D) with the same strides, anywhere on the device.
        Positions past a request's own pages read as zero keys and values.
        `status`: an int32 word on the device that several views share."""
        flat = [p for request in pages for p in request]
        if not flat:
            raise ValueError("a view of pages needs at least one page")
        k0, v0 = flat[0]
        kw, vw, ks, vs = k0.stride(), v0.stride(), _steps(k0), _steps(v0)
        for k, v in flat:
            if k.shape != k0.shape or v.shape != k0.shape or (k.stride() != kw and _steps(k) != ks) or \
                    (v.stride() != vw and _steps(v) != vs):
                raise ValueError("all pages must have one shape and one set of strides")
            if k.dtype != k0.dtype or v.dtype != k0.dtype or k.device != k0.device or v.device != k0.device:
                raise ValueError("all pages must have one type and lie on one device")
            _rows(k, "k page")
            _rows(v, "v page")
        if k0.dim() not in (3, 4) or (k0.dim() == 4 and k0.shape[0] != 1):
            raise ValueError(f"pages of (1, heads, positions, D) wanted, got {tuple(k0.shape)}")
        H, P, D = k0.shape[-3:]
        per = max(len(request) for request in pages)
        e = k0.element_size()
        off = np.full((len(pages), per, 2), NO_PAGE, np.int64)
        for b, request in enumerate(pages):
            for p, (k, v) in enumerate(request):
                off[b, p] = (k.data_ptr() - k0.data_ptr()) // e, (v.data_ptr() - v0.data_ptr()) // e
        # from pinned memory: a copy from pageable memory waits for all that the stream has to do
        offsets = torch.from_numpy(off).pin_memory().to(k0.device, non_blocking=True)
        return cls(k0, v0, lengths, batch=len(pages), heads=H, head_dim=D, page=P, offsets=offsets, table_stride=per,
                   max_len=P * per if max_len is None else max_len, strides=(0, ks[0], ks[1], 0, vs[0], vs[1]),
                   keep=flat, status=status)

    def check_status(self) -> None:
        """Raises RuntimeError if a wait inside an attention kernel ran out since
        the last check (its outputs are then not valid); clears the status.
        Synchronises; calls never do, so callers check where they read results."""
        check_wait_status(self.status)

    def more_scratch(self, n: int, stream_ptr: int) -> tuple[int, int]:
        """(address, bytes) of a workspace of at least n bytes for the calls on
        one stream, kept with the view until a call needs more.  Calls that are
        captured do not use it: a graph keeps the address that it was given."""
        t = torch.empty(n, dtype=torch.uint8, device=self.device)
        self._scratch[stream_ptr] = t
        s = self.scratch[stream_ptr] = (t.data_ptr(), n)
        return s


class DraftTree:
    """The new tokens of one step.  `parents` (B, n) int32: the parent of each
    drafted token (a lower index), -1 for a root, which follows the last cached
    position, -2 for no token (requests with fewer drafts than n).  A token sees
    the whole cache, its ancestors and itself.  The masks and depths are made
    on the device once and serve every layer of the step."""

    def __init__(self, parents: torch.Tensor, stream: torch.cuda.Stream | None = None):
        if parents.dim() != 2 or parents.dtype != torch.int32:
            raise ValueError(f"parents: an int32 (B, n) tensor wanted, got {tuple(parents.shape)} {parents.dtype}")
        if parents.shape[1] > MAX_TREE:
            raise ValueError(f"a tree of {parents.shape[1]} tokens: at most {MAX_TREE}")
        self.device = _device.require_cuda(parents.device)
        self.index = self.device.index
        self.batch, self.n = parents.shape
        with _device.on_stream(self.device, stream) as sp:
            parents = parents.contiguous()
            self.mask: torch.Tensor | None = torch.empty((self.batch, self.n, (self.n + 31) // 32), dtype=torch.int32,
                                                         device=self.device)
            self.depth = torch.empty((self.batch, self.n), dtype=torch.int32, device=self.device)
            if parents.numel():
                check(load().voom_tree_mask(parents.data_ptr(), self.batch, self.n, self.mask.data_ptr(),
                                            self.depth.data_ptr(), sp), "voom_tree_mask")
        self.mask_ptr = self.mask.data_ptr() if parents.numel() else 0

    @classmethod
    def chain(cls, batch: int, n: int, device=None) -> "DraftTree":
        """n tokens that follow one another in every request: one new token, a
        prompt or a chunk of one.  Any length; needs no mask."""
        t = cls.__new__(cls)
        t.device = _device.require_cuda(device)
        t.index, t.mask_ptr = t.device.index, 0
        t.batch, t.n, t.mask = int(batch), int(n), None
        t.depth = torch.arange(n, dtype=torch.int32, device=t.device).expand(batch, n)
        return t

    def positions(self, lengths: torch.Tensor) -> torch.Tensor:
        """Cached positions + depth of every new token, (B, n) int32: its rotary
        position only where nothing was evicted.  After an eviction add the depth
        to the count of all positions seen (PagedKVCache.offset)."""
        return lengths[:, None] + self.depth


# voom_tree_attention_args and voom_kv_evict_args as bytes: cheaper to make than
# ctypes structures, and one-token calls are bound by the host
_ATTN = struct.Struct("9Q14q2If4x")
_EVICT = struct.Struct("Q2q5Q4I")
assert _ATTN.size == ctypes.sizeof(TreeAttentionArgs) and _EVICT.size == ctypes.sizeof(KvEvictArgs)


def _new(x: torch.Tensor, name: str, B: int, n: int, heads: int, cache: KVView) -> tuple:
    """Checks a (B, n, heads, D) tensor of new tokens; its first three strides."""
    s = x.stride()
    if x.shape != (B, n, heads, cache.head_dim) or x.dtype != cache.dtype or x.get_device() != cache.index:
        raise ValueError(f"{name}: ({B}, {n}, {heads}, {cache.head_dim}) {cache.dtype} on {cache.device} wanted, got "
                         f"{tuple(x.shape)} {x.dtype} on {x.device}")
    if s[3] != 1 or (s[0] | s[1] | s[2]) & 7 or x.data_ptr() & 15:
        raise ValueError(f"{name}: heads must be contiguous and every row must start on 16 bytes")
    return s


def _sums(weights: torch.Tensor, cache: KVView, positions: int) -> tuple:
    """Checks the positions' weight sums; their strides."""
    s = weights.stride()
    if weights.dim() != 3 or weights.shape[:2] != (cache.batch, cache.heads) or weights.shape[2] < positions or \
            weights.dtype != torch.float32 or s[2] != 1 or weights.get_device() != cache.index:
        raise ValueError(f"weights: fp32 ({cache.batch}, {cache.heads}, at least {positions}) on {cache.device} wanted, "
                         f"got {tuple(weights.shape)} {weights.dtype}")
    return s


def tree_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, tree: DraftTree, cache: KVView, *,
                   scale: float | None = None, weights: torch.Tensor | None = None,
                   token_weight: torch.Tensor | None = None, out: torch.Tensor | None = None,
                   return_lse: bool = False, stream: torch.cuda.Stream | None = None):
    """Attention of the new tokens (q: (B, n, Hq, D); k, v: (B, n, heads, D),
    any strides with 16-byte rows) over the cache and over one another, as
    `tree` says: (B, n, Hq, D) in the cache's type, and with `return_lse` the
    natural log of each row's softmax denominator, (B, n, Hq) fp32.  Query head
    h reads key head h // (Hq // heads); `scale` defaults to D ** -0.5.  A row
    of no token gives zeros and lse -inf.  `out` must not share memory with q, k
    or v, nor rows of `out` or `weights` with one another.

    `weights` (B, heads, >= max_len + n) fp32: each position's softmax weight,
    summed over the rows that share its head (each times `token_weight` (B, n)
    fp32, if given), is added in place: cached positions at their index, new
    token j at lengths[b] + j.  kv_evict reads these sums.  Up to 16 rows (tokens
    x query heads) per key head, the workspace holds their scores: 4 bytes a row
    and position, for max_len positions of every request."""
    if stream is not None or _device.current_index() != cache.index:
        with _device.on_stream(cache.device, stream):
            return tree_attention(q, k, v, tree, cache, scale=scale, weights=weights, token_weight=token_weight,
                                  out=out, return_lse=return_lse)
    if q.dim() != 4:
        raise ValueError(f"q: (B, n, Hq, D) wanted, got {tuple(q.shape)}")
    B, n, hq, D = q.shape
    heads = cache.heads
    if B != cache.batch or B != tree.batch or n != tree.n:
        raise ValueError(f"{B} requests of {n} new tokens in q, {tree.batch} of {tree.n} in the tree, {cache.batch} cached")
    if hq % heads or not hq:
        raise ValueError(f"{hq} query heads do not divide into {heads} key heads")
    if scale is not None and not 0.0 < scale < 3e38:
        raise ValueError(f"scale {scale}: a positive number wanted")
    qs = _new(q, "q", B, n, hq, cache)
    ks = _new(k, "k", B, n, heads, cache)
    vs = _new(v, "v", B, n, heads, cache)
    if tree.index != cache.index:
        raise ValueError(f"the tree is on {tree.device}, the cache on {cache.device}")
    wp = wb = wh = tw = 0
    if weights is not None:
        wb, wh, _ = _sums(weights, cache, cache.max_len + n)
        wp = weights.data_ptr()
    if token_weight is not None:
        if weights is None:
            raise ValueError("token_weight goes with weights")
        if token_weight.shape != (B, n) or token_weight.dtype != torch.float32 or not token_weight.is_contiguous() \
                or token_weight.get_device() != cache.index:
            raise ValueError(f"token_weight: contiguous fp32 ({B}, {n}) on {cache.device} wanted")
        tw = token_weight.data_ptr()
    if out is None:
        out = q.new_empty((B, n, hq, D))
    os = _new(out, "out", B, n, hq, cache)
    lse = q.new_empty((B, n, hq), dtype=torch.float32) if return_lse else None
    if n:
        a = _ATTN.pack(q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 0 if lse is None else lse.data_ptr(),
                       tree.mask_ptr, wp, tw, cache.status_ptr, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], vs[0], vs[1], vs[2], os[0],
                       os[1], os[2], wb, wh, n, hq, cache.scale if scale is None else scale)
        lib, sp = load(), _device.raw_stream(cache.index)
        if _device.capturing():
            # a workspace from the graph's own pool, which no tensor outside the graph gets for as long as it lives
            ws = q.new_empty(lib.voom_tree_attention_scratch_bytes(cache.packed, a), dtype=torch.uint8)
            rc = lib.voom_tree_attention(cache.packed, a, ws.data_ptr(), ws.numel(), sp)
        else:
            with cache.lock:
                ws = cache.scratch.get(sp, _NO_SCRATCH)
                rc = lib.voom_tree_attention(cache.packed, a, ws[0], ws[1], sp)
                if rc == VOOM_E_CAPACITY:  # refused before anything was launched
                    ws = cache.more_scratch(lib.voom_tree_attention_scratch_bytes(cache.packed, a), sp)
                    rc = lib.voom_tree_attention(cache.packed, a, ws[0], ws[1], sp)
        if rc == VOOM_E_OVERLAP:
            raise ValueError("rows of out or of weights overlap one another, or out shares memory with q, k or v")
        check(rc, "voom_tree_attention")
    return (out, lse) if return_lse else out


class Evicted(NamedTuple):
    """What kv_evict kept: k, v (B, heads, budget, D), the weights (B, heads,
    budget) and original positions (int32, -1 past the length) of the kept
    rows, in order, and the requests' new lengths (B) int32."""

    k: torch.Tensor
    v: torch.Tensor
    weights: torch.Tensor
    index: torch.Tensor
    lengths: torch.Tensor


def kv_evict(cache: KVView, weights: torch.Tensor, *, budget: int, sinks: int = 4, recent: int = 0,
             stream: torch.cuda.Stream | None = None) -> Evicted:
    """Cuts every request to at most `budget` positions: the first `sinks`, the
    newest `recent`, and of the others those with the largest `weights` (B,
    heads, >= max_len) fp32 (equal ones: the lower position), each head by
    itself.  Rows past a request's new length are zero."""
    if stream is not None or _device.current_index() != cache.index:
        with _device.on_stream(cache.device, stream):
            return kv_evict(cache, weights, budget=budget, sinks=sinks, recent=recent)
    B, H, D = cache.batch, cache.heads, cache.head_dim
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError(f"a budget of {budget} positions cannot hold {sinks} first and {recent} newest ones")
    wb, wh, _ = _sums(weights, cache, cache.max_len)
    k, v = cache.k.new_empty((2, B, H, budget, D)).unbind(0)
    w, index = weights.new_empty((2, B, H, budget)).unbind(0)
    index = index.view(torch.int32)
    lengths = cache.lengths.new_empty(B)
    a = _EVICT.pack(weights.data_ptr(), wb, wh, k.data_ptr(), v.data_ptr(), w.data_ptr(), index.data_ptr(),
                    lengths.data_ptr(), budget, sinks, recent, 0)
    check(load().voom_kv_evict(cache.packed, a, _device.raw_stream(cache.index)), "voom_kv_evict")
    return Evicted(k, v, w, index, lengths)
