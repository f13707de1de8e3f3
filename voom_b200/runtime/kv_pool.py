"""A pool of cache pages that rows share: written to, forked, compacted.

  kv_append      - new tokens' keys and values to their places in a cache.
  fork_pages     - rows of a page table become continuations of others; pages
                   are shared, open ones copied, fresh ones handed out, those of
                   ended rows free again.
  compact_pages  - the pages in use to the front of the pool.
  PagePool       - a pool with its table and lengths, over all layers, that does
                   these in place (csrc/kv_pool.cu).

A row's pages are the first ceil(length / page) entries of its table row, and
what the rows hold is all that is kept: nothing counts up and down beside the
table.  Lengths, tables and parents are read on the device; only
PagePool.check_status and PagePool.resize synchronise with the host.

Counterpart in the reference: the concatenating caches of runtime/kv_paged.py:143-181
and the paged pool of runtime/kv_cache.py:255-810 (outside its ported path).
"""

from __future__ import annotations

import ctypes
import functools
import struct
import threading
from typing import NamedTuple

import torch

from .. import _device
from .._lib import VOOM_E_OVERLAP, KvAppendArgs, KvCompactArgs, KvForkArgs, check, load
from .kv_attention import _CACHE_TYPES, MAX_HEAD_DIM, KVView, _new

MAX_PAGE = 32768
MAX_ROWS = 65535

_APPEND = struct.Struct("3Q6q2I")
_FORK = struct.Struct("10Q8q10I")
_COMPACT = struct.Struct("6Q8q8I")
assert _APPEND.size == ctypes.sizeof(KvAppendArgs) and _FORK.size == ctypes.sizeof(KvForkArgs) and \
    _COMPACT.size == ctypes.sizeof(KvCompactArgs)


def kv_append(cache: KVView, k: torch.Tensor, v: torch.Tensor, *, index: torch.Tensor | None = None,
              stream: torch.cuda.Stream | None = None) -> None:
    """Writes new tokens' k and v (B, n, heads, D) into the cache behind each
    request's positions: lengths[b] + j gets token j or, with `index` (B, m)
    int32, token index[b, j] (an accepted path of a drafted tree; an entry
    outside [0, n) writes nothing), whatever the view's max_len.  Positions that
    the cache has no page for are not written.  The lengths stay: every layer is written before they grow.
    Rows that share the page they would write to must be forked first
    (fork_pages makes it theirs).  A PagedKVCache's view holds copies and is
    refused: its own append() stores positions."""
    if not cache.writable:
        raise ValueError("this view holds copies of its cache's positions: what is written there would be lost; use the cache's append()")
    if stream is not None or _device.current_index() != cache.index:
        with _device.on_stream(cache.device, stream):
            return kv_append(cache, k, v, index=index)
    if k.dim() != 4 or k.shape[0] != cache.batch:
        raise ValueError(f"k: ({cache.batch}, n, {cache.heads}, {cache.head_dim}) wanted, got {tuple(k.shape)}")
    B, n = k.shape[:2]
    ks, vs = _new(k, "k", B, n, cache.heads, cache), _new(v, "v", B, n, cache.heads, cache)
    m, at = n, 0
    if index is not None:
        if index.dim() != 2 or index.shape[0] != B or index.dtype != torch.int32 or not index.is_contiguous() or \
                index.get_device() != cache.index:
            raise ValueError(f"index: contiguous int32 ({B}, m) on {cache.device} wanted, got {tuple(index.shape)} {index.dtype}")
        m, at = index.shape[1], index.data_ptr()
    if not n or not m:
        return
    a = _APPEND.pack(k.data_ptr(), v.data_ptr(), at, *ks[:3], *vs[:3], n, m)
    rc = load().voom_kv_append(cache.packed, a, _device.raw_stream(cache.index))
    if rc == VOOM_E_OVERLAP:
        raise ValueError("positions of the cache overlap one another, or share memory with k or v")
    check(rc, "voom_kv_append")


def _pool(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor) -> tuple:
    """Checks a pool, its table and lengths; device index, sizes, strides."""
    size, kind, index = k.shape, k.dtype, k.get_device()
    if len(size) != 5 or v.shape != size or kind not in _CACHE_TYPES or v.dtype is not kind:
        raise ValueError(f"k and v: (layers, pages, heads, positions, D) BF16 or FP16 wanted, got {tuple(k.shape)} {k.dtype} and "
                         f"{tuple(v.shape)} {v.dtype}")
    L, N, H, P, D = size
    if not (L and N and H and P and D) or D % 8 or D > MAX_HEAD_DIM or P > MAX_PAGE:
        raise ValueError(f"{tuple(size)}: no dimension may be empty, D a multiple of 8 up to {MAX_HEAD_DIM}, pages of at most "
                         f"{MAX_PAGE} positions")
    ks, vs = k.stride(), v.stride()
    if ks[4] != 1 or vs[4] != 1 or (ks[0] | ks[1] | ks[2] | ks[3] | vs[0] | vs[1] | vs[2] | vs[3]) & 7 or \
            (k.data_ptr() | v.data_ptr()) & 15:
        raise ValueError("k and v: the values of a position must be adjacent and every row must start on 16 bytes")
    if table.dim() != 2 or table.dtype is not torch.int32 or not table.is_contiguous() or not table.numel():
        raise ValueError(f"table: a contiguous int32 (rows, pages) tensor wanted, one of each at least, got {tuple(table.shape)} "
                         f"{table.dtype}")
    R, per = table.shape
    if R > MAX_ROWS or per * P >= 2 ** 31 or R * per >= 2 ** 31:
        raise ValueError(f"{R} rows of {per} pages of {P} positions: at most {MAX_ROWS} rows, fewer than 2^31 positions and entries")
    _row_numbers(lengths, "lengths", R)
    if index < 0 or not index == v.get_device() == table.get_device() == lengths.get_device():
        raise ValueError("keys, values, table and lengths must be on one CUDA device")
    return index, L, N, H, P, D, R, per, (*ks[:4], *vs[:4])


def _row_numbers(x: torch.Tensor, name: str, rows: int) -> None:
    if x.shape != (rows,) or x.dtype != torch.int32 or not x.is_contiguous():
        raise ValueError(f"{name}: {rows} contiguous int32 wanted, got {tuple(x.shape)} {x.dtype}")


def _refused(rc: int, what: str) -> None:
    if rc == VOOM_E_OVERLAP:
        raise ValueError("positions of the pool overlap one another, or keys share memory with values")
    check(rc, what)


@functools.lru_cache(maxsize=256)
def _fork_words(rows: int, per: int, pages: int, in_place: bool) -> int:
    return load().voom_kv_fork_scratch_bytes(rows, per, pages, in_place) // 4


@functools.lru_cache(maxsize=256)
def _compact_words(pages: int) -> int:
    return load().voom_kv_compact_scratch_bytes(pages) // 4


def _changes(parents: torch.Tensor | None, grow: int | torch.Tensor, rows: int, index: int) -> tuple[int, int, int]:
    """Checks parents and grow: their addresses (0: none), and the one number that all rows grow by."""
    at = each = 0
    if parents is not None:
        _row_numbers(parents, "parents", rows)
        if parents.get_device() != index:
            raise ValueError("parents must be on the pool's device")
        at = parents.data_ptr()
    if isinstance(grow, torch.Tensor):
        _row_numbers(grow, "grow", rows)
        if grow.get_device() != index:
            raise ValueError("grow must be on the pool's device")
        return at, grow.data_ptr(), 0
    if not 0 <= grow < 2 ** 31:
        raise ValueError(f"grow {grow}: not a number of positions")
    return at, each, int(grow)


class Forked(NamedTuple):
    """The new table (rows, pages) and lengths (rows), how many rows hold each
    page (pages of the pool), and the count (1) of pages that were wanted and not
    to be had; int32."""

    table: torch.Tensor
    lengths: torch.Tensor
    refs: torch.Tensor
    missing: torch.Tensor


def fork_pages(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor,
               parents: torch.Tensor | None = None, *, grow: int | torch.Tensor = 0, out: Forked | None = None,
               stream: torch.cuda.Stream | None = None) -> Forked:
    """Row r of the page table becomes a continuation of row parents[r] (int32;
    None: of itself; outside [0, rows): it ends, and is empty), with room for
    `grow` more positions (one number, or int32 for each row; none for a row
    that ended).  k, v: the pool's pages in all layers, (layers, pages, heads,
    positions, D).  Pages are shared; where the row grows, an open page that it may
    not write on in is replaced by a fresh copy of its filled positions: of the
    rows that hold a page, the longest may (equal ones: the first), unless one
    holds it full.  Fresh pages are the lowest that no row holds any more, in
    the order of the rows; where there are none left, entries are -1 and `missing`
    says how many.  An open page that found no copy is not lost: its entry is page
    - 2^31, which reads as zeros and takes nothing, until a later fork has a page.

    `out`: where the results go.  Its table and lengths may be `table` and
    `lengths` themselves (both); `missing` is then added to."""
    index, L, N, H, P, D, R, per, strides = _pool(k, v, table, lengths)
    if stream is not None or _device.current_index() != index:
        with _device.on_stream(k.device, stream):
            return fork_pages(k, v, table, lengths, parents, grow=grow, out=out)
    rows, each, more = _changes(parents, grow, R, index)
    if out is None:
        # the workspace and the results in one piece
        words = _fork_words(R, per, N, False)
        ws, new, lens, refs, missing = table.new_empty(words + R * per + R + N + 1).split_with_sizes((words, R * per, R, N, 1))
        out, same = Forked(new.view(R, per), lens, refs, missing), False
    else:
        same = out.table.data_ptr() == table.data_ptr()
        for x, name, shape in zip(out, Forked._fields, ((R, per), (R,), (N,), (1,))):
            if x.shape != shape or x.dtype != torch.int32 or not x.is_contiguous() or x.get_device() != index:
                raise ValueError(f"out.{name}: contiguous int32 {shape} on the pool's device wanted, got {tuple(x.shape)} {x.dtype}")
        _apart(out, [table, lengths] + [x for x in (parents, grow) if isinstance(x, torch.Tensor)], same)
        words = _fork_words(R, per, N, same)
        ws = table.new_empty(words)
    a = _FORK.pack(k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr(), rows, each, out.table.data_ptr(),
                   out.lengths.data_ptr(), out.refs.data_ptr(), out.missing.data_ptr(), *strides, L, N, H, P, D, R, per, more,
                   same, 0)
    _refused(load().voom_kv_fork(a, ws.data_ptr(), 4 * words, _device.raw_stream(index)), "voom_kv_fork")
    return out


def _apart(out: tuple, given: list, in_place: bool) -> None:
    """Refuses results that share memory with one another or with what is read,
    but for a table and lengths that are changed in place."""
    def span(x):
        return x.data_ptr(), x.data_ptr() + 4 * x.numel()

    def meet(x, y):
        (a, b), (c, d) = span(x), span(y)
        return a < d and c < b

    for i, x in enumerate(out):
        for y in out[i + 1:]:
            if meet(x, y):
                raise ValueError("the results share memory with one another")
        for j, y in enumerate(given):
            if meet(x, y) and not (in_place and i == j and span(x) == span(y)):
                raise ValueError("the results share memory with what is read")
        if in_place and i < len(given) and i < 2 and span(x) != span(given[i]):
            raise ValueError("the table and the lengths are changed in place together, or neither")


class Compacted(NamedTuple):
    """The new table (rows, pages) and the number (1) of pages in use; int32."""

    table: torch.Tensor
    live: torch.Tensor


def compact_pages(k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, lengths: torch.Tensor, *, room: bool = False,
                  out: Compacted | None = None, stream: torch.cuda.Stream | None = None) -> Compacted:
    """Moves the pages that the rows hold to the front of the pool, in all layers:
    pages past their number go, in order, to the free ones below it.  `room`: a row
    holds the pages past its length too, which a fork has made ready; else they are
    let go.  `out.table` may be `table` itself."""
    index, L, N, H, P, D, R, per, strides = _pool(k, v, table, lengths)
    if stream is not None or _device.current_index() != index:
        with _device.on_stream(k.device, stream):
            return compact_pages(k, v, table, lengths, room=room, out=out)
    words = _compact_words(N)
    if out is None:
        ws, new, live = table.new_empty(words + R * per + 1).split_with_sizes((words, R * per, 1))
        out = Compacted(new.view(R, per), live)
    else:
        for x, name, shape in zip(out, Compacted._fields, ((R, per), (1,))):
            if x.shape != shape or x.dtype != torch.int32 or not x.is_contiguous() or x.get_device() != index:
                raise ValueError(f"out.{name}: contiguous int32 {shape} on the pool's device wanted, got {tuple(x.shape)} {x.dtype}")
        same = out.table.data_ptr() == table.data_ptr()
        _apart(out[:1], [table], same)
        _apart((out.live, out.table), [lengths] if same else [lengths, table], False)
        ws = table.new_empty(words)
    a = _COMPACT.pack(k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr(), out.table.data_ptr(), out.live.data_ptr(),
                      *strides, L, N, H, P, D, R, per, room)
    _refused(load().voom_kv_compact(a, ws.data_ptr(), 4 * words, _device.raw_stream(index)), "voom_kv_compact")
    return out


class PagePool:
    """Keys and values of `rows` continuations over all layers, in pages that rows
    share; a row holds at most `max_len` positions, rounded up to whole pages.  A
    step: fork(parents, grow=n) makes room, every layer attends over view(layer)
    and append()s its new tokens, advance(n) counts them.  The table and the
    lengths keep their addresses, so a captured step stays valid (but for resize).
    Pages that a row does not hold (rows that never grew, or ended) read as zeros.
    `refs` says how many rows held each page after the last fork, by the page
    numbers of that time: compact and resize change them, the next fork counts anew."""

    def __init__(self, layers: int, heads: int, head_dim: int, *, pages: int, rows: int, max_len: int, page: int = 64,
                 dtype: torch.dtype = torch.bfloat16, device=None):
        dev = _device.require_cuda(device)
        if min(layers, heads, head_dim, pages, rows, max_len, page) < 1:
            raise ValueError("a pool of at least one layer, head, value, page, row and position wanted")
        per = -(-max_len // page)
        self.page, self.rows, self.max_len = int(page), int(rows), int(per * page)
        self.k, self.v = (torch.empty((layers, pages, heads, page, head_dim), dtype=dtype, device=dev) for _ in range(2))
        self.table = torch.full((rows, per), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(rows, dtype=torch.int32, device=dev)
        self.missing = torch.zeros(1, dtype=torch.int32, device=dev)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=dev)
        self._wait_status = torch.zeros(1, dtype=torch.int32, device=dev)
        self._lock = threading.Lock()
        self._views: list[KVView] = []
        self._make_views()

    def _make_views(self) -> None:
        self._views = [KVView.pool(k, v, self.table, self.lengths, max_len=self.max_len, status=self._wait_status)
                       for k, v in zip(self.k.unbind(0), self.v.unbind(0))]
        # fork's arguments but for those that change from call to call
        self._index, *sizes, strides = _pool(self.k, self.v, self.table, self.lengths)
        at = [x.data_ptr() for x in (self.k, self.v, self.table, self.lengths, self.table, self.lengths, self.refs, self.missing)]
        self._fork_to = (*at, *strides, *sizes)

    @property
    def pages(self) -> int:
        return self.k.shape[1]

    def view(self, layer: int) -> KVView:
        """The layer's positions for tree_attention and kv_append."""
        return self._views[layer]

    def fork(self, parents: torch.Tensor | None = None, *, grow: int | torch.Tensor = 0,
             stream: torch.cuda.Stream | None = None) -> None:
        """fork_pages of the pool's own table, in place."""
        index = self._index
        if stream is not None or _device.current_index() != index:
            with _device.on_stream(self.k.device, stream):
                return self.fork(parents, grow=grow)
        rows, each, more = _changes(parents, grow, self.rows, index)
        words = _fork_words(*self.table.shape, self.pages, True)
        ws = self.table.new_empty(words)
        a = _FORK.pack(*self._fork_to[:4], rows, each, *self._fork_to[4:], more, True, 0)
        with self._lock:  # the launches of one call stay together
            rc = load().voom_kv_fork(a, ws.data_ptr(), 4 * words, _device.raw_stream(index))
        _refused(rc, "voom_kv_fork")

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, *, index: torch.Tensor | None = None,
               stream: torch.cuda.Stream | None = None) -> None:
        """kv_append to one layer, into room that the last fork has made with grow=..;
        what there is no room for is not written."""
        kv_append(self._views[layer], k, v, index=index, stream=stream)

    def advance(self, n: int | torch.Tensor) -> None:
        """Counts n (one number, or int32 for each row) appended positions: after
        the last layer's append.  An ended or empty row that was not written to
        must get 0, and no row more than the last fork made room for: nothing else
        says that a position was not written."""
        self.lengths.add_(n).clamp_(0, self.max_len)

    def compact(self, *, stream: torch.cuda.Stream | None = None) -> torch.Tensor:
        """compact_pages in place; the number of pages in use, on the device.  Room
        that the last fork made and nothing has filled yet stays."""
        if stream is not None or _device.current_index() != self._index:
            with _device.on_stream(self.k.device, stream):
                return self.compact()
        with self._lock:
            return compact_pages(self.k, self.v, self.table, self.lengths, room=True,
                                 out=Compacted(self.table, self.table.new_empty(1))).live

    def resize(self, pages: int) -> None:
        """Compacts the pool and gives it `pages` pages, those in use at least.
        Synchronises; views taken before are not valid any more, and hold the old
        memory for as long as they live.  Beside the pool it needs room for the new
        keys, then for the new values.  Where that is not to be had the error goes
        on to the caller and the pool stays usable: it keeps its pages, or (where
        the values of a smaller one had no room) the fewer that were asked for."""
        live = int(self.compact().item())
        if pages < max(live, 1):
            raise ValueError(f"{live} pages are in use, {pages} do not hold them")
        refs = self.refs.new_zeros(pages)

        def moved(x):
            y = x.new_empty((x.shape[0], pages, *x.shape[2:]))
            y[:, :live] = x[:, :live]
            return y

        with self._lock:
            self._views = []  # they hold the old keys and values: these are given back one after the other
            try:
                self.k = moved(self.k)
                self.v = moved(self.v)
            finally:
                if self.k.shape != self.v.shape:  # the values had no room: both hold this many
                    n = min(self.k.shape[1], self.v.shape[1])
                    self.k, self.v = self.k[:, :n], self.v[:, :n]
                self.refs = refs if self.pages == pages else self.refs[:self.pages]
                self._make_views()

    def check_status(self) -> None:
        """Raises RuntimeError if pages were missing in a fork since the last
        check (positions past the pool's room were not written), or a wait inside an
        attention kernel over view() ran out.  Synchronises; call it where results
        are read.  Right after a fork that lacked pages nothing is lost yet: resize,
        then fork(grow=..) again, and go on."""
        from .kv_attention import check_wait_status

        check_wait_status(self._wait_status)
        n = int(self.missing.item())
        if n:
            self.missing.zero_()
            raise RuntimeError(f"the pool of {self.pages} pages had {n} too few")
