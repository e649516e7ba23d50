"""The paged key-value cache that attention layers are served from.

A pool of fixed-size pages [layers, n_pages, Hkv, page, D] for keys and one for
values; a table [rows, width] says which pages hold a row's tokens (one table
for all layers), ``lengths`` how many there are, ``refs`` how many rows use a
page (0: free).  All of it is on the device, and so is the bookkeeping
(csrc/kv_pages.hip): nothing here waits for the host, and pages are taken
lowest index first, so results do not depend on timing.  Tokens are taken back by
lowering a row's length, not below what it shares with a fork: the pages behind
it stay the row's until it is freed, or until a reserve that comes to their
entries gives them back for the ones that it takes.

The functions work on the tensors; ``PagedKVCache`` keeps them together with
the rows' lengths on the host, and raises before a call that cannot be served.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib, attention
from .ops import _need, tensor_version, upload_ints


def _ints(*ts):
    for t in ts:
        _need(t.is_cuda and t.dtype == torch.int32 and t.is_contiguous() and t.device == ts[0].device,
              "tables, lengths, counts and slots must be contiguous int32 tensors on one CUDA (HIP) device")


def _state(table, lengths, refs):
    _ints(table, lengths, refs)
    _need(table.dim() == 2 and tuple(lengths.shape) == (table.shape[0],) and refs.dim() == 1,
          "table must be [rows,width], lengths [rows], refs [n_pages]")
    return table.shape[0], table.shape[1], refs.shape[0]


def _pools(k_pages, v_pages, ints, n_pages=None):
    """(layers, n_pages, Hkv, page, D, dtype code) of a pool with or without its layer axis."""
    _need(k_pages.is_cuda and k_pages.shape == v_pages.shape and k_pages.dim() in (4, 5)
          and k_pages.dtype == v_pages.dtype and k_pages.is_contiguous() and v_pages.is_contiguous()
          and k_pages.device == v_pages.device == ints.device,
          "k_pages and v_pages must be contiguous CUDA (HIP) tensors of one shape [(layers,)n_pages,Hkv,page,D], "
          "on the table's device")
    shape = tuple(k_pages.shape) if k_pages.dim() == 5 else (1, *k_pages.shape)
    _need(n_pages is None or shape[1] == n_pages, f"the pool has {shape[1]} pages, refs {n_pages}")
    return (*shape, _lib.dtype_code(k_pages.dtype))


def _workspace(n, n_pages, device):
    return torch.empty(_lib.load().gdnx_pages_workspace_bytes(n, n_pages), dtype=torch.uint8, device=device)


def pages_reserve(table, lengths, refs, slots, n_new: int, page: int, status):
    """Pages for the next n_new tokens of every row of slots (int32 [n]; outside
    the table: an empty row), whose lengths grow by as much.  Returns start
    [n], the old lengths (-1: an empty row).  If the pool or a table row is too
    small for any of them, nothing changes, start is -1 and status (int32 [2])
    holds the pages missing and the rows too short."""
    rows, width, n_pages = _state(table, lengths, refs)
    _ints(table, slots, status)
    _need(slots.dim() == 1 and tuple(status.shape) == (2,), "slots must be [n], status [2]")
    start = torch.empty_like(slots)
    if slots.numel() == 0:
        return start
    ws = _workspace(slots.numel(), n_pages, table.device)
    _lib.call("gdnx_pages_reserve", table.device, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(),
              slots.data_ptr(), start.data_ptr(), status.data_ptr(), ws.data_ptr(), slots.numel(), int(n_new), rows,
              width, n_pages, int(page))
    return start


def pages_write(k, v, k_pages, v_pages, table, slots, start):
    """Keys and values k, v [(layers,)n,T,Hkv,D] to the positions start[i] ..
    start[i] + T - 1 of table row slots[i] (start < 0: none of it)."""
    layers, n_pages, Hkv, page, D, code = _pools(k_pages, v_pages, table)
    _ints(table, slots, start)
    _need(table.dim() == 2 and slots.dim() == 1 and start.shape == slots.shape,
          "table must be [rows,width], slots and start [n]")
    lead = (layers,) if k_pages.dim() == 5 else ()
    _need(k.shape == v.shape and k.dim() == len(lead) + 4 and tuple(k.shape[:len(lead) + 1]) == (*lead, slots.numel())
          and tuple(k.shape[-2:]) == (Hkv, D), "k and v must be [(layers,)n,T,Hkv,D]")
    _need(k.dtype == v.dtype == k_pages.dtype and k.device == v.device == k_pages.device,
          "k, v and the pages must share dtype and device")
    if k.numel() == 0:
        return
    k, v = attention._rows16(k.contiguous()), attention._rows16(v.contiguous())
    _lib.call("gdnx_pages_write", table.device, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(),
              table.data_ptr(), slots.data_ptr(), start.data_ptr(), layers, slots.numel(), k.shape[-3],
              table.shape[0], table.shape[1], n_pages, page, Hkv, D, code)


class PackedTokens(NamedTuple):
    """A batch of packed rows, as ``pages_reserve_packed`` lays it out (all int32, on the device)."""
    offsets: torch.Tensor     # [n+1] row i has tokens offsets[i] .. offsets[i+1] - 1
    start: torch.Tensor       # [n] the rows' lengths before (-1: an empty row)
    positions: torch.Tensor   # [tokens] a token's position in its row (-1: it has none)
    places: torch.Tensor      # [tokens] its place in the pool, page * page size + place in the page (-1: none)


def pages_reserve_packed(table, lengths, refs, slots, n_new, page: int, status, tokens: int) -> PackedTokens:
    """Pages for the next n_new[i] tokens (int32 [n], on the device; below 0:
    none) of every row slots[i] (outside the table: an empty row), whose
    lengths grow by as much, and the packed batch that these tokens make.
    tokens: the batch's size, which may be more than the rows' tokens (those
    behind the last row's are nobody's).  No row may be named twice.  If the pool
    or a table row is too small for any of them, or the batch is, nothing changes, all offsets are 0,
    start, positions and places -1, and status (int32 [2]) holds the pages
    missing and the rows that do not fit."""
    rows, width, n_pages = _state(table, lengths, refs)
    _ints(table, slots, n_new, status)
    _need(slots.dim() == 1 and n_new.shape == slots.shape and tuple(status.shape) == (2,),
          "slots and n_new must be [n], status [2]")
    n, tokens, dev = slots.numel(), int(tokens), table.device
    _need(tokens >= 0, "tokens must not be negative")
    buf = torch.empty(2 * n + 1 + 2 * tokens, dtype=torch.int32, device=dev)
    plan = PackedTokens(buf[:n + 1], buf[n + 1:2 * n + 1], buf[2 * n + 1:2 * n + 1 + tokens], buf[2 * n + 1 + tokens:])
    if n == 0:
        plan.offsets.zero_()
        buf[1:].fill_(-1)
        return plan
    ws = torch.empty(attention._bytes("gdnx_pages_packed_workspace_bytes", n, n_pages), dtype=torch.uint8, device=dev)
    _lib.call("gdnx_pages_reserve_packed", dev, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(), slots.data_ptr(),
              n_new.data_ptr(), *(t.data_ptr() for t in plan), status.data_ptr(), ws.data_ptr(), n, tokens, rows, width,
              n_pages, int(page))
    return plan


def pages_write_packed(k, v, k_pages, v_pages, places):
    """Keys and values k, v [(layers,)N,Hkv,D] (any strides: views of a fused
    projection are read as they are) of packed tokens to their places in the
    pool (int32 [N]; outside it: not written).  No place may be named twice."""
    layers, n_pages, Hkv, page, D, code = _pools(k_pages, v_pages, places)
    _ints(places)
    lead = (layers,) if k_pages.dim() == 5 else ()
    N = places.numel()
    _need(places.dim() == 1 and tuple(k.shape) == tuple(v.shape) == (*lead, N, Hkv, D),
          "k and v must be [(layers,)N,Hkv,D], places [N]")
    _need(k.dtype == v.dtype == k_pages.dtype and k.device == v.device == k_pages.device,
          "k, v and the pages must share dtype and device")
    if k.numel() == 0:
        return
    k, v = (attention._rows16(t if lead else t.unsqueeze(0)) for t in (k, v))
    _lib.call("gdnx_pages_write_packed", places.device, k.data_ptr(), v.data_ptr(), k_pages.data_ptr(),
              v_pages.data_ptr(), places.data_ptr(), *attention._strides(k), *attention._strides(v), layers, N, n_pages,
              page, Hkv, D, code)


def pages_copy(k_pages, v_pages, src, dst):
    """Page src[i] onto page dst[i] (int32 [n]; either outside the pool:
    nothing) in every layer.  No page may be both a source and a destination."""
    layers, n_pages, Hkv, page, D, code = _pools(k_pages, v_pages, src)
    _ints(src, dst)
    _need(src.dim() == 1 and src.shape == dst.shape, "src and dst must be [n]")
    if src.numel() == 0:
        return
    _lib.call("gdnx_pages_copy", src.device, k_pages.data_ptr(), v_pages.data_ptr(), src.data_ptr(), dst.data_ptr(),
              layers, src.numel(), n_pages, page, Hkv, D, code)


def pages_fork(k_pages, v_pages, table, lengths, refs, parents, children, status):
    """Row children[i] (empty until now) becomes a copy of row parents[i]: full
    pages are shared, a started last page is copied to a free one.  If the pool
    lacks pages, nothing changes and status[0] holds how many were missing."""
    rows, width, n_pages = _state(table, lengths, refs)
    layers, _, Hkv, page, D, code = _pools(k_pages, v_pages, table, n_pages)
    _ints(table, parents, children, status)
    _need(parents.dim() == 1 and parents.shape == children.shape and tuple(status.shape) == (2,),
          "parents and children must be [n], status [2]")
    n = parents.numel()
    if n == 0:
        return
    ws = _workspace(n, n_pages, table.device)
    _lib.call("gdnx_pages_fork", table.device, k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(),
              lengths.data_ptr(), refs.data_ptr(), parents.data_ptr(), children.data_ptr(), status.data_ptr(),
              ws.data_ptr(), layers, n, rows, width, n_pages, page, Hkv, D, code)


def pages_free(table, lengths, refs, slots):
    """The rows of slots give back their pages and are empty."""
    rows, width, n_pages = _state(table, lengths, refs)
    _ints(table, slots)
    if slots.numel() == 0:
        return
    _lib.call("gdnx_pages_free", table.device, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(),
              slots.data_ptr(), slots.numel(), rows, width, n_pages)


def pages_trim(table, lengths, refs, slots, window: int, sinks: int, page: int):
    """The rows of slots give back the pages that hold no sink and lie wholly
    before their last ``window`` tokens; they keep their lengths."""
    rows, width, n_pages = _state(table, lengths, refs)
    _ints(table, slots)
    if slots.numel() == 0:
        return
    _lib.call("gdnx_pages_trim", table.device, table.data_ptr(), lengths.data_ptr(), refs.data_ptr(),
              slots.data_ptr(), int(window), int(sinks), slots.numel(), rows, width, n_pages, int(page))


def pages_compact(k_pages, v_pages, table, refs, out=None):
    """Moves the used pages at or beyond the number of used pages, in order, into
    the free pages below it.  Returns (table, refs) as they are then: the
    inputs, changed in place, or the pair of tensors ``out``."""
    layers, n_pages, Hkv, page, D, code = _pools(k_pages, v_pages, table, refs.shape[0])
    _ints(table, refs)
    _need(table.dim() == 2 and refs.dim() == 1, "table must be [rows,width], refs [n_pages]")
    t_out, r_out = (table, refs) if out is None else out
    _ints(table, t_out, r_out)
    _need(t_out.shape == table.shape and r_out.shape == refs.shape, "out must have the shapes of table and refs")
    ws = _workspace(0, n_pages, table.device)
    _lib.call("gdnx_pages_compact", table.device, k_pages.data_ptr(), v_pages.data_ptr(), table.data_ptr(),
              refs.data_ptr(), t_out.data_ptr(), r_out.data_ptr(), ws.data_ptr(), layers, table.shape[0],
              table.shape[1], n_pages, page, Hkv, D, code)
    return t_out, r_out


class PagedKVCache:
    """A page pool with its table.  Rows are named by the caller as ints, or as
    the int32 tensor that ``rows_tensor`` made of them, so that a step's calls
    share one upload; neither waits for the device (another tensor is read
    back).  A graph captures the functions above on the cache's tensors: the
    lengths that the cache keeps on the host do not advance with a replay.  Lengths
    are not lowered here: tokens that may have to go again are tried on a fork."""

    def __init__(self, n_pages: int, page: int, Hkv: int, D: int, rows: int, max_len: int, layers: int = 1,
                 dtype=torch.bfloat16, device="cuda"):
        _need(n_pages > 0 and rows > 0 and max_len > 0 and layers > 0, "sizes must be positive")
        _need(page > 0 and page & (page - 1) == 0, f"page must be a power of two, got {page}")
        self.n_pages, self.page, self.Hkv, self.D, self.rows, self.layers = n_pages, page, Hkv, D, rows, layers
        self.device = torch.device(device)
        self.width = -(-max_len // page)
        self.k_pages = torch.zeros(layers, n_pages, Hkv, page, D, dtype=dtype, device=self.device)
        self.v_pages = torch.zeros_like(self.k_pages)
        ints = dict(dtype=torch.int32, device=self.device)
        self.table = torch.full((rows, self.width), -1, **ints)
        self.lengths = torch.zeros(rows, **ints)
        self.refs = torch.zeros(n_pages, **ints)
        self.status = torch.zeros(2, **ints)
        self.lens = [0] * rows                   # the lengths, on the host
        self._free_rows = list(range(rows - 1, -1, -1))
        self._free_bound = n_pages               # at least so many pages are free

    # ---- rows ----
    def alloc(self, n: int = 1) -> list:
        """n empty rows."""
        if n > len(self._free_rows):
            raise RuntimeError(f"page cache full: {n} rows asked, {len(self._free_rows)} free")
        return [self._free_rows.pop() for _ in range(n)]

    def _check_rows(self, rows):
        if isinstance(rows, torch.Tensor):
            made = getattr(rows, "named_rows", None)
            rows = made[0] if made and made[1] == tensor_version(rows) else rows.tolist()
        rows = [int(r) for r in rows]
        free = set(self._free_rows)
        if len(set(rows)) != len(rows):
            raise ValueError(f"rows {rows} name a row twice")
        for r in rows:
            if not 0 <= r < self.rows or r in free:
                raise ValueError(f"row {r} is not allocated")
        return rows

    def _upload(self, xs):
        return upload_ints(xs, self.device,
                           "rows named as ints cannot be captured: name them by a tensor that rows_tensor made before")

    def _named(self, rows):
        """The rows, checked, as a list and as a device tensor."""
        host = self._check_rows(rows)
        if isinstance(rows, torch.Tensor) and rows.dtype == torch.int32 and rows.device == self.table.device and (
                rows.is_contiguous()):
            return host, rows
        return host, self._upload(host)

    def rows_tensor(self, rows):
        """The rows as an int32 device tensor, checked (-1 is not a row here)."""
        if isinstance(rows, torch.Tensor):
            return rows
        host, t = self._named(rows)
        t.named_rows = host, tensor_version(t)
        return t

    def free(self, rows) -> None:
        rows, named = self._named(rows)
        pages_free(self.table, self.lengths, self.refs, named)
        for r in rows:
            self.lens[r] = 0
        self._free_rows.extend(rows)

    # ---- pages ----
    def pages_in_use(self) -> int:
        """Waits for the device."""
        return int((self.refs != 0).sum())

    def _take(self, need: int) -> None:
        if need > self._free_bound:              # what was freed since is not in the bound
            self._free_bound = self.n_pages - self.pages_in_use()
            if need > self._free_bound:
                raise RuntimeError(f"page cache full: {need} pages asked, {self._free_bound} free")
        self._free_bound -= need

    def reserve(self, rows, n_new: int = 1):
        """Room for the next n_new tokens of every row; returns start (int32 [n])."""
        n_new, (rows, named) = int(n_new), self._named(rows)
        _need(n_new >= 0, "n_new must not be negative")
        for r in rows:
            if self.lens[r] + n_new > self.width * self.page:
                raise ValueError(f"row {r}: {self.lens[r]} + {n_new} tokens, the table holds {self.width * self.page}")
        self._take(sum(-(-(self.lens[r] + n_new) // self.page) - -(-self.lens[r] // self.page) for r in rows))
        start = pages_reserve(self.table, self.lengths, self.refs, named, n_new, self.page, self.status)
        for r in rows:
            self.lens[r] += n_new
        return start

    def write(self, rows, start, k, v, layer=None) -> None:
        """Keys and values [(layers,)n,T,Hkv,D] (of one layer: [n,T,Hkv,D]) at the positions from start on."""
        kp, vp = (self.k_pages, self.v_pages) if layer is None else (self.k_pages[layer], self.v_pages[layer])
        pages_write(k, v, kp, vp, self.table, self.rows_tensor(rows), start)

    def step(self, layer: int, rows, q, k, v, *, window=None, sinks=0, scale=None, out=None):
        """One layer's attention of the rows' newest token (reserved before):
        ``attention.paged_attention_step`` on the cache's tensors."""
        return attention.paged_attention_step(q, k, v, self.k_pages[layer], self.v_pages[layer], self.table,
                                              self.lengths, slots=self.rows_tensor(rows), window=window, sinks=sinks,
                                              scale=scale, out=out)

    def reserve_packed(self, rows, n_new, tokens=None) -> PackedTokens:
        """Room for the next n_new[i] tokens (ints) of every row, and the packed
        batch that they make, of ``tokens`` tokens (None: as many as the rows')."""
        n_new, (rows, named) = [int(c) for c in n_new], self._named(rows)
        tokens = sum(n_new) if tokens is None else int(tokens)
        _need(len(n_new) == len(rows) and min(n_new, default=0) >= 0, "n_new must name a number of tokens for every row")
        _need(tokens >= sum(n_new), f"{sum(n_new)} tokens in a batch of {tokens}")
        for r, c in zip(rows, n_new):
            if self.lens[r] + c > self.width * self.page:
                raise ValueError(f"row {r}: {self.lens[r]} + {c} tokens, the table holds {self.width * self.page}")
        up = self._upload(n_new)
        self._take(sum(-(-(self.lens[r] + c) // self.page) - -(-self.lens[r] // self.page) for r, c in zip(rows, n_new)))
        plan = pages_reserve_packed(self.table, self.lengths, self.refs, named, up, self.page, self.status, tokens)
        for r, c in zip(rows, n_new):
            self.lens[r] += c
        return plan

    def write_packed(self, plan, k, v, layer=None) -> None:
        """Keys and values [(layers,)N,Hkv,D] (of one layer: [N,Hkv,D]) of a packed batch to their places."""
        kp, vp = (self.k_pages, self.v_pages) if layer is None else (self.k_pages[layer], self.v_pages[layer])
        pages_write_packed(k, v, kp, vp, plan.places)

    def chunk(self, layer: int, rows, plan, q, *, window=None, sinks=0, scale=None, out=None):
        """One layer's attention of a packed batch's tokens (reserved and written
        before): ``attention.paged_attention_chunk`` on the cache's tensors."""
        return attention.paged_attention_chunk(q, self.k_pages[layer], self.v_pages[layer], self.table, self.lengths,
                                               plan.offsets, slots=self.rows_tensor(rows), window=window, sinks=sinks,
                                               scale=scale, out=out)

    def fork(self, parents) -> list:
        """A new row for every entry of parents (a row may be named more than once), holding what it holds."""
        parents = [int(r) for r in (parents.tolist() if isinstance(parents, torch.Tensor) else parents)]
        self._check_rows(set(parents))
        if len(parents) > len(self._free_rows):
            raise RuntimeError(f"page cache full: {len(parents)} rows asked, {len(self._free_rows)} free")
        children = self._free_rows[::-1][:len(parents)]             # (what alloc gives)
        up = self._upload(parents + children)
        self._take(sum(self.lens[r] % self.page != 0 for r in parents))
        self.alloc(len(parents))
        pages_fork(self.k_pages, self.v_pages, self.table, self.lengths, self.refs, up[:len(parents)], up[len(parents):],
                   self.status)
        for p, c in zip(parents, children):
            self.lens[c] = self.lens[p]
        return children

    def trim(self, rows, window: int, sinks: int = 0) -> None:
        """For layers that all have this window: drops the pages it has left behind."""
        pages_trim(self.table, self.lengths, self.refs, self.rows_tensor(rows), window, sinks, self.page)

    def compact(self) -> None:
        """Gathers the pages in use at the front of the pool."""
        pages_compact(self.k_pages, self.v_pages, self.table, self.refs)
