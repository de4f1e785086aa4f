"""A key-value cache in pages, shared by many requests, and the operators over it (include/vpass.h, vp_paged_*).

    kv = PagedKV(n_layers=24, n_pages=4096, page_size=64, max_seqs=64, max_len=4096)
    kv.reserve(seq, n_slots)                              # pages for a request, from the pool
    q = kv[l].append(q, k, v, seq, slot, pos, rope)       # rotate; keys and values into their pages
    o = kv[l].prefill(q, q_start, lens)                   # attention of prompt rows, ragged batch
    o = kv[l].decode(q, lens, mask=ancestors)             # attention of the newest row(s) per request
    kv.release(seq)

`kv[l]` is a PagedLayer; it can also be built over pools and a table that the caller owns. Like an engine's context, a cache
(and the layers of one PagedKV) serves one stream at a time. Calls run on torch's current stream, allocate only their
results, synchronise nothing and can be captured in a CUDA graph; they have no gradients, and refuse tensors that want
one. What the device finds wrong (a page or slot outside the table) is told by `check()`. The reference keeps one contiguous
cache of one request (Engine.swift:113).
"""
from __future__ import annotations

import ctypes
from typing import Optional

import torch

from . import _lib
from ._lib import VpError, VpPaged, check
from .synth import tree_to_buffer

TYPES = {torch.float16: 0, torch.bfloat16: 1}
DEV_ERR_TIMEOUT, DEV_ERR_PAGE, DEV_ERR_SLOT = 4, 16, 32
MAX_ROWS = 16
WORK_ZEROED = 16384  # VP_PAGED_WORK_ZEROED


def _extension():
    """The tensor side of the calls (csrc/paged_torch.cpp); like the library below it, it has no fallback."""
    try:
        from . import _paged
    except ImportError as e:
        raise VpError(f"instantllm_b200/_paged.so cannot be loaded ({e}): build it with instantllm_b200.build.build_torch()") from e
    return _paged


def _not_captured() -> None:
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise VpError("a layer cannot get its status or workspace while a graph is captured: only the replay would zero them")


def _workspace(work: list, head_dim: int, device: torch.device) -> None:
    """work[0] becomes a workspace for every call over heads of this size, its counters zeroed: a call never allocates one, since
    a captured graph holds its address and would only record the zeroing. A smaller one that was there moves back in the
    list: graphs may hold its address too."""
    # a record has 256 rows at most, whatever the call: this is the most (0 for heads that every call refuses)
    need = _lib.load().vp_paged_work_bytes(head_dim, 64, 1, MAX_ROWS)
    if work and work[0] is not None and work[0].nbytes >= need:
        return
    _not_captured()
    new = torch.empty(max(need, WORK_ZEROED), dtype=torch.uint8, device=device)
    new[:WORK_ZEROED].zero_()
    work[:] = [new] + [w for w in work if w is not None]


def rope_table(rows: int, rot_dim: int = 64, theta: float = 1e6, device=0) -> torch.Tensor:
    """(cos, sin) of the rotation, fp32 [rows][rot_dim / 2][2], angles computed in double."""
    f = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    a = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def ancestor_masks(trees) -> torch.Tensor:
    """Ancestor bitmasks int32 [n][16] of draft trees (dicts as in synth.seeded_tree), the row's own bit included: the last
    part of the verify pass's tree buffer. Unused rows are 0."""
    out = torch.zeros((len(trees), MAX_ROWS), dtype=torch.int32)
    for i, t in enumerate(trees):
        out[i, :t["n"]] = torch.from_numpy(tree_to_buffer(t)[49:49 + t["n"]])
    return out


class PagedLayer:
    """One layer of a paged cache. k, v: [pages][heads][page_size][head_dim] in fp16 or bf16, elements of a slot adjacent, any
    strides in multiples of 8 elements (a [pages][page_size][heads][head_dim] pool transposed will do), the same for both;
    table: int32 [requests][pages per request]. status (int32 [1]) and work (a list that holds the workspace, or [None]) may be
    shared between layers that run on one stream. The workspace (43 MB at head_dim 64, 85 at 128) is made here, once, for
    calls of any size, so that graphs may capture any of them, the first one included."""

    def __init__(self, k: torch.Tensor, v: torch.Tensor, table: torch.Tensor, status: Optional[torch.Tensor] = None,
                 work: Optional[list] = None):
        if k.dim() != 4 or k.shape != v.shape or k.stride() != v.stride() or k.dtype != v.dtype or k.device != v.device:
            raise ValueError("k and v must be [pages][heads][page_size][head_dim] pools of one shape, layout and type")
        if k.dtype not in (torch.float16, torch.bfloat16) or not k.is_cuda:
            raise ValueError("the pools must be fp16 or bf16 on a CUDA device")
        if k.stride(3) != 1:
            raise ValueError("the elements of a slot must be adjacent")
        if table.dtype != torch.int32 or table.dim() != 2 or table.device != k.device or table.stride(1) != 1:
            raise ValueError("table must be an int32 [requests][pages] tensor on the pools' device, rows contiguous")
        _lib.load()
        self.k, self.v, self.table, self.device, self.dtype = k, v, table, k.device, k.dtype
        self.pages, self.n_kv, self.page_size, self.head_dim = k.shape
        if status is None:
            _not_captured()
            status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self.status, self._work = status, [None] if work is None else work
        _workspace(self._work, self.head_dim, k.device)
        n, width = table.shape
        # strides of extents of 1 mean nothing: the dense ones stand in for them
        slot = k.stride(2)
        head = k.stride(1) if self.n_kv > 1 else slot * self.page_size
        page = k.stride(0) if self.pages > 1 else max(head * self.n_kv, slot * self.page_size)
        self._c = VpPaged(k.data_ptr(), v.data_ptr(), table.data_ptr(), status.data_ptr(), page, head, slot,
                          table.stride(0) if n > 1 else width, TYPES[k.dtype], self.n_kv, self.head_dim, self.page_size,
                          self.pages, n, width)
        self._at = ctypes.addressof(self._c)
        ext = _extension()
        self._append, self._attend = ext.append, ext.attend

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seq: torch.Tensor, slot: torch.Tensor,
               pos: Optional[torch.Tensor], rope: Optional[torch.Tensor], interleaved: bool = False,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Rows q [rows][query heads][head_dim], k, v [rows][heads][head_dim] (the cache's type or fp32; slices of one fused
        projection will do): keys rotated to pos and values go to slot[t] of request seq[t] (seq < 0: not stored), the
        rotated queries are returned, in the cache's type. rope: fp32 [positions][rot_dim / 2][2] (rope_table), None for
        no rotation; interleaved: pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)."""
        r = self._append(self._at, self.device.index, q, k, v, seq, slot, pos, rope, interleaved, out)
        return r if r.__class__ is not int else check(r, "vp_paged_append")

    def decode(self, q: torch.Tensor, lens: torch.Tensor, mask: Optional[torch.Tensor] = None,
               seqs: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of the newest rows: q [n][rows][query heads][head_dim] (or [n][query heads][head_dim] for one row each) are
        the last slots of lens[i] (already appended); rows <= 16. mask: int32 [n][rows], bit j of a row's word shows it new
        slot j (its own bit included; ancestor_masks), None for a causal chain. seqs: int32 [n], the requests' rows of the
        table (None: 0 .. n - 1). window > 0: a row sees the last `window` positions and the first `sinks`. Returns out
        like q, and with return_lse the log sum exp fp32 [n][rows][query heads]."""
        r = self._attend(False, self._at, self.device.index, self._work, q, lens, mask, None, seqs, window, sinks, scale, out, return_lse)
        return r if r.__class__ is not int else check(r, "vp_paged_decode")

    def prefill(self, q: torch.Tensor, q_start: torch.Tensor, lens: torch.Tensor, seqs: Optional[torch.Tensor] = None,
                window: int = 0, sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                return_lse: bool = False):
        """Causal attention of prompt rows: q [rows][query heads][head_dim], rows q_start[i] .. q_start[i + 1] - 1 being the last
        slots of lens[i] (already appended). Other arguments and results as in decode."""
        r = self._attend(True, self._at, self.device.index, self._work, q, lens, None, q_start, seqs, window, sinks, scale, out, return_lse)
        return r if r.__class__ is not int else check(r, "vp_paged_prefill")

    def check(self) -> None:
        """Raises VpError if a call met a page or slot outside the table, or gave up a wait, since the last check();
        synchronises."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
            if bits & DEV_ERR_TIMEOUT:  # a call that gave up may have left counters that the next one would start from
                for w in self._work:
                    w[:WORK_ZEROED].zero_()
            raise VpError("the cache's calls met " + " and ".join(t for b, t in (
                (DEV_ERR_PAGE, "a page outside the pool"),
                (DEV_ERR_SLOT, "a request, slot, position or length outside the table"),
                (DEV_ERR_TIMEOUT, "a wait that ran out: their results are void")) if bits & b))


class PagedKV:
    """The pools, the table and the free pages of one model's cache: k, v [layers][pages][heads][page_size][head_dim].
    Pages are handed out on the host; the table's rows follow on the stream."""

    def __init__(self, n_layers: int, n_pages: int, page_size: int = 64, max_seqs: int = 64, max_len: int = 4096,
                 n_kv: int = 2, head_dim: int = 64, dtype: torch.dtype = torch.float16, device: int = 0):
        if min(n_layers, n_pages, max_seqs, max_len) < 1:
            raise ValueError("layers, pages, requests and lengths must be positive")
        self.device = torch.device("cuda", device)
        self.page_size, self.max_len, self.n_pages = page_size, max_len, n_pages
        shape = (n_layers, n_pages, n_kv, page_size, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=self.device)
        self.v = torch.zeros(shape, dtype=dtype, device=self.device)
        width = -(-max_len // page_size)
        self.table = torch.full((max_seqs, width), -1, dtype=torch.int32, device=self.device)
        self.status = torch.zeros(1, dtype=torch.int32, device=self.device)
        work = [None]
        self.layers = [PagedLayer(self.k[i], self.v[i], self.table, self.status, work) for i in range(n_layers)]
        self._pool = PagePool(n_pages, page_size, max_seqs, width)

    def __getitem__(self, layer: int) -> PagedLayer:
        return self.layers[layer]

    def __len__(self) -> int:
        return len(self.layers)

    def reserve(self, seq: int, n_slots: int) -> None:
        """Pages so that request `seq` holds n_slots slots (its present pages stay). VpError when the pool is empty."""
        at, new = self._pool.reserve(seq, n_slots)
        if new:
            self.table[seq, at:at + len(new)] = torch.tensor(new, dtype=torch.int32).to(self.device)

    def reserve_all(self, slots: dict) -> None:
        """reserve(request, slots) for each of several requests, or VpError and no page to any of them."""
        self._pool.fits(slots)
        for seq, n_slots in slots.items():
            self.reserve(seq, n_slots)

    def release(self, seq: int) -> None:
        """All pages of request `seq` go back to the pool."""
        if self._pool.release(seq):
            self.table[seq].fill_(-1)

    @property
    def free_pages(self) -> int:
        return len(self._pool.free)

    def check(self) -> None:
        self.layers[0].check()


class PagePool:
    """Host side of the page table: which pages are free and which requests hold the others."""

    def __init__(self, n_pages: int, page_size: int, max_seqs: int, width: int):
        self.free = list(range(n_pages - 1, -1, -1))
        self.page_size, self.width = page_size, width
        self.held = [[] for _ in range(max_seqs)]

    def _known(self, seq: int) -> None:
        if not 0 <= seq < len(self.held):
            raise IndexError(f"request {seq}, and a table of {len(self.held)}")

    def fits(self, slots: dict) -> int:
        """Pages that the requests lack for these numbers of slots; VpError when the pool or a row of the table cannot hold them."""
        more = 0
        for seq, n_slots in slots.items():
            self._known(seq)
            need = -(-n_slots // self.page_size)
            if need > self.width:
                raise VpError(f"{n_slots} slots, and a table row of {self.width} pages of {self.page_size}")
            more += max(0, need - len(self.held[seq]))
        if more > len(self.free):
            raise VpError(f"{more} pages wanted, {len(self.free)} free")
        return more

    def reserve(self, seq: int, n_slots: int):
        """(first new entry of the request's row, the new pages). Nothing changes when the pool cannot serve it."""
        more = self.fits({seq: n_slots})
        held = self.held[seq]
        at = len(held)
        new = [self.free.pop() for _ in range(more)]
        held.extend(new)
        return at, new

    def release(self, seq: int):
        self._known(seq)
        held, self.held[seq] = self.held[seq], []
        self.free.extend(reversed(held))
        return held
