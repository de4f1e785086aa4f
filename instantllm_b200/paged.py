"""A key-value cache in pages, shared by many requests, and the operators over it (include/vpass.h, vp_paged_*).

    kv = PagedKV(n_layers=24, n_pages=4096, page_size=64, max_seqs=64, max_len=4096)
    kv.reserve(seq, n_slots)                              # pages for a request, from the pool
    q = kv[l].append(q, k, v, seq, slot, pos, rope)       # rotate; keys and values into their pages
    o = kv[l].prefill(q, q_start, lens)                   # attention of prompt rows, ragged batch
    o = kv[l].decode(q, lens, mask=ancestors)             # attention of the newest row(s) per request
    kv.release(seq)

`kv[l]` is a PagedLayer; it can also be built over pools and a table that the caller owns. Like an engine's context, a cache
(and the layers of one PagedKV) serves one stream at a time. Calls run on torch's current stream, allocate only their
results, synchronise nothing and can be captured in a CUDA graph; what the device finds wrong (a page or slot outside the
table) is told by `check()`. The reference keeps one contiguous cache of one request (Engine.swift:113).
"""
from __future__ import annotations

import ctypes
import struct
from typing import Optional

import torch

from . import _lib
from ._lib import VpError, VpPaged, VpPagedAttn, VpPagedRows, check
from .synth import tree_to_buffer

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
DEV_ERR_TIMEOUT, DEV_ERR_PAGE, DEV_ERR_SLOT = 4, 16, 32
MAX_ROWS = 16
WORK_ZEROED = 16384

# The argument structs (VpPagedRows, VpPagedAttn) are packed in one go: a call of a few microseconds on the GPU should
# not take longer to prepare, and setting two dozen ctypes fields takes 2 us.
_ROWS = struct.Struct("8P8q6i")
_ATTN = struct.Struct("8PQ6qf5i")
assert _ROWS.size == ctypes.sizeof(VpPagedRows) and _ATTN.size <= ctypes.sizeof(VpPagedAttn)
_I32, _F32 = torch.int32, torch.float32


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


# the current stream's handle without a Stream object around it (2 us), where torch has it
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", lambda i: torch.cuda.current_stream(i).cuda_stream)


def _index(t: torch.Tensor, what: str, shape, device: int) -> int:
    if t.dtype is not _I32 or t.shape != shape or t.get_device() != device or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape} on cuda:{device}")
    return t.data_ptr()


class PagedLayer:
    """One layer of a paged cache. k, v: [pages][heads][page_size][head_dim] in fp16 or bf16, elements of a slot adjacent, any
    strides in multiples of 8 elements (a [pages][page_size][heads][head_dim] pool transposed will do), the same for both;
    table: int32 [requests][pages per request]. status: int32 [1] and work (uint8, zeroed) may be shared between layers that
    run on one stream."""

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
        self.lib = _lib.load()
        self.k, self.v, self.table, self.device, self.dtype = k, v, table, k.device, k.dtype
        self.pages, self.n_kv, self.page_size, self.head_dim = k.shape
        if status is None:
            status = torch.zeros(1, dtype=torch.int32, device=k.device)
        self.status, self._work = status, [None] if work is None else work
        n, width = table.shape
        # strides of extents of 1 mean nothing: the dense ones stand in for them
        slot = k.stride(2)
        head = k.stride(1) if self.n_kv > 1 else slot * self.page_size
        page = k.stride(0) if self.pages > 1 else max(head * self.n_kv, slot * self.page_size)
        self._c = VpPaged(k.data_ptr(), v.data_ptr(), table.data_ptr(), status.data_ptr(), page, head, slot,
                          table.stride(0) if n > 1 else width, TYPES[k.dtype], self.n_kv, self.head_dim, self.page_size,
                          self.pages, n, width)
        self._r, self._a = VpPagedRows(), VpPagedAttn()
        self._cp, self._rp, self._ap = (ctypes.addressof(x) for x in (self._c, self._r, self._a))
        self._index_of_device, self._need = self.device.index, {}

    def _stream(self) -> int:
        if torch.cuda.current_device() != self._index_of_device:
            raise ValueError(f"the cache lives on {self.device}: make it the current device")
        return _raw_stream(self._index_of_device)

    def _out(self, like: torch.Tensor, out: Optional[torch.Tensor]) -> torch.Tensor:
        if out is None:
            if like.dtype is self.dtype and like.is_contiguous():
                return torch.empty_like(like)
            return torch.empty(like.shape, dtype=self.dtype, device=self.device)
        if out.shape != like.shape or out.dtype is not self.dtype or out.get_device() != self._index_of_device or out.stride(-1) != 1:
            raise ValueError("out must have q's shape and the cache's type, elements of a head adjacent")
        return out

    def append(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seq: torch.Tensor, slot: torch.Tensor,
               pos: Optional[torch.Tensor], rope: Optional[torch.Tensor], interleaved: bool = False,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Rows q [rows][query heads][head_dim], k, v [rows][heads][head_dim] (the cache's type or fp32; slices of one fused
        projection will do): keys rotated to pos and values go to slot[t] of request seq[t] (seq < 0: not stored), the
        rotated queries are returned, in the cache's type. rope: fp32 [positions][rot_dim / 2][2] (rope_table), None for
        no rotation; interleaved: pairs (2i, 2i + 1) instead of (i, i + rot_dim / 2)."""
        if q.dim() != 3 or k.dim() != 3 or v.shape != k.shape or k.dtype != q.dtype or v.dtype != q.dtype:
            raise ValueError("q, k and v must be [rows][heads][head_dim] of one type")
        n, nq, hd = q.shape
        if k.shape != (n, self.n_kv, self.head_dim) or hd != self.head_dim:
            raise ValueError(f"expected k and v of shape {(n, self.n_kv, self.head_dim)} and heads of {self.head_dim}")
        if q.dtype is not self.dtype and q.dtype is not torch.float32:
            raise ValueError("rows must have the cache's type or fp32")
        qs, ks, vs = q.stride(), k.stride(), v.stride()
        if qs[2] != 1 or ks[2] != 1 or vs[2] != 1:
            raise ValueError("the elements of a head must be adjacent")
        dev = self._index_of_device
        if q.get_device() != dev or k.get_device() != dev or v.get_device() != dev:
            raise ValueError(f"rows must be on cuda:{dev}")
        shape = (n,)
        places = _index(seq, "seq", shape, dev), _index(slot, "slot", shape, dev)
        if rope is None:
            places += None, None
            turns = 0, 0
        else:
            if pos is None:
                raise ValueError("a rotation needs pos")
            rs = rope.shape
            if len(rs) != 3 or rs[2] != 2 or rope.dtype is not _F32 or not rope.is_contiguous() or rope.get_device() != dev:
                raise ValueError(f"rope must be a contiguous fp32 [positions][rot_dim / 2][2] tensor on cuda:{dev}")
            places += _index(pos, "pos", shape, dev), rope.data_ptr()
            turns = rs[0], 2 * rs[1]
        out = self._out(q, out)
        os = out.stride()
        _ROWS.pack_into(self._r, 0, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), *(x or 0 for x in places),
                        qs[0], qs[1], ks[0], ks[1], vs[0], vs[1], os[0], os[1],
                        TYPES[q.dtype], n, nq, *turns, 1 if interleaved else 0)
        rc = self.lib.vp_paged_append(self._cp, self._rp, self._stream())
        if rc:
            check(rc, "vp_paged_append")
        return out

    def decode(self, q: torch.Tensor, lens: torch.Tensor, mask: Optional[torch.Tensor] = None,
               seqs: Optional[torch.Tensor] = None, window: int = 0, sinks: int = 0, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None, return_lse: bool = False):
        """Attention of the newest rows: q [n][rows][query heads][head_dim] (or [n][query heads][head_dim] for one row each) are
        the last slots of lens[i] (already appended); rows <= 16. mask: int32 [n][rows], bit j of a row's word shows it new
        slot j (its own bit included; ancestor_masks), None for a causal chain. seqs: int32 [n], the requests' rows of the
        table (None: 0 .. n - 1). window > 0: a row sees the last `window` positions and the first `sinks`. Returns out
        like q, and with return_lse the log sum exp fp32 [n][rows][query heads]."""
        shape, qs = q.shape, q.stride()
        if len(shape) == 4:
            n, rows, nq, _ = shape
        elif len(shape) == 3:
            (n, nq, _), rows, qs = shape, 1, (qs[0], 0, qs[1], qs[2])
        else:
            raise ValueError("q must be [n][rows][query heads][head_dim] or [n][query heads][head_dim]")
        masks = 0 if mask is None else _index(mask, "mask", (n, rows), self._index_of_device)
        return self._attend(self.lib.vp_paged_decode, "vp_paged_decode", q, qs, n, rows, nq, lens, seqs, masks, 0, window, sinks,
                            scale, out, return_lse)

    def prefill(self, q: torch.Tensor, q_start: torch.Tensor, lens: torch.Tensor, seqs: Optional[torch.Tensor] = None,
                window: int = 0, sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                return_lse: bool = False):
        """Causal attention of prompt rows: q [rows][query heads][head_dim], rows q_start[i] .. q_start[i + 1] - 1 being the last
        slots of lens[i] (already appended). Other arguments and results as in decode."""
        if q.dim() != 3:
            raise ValueError("q must be [rows][query heads][head_dim]")
        n, qs = lens.shape[0], q.stride()
        starts = _index(q_start, "q_start", (n + 1,), self._index_of_device)
        return self._attend(self.lib.vp_paged_prefill, "vp_paged_prefill", q, (0, *qs), n, q.shape[0], q.shape[1], lens, seqs, 0,
                            starts, window, sinks, scale, out, return_lse)

    def _attend(self, call, name, q, qs, n, rows, nq, lens, seqs, masks, starts, window, sinks, scale, out, return_lse):
        dev = self._index_of_device
        if q.shape[-1] != self.head_dim or q.dtype is not self.dtype or q.get_device() != dev or qs[3] != 1:
            raise ValueError(f"q must be {self.dtype} heads of {self.head_dim} on {self.device}, elements of a head adjacent")
        places = _index(lens, "lens", (n,), dev)
        if seqs is not None:
            seqs = _index(seqs, "seqs", (n,), dev)
        elif n > self._c.n_seqs:
            raise ValueError(f"{n} requests, and a table of {self._c.n_seqs}")
        out = self._out(q, out)
        os = out.stride()
        if len(os) == 3:
            os = (0, *os) if starts else (os[0], 0, *os[1:])
        lse = torch.empty(q.shape[:-1], dtype=_F32, device=self.device) if return_lse else None
        need = self._need.get((nq, rows))
        if need is None:
            need = self._need[nq, rows] = self.lib.vp_paged_work_bytes(self.head_dim, nq, self.n_kv, rows)
        work = self._work[0]
        if work is None or work.numel() < need:
            work = self._work[0] = torch.empty(max(need, WORK_ZEROED), dtype=torch.uint8, device=self.device)
            work[:WORK_ZEROED].zero_()
        _ATTN.pack_into(self._a, 0, q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else 0, places, seqs or 0, masks, starts,
                        work.data_ptr(), work.numel(), qs[0], qs[1], qs[2], os[0], os[1], os[2],
                        self.head_dim ** -0.5 if scale is None else scale, n, rows, nq, window, sinks)
        rc = call(self._cp, self._ap, self._stream())
        if rc:
            check(rc, name)
        return (out, lse) if return_lse else out

    def check(self) -> None:
        """Raises VpError if a call met a page or slot outside the table, or gave up a wait, since the last check();
        synchronises."""
        bits = int(self.status.item())
        if bits:
            self.status.zero_()
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

    def reserve(self, seq: int, n_slots: int):
        """(first new entry of the request's row, the new pages). Nothing changes when the pool cannot serve it."""
        held = self.held[seq]
        need = -(-n_slots // self.page_size)
        if need > self.width:
            raise VpError(f"{n_slots} slots, and a table row of {self.width} pages of {self.page_size}")
        more = need - len(held)
        if more > len(self.free):
            raise VpError(f"{more} pages wanted, {len(self.free)} free")
        at = len(held)
        new = [self.free.pop() for _ in range(max(0, more))]
        held.extend(new)
        return at, new

    def release(self, seq: int):
        held, self.held[seq] = self.held[seq], []
        self.free.extend(reversed(held))
        return held
