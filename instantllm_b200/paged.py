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
from typing import Optional

import torch

from . import _lib
from ._lib import VpError, VpPaged, VpPagedAttn, VpPagedRows, check

TYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
DEV_ERR_TIMEOUT, DEV_ERR_PAGE, DEV_ERR_SLOT = 4, 16, 32
MAX_ROWS = 16
WORK_ZEROED = 8192


def rope_table(rows: int, rot_dim: int = 64, theta: float = 1e6, device=0) -> torch.Tensor:
    """(cos, sin) of the rotation, fp32 [rows][rot_dim / 2][2], angles computed in double."""
    f = theta ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64, device=device) / rot_dim)
    a = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * f
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def ancestor_masks(trees) -> torch.Tensor:
    """Ancestor bitmasks int32 [n][16] of trees in the verify pass's form (dicts of synth.seeded_tree and the like: n and
    parent), the row's own bit included; unused rows are 0."""
    out = torch.zeros((len(trees), MAX_ROWS), dtype=torch.int32)
    for i, t in enumerate(trees):
        anc = []
        for r in range(t["n"]):
            anc.append((0 if r == 0 else anc[t["parent"][r]]) | 1 << r)
        out[i, :t["n"]] = torch.tensor(anc, dtype=torch.int32)
    return out


def _index(t: torch.Tensor, what: str, shape, device) -> int:
    if t.dtype != torch.int32 or tuple(t.shape) != shape or t.device != device or not t.is_contiguous():
        raise ValueError(f"{what} must be a contiguous int32 tensor of shape {shape} on {device}")
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

    def _stream(self) -> int:
        if torch.cuda.current_device() != self.device.index:
            raise ValueError(f"the cache lives on {self.device}: make it the current device")
        return torch.cuda.current_stream(self.device).cuda_stream

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
        if q.device != self.device or k.device != self.device or v.device != self.device:
            raise ValueError(f"rows must be on {self.device}")
        if out is None:
            out = torch.empty((n, nq, hd), dtype=self.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype is not self.dtype or out.device != self.device or out.stride(2) != 1:
            raise ValueError("out must have q's shape and the cache's type, elements of a head adjacent")
        r, os = self._r, out.stride()
        r.q, r.k, r.v, r.q_out = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr()
        shape = (n,)
        r.seq, r.slot = _index(seq, "seq", shape, self.device), _index(slot, "slot", shape, self.device)
        if rope is None:
            r.pos = r.rope = None
            r.rope_rows = r.rot_dim = 0
        else:
            if pos is None:
                raise ValueError("a rotation needs pos")
            if rope.dim() != 3 or rope.shape[2] != 2 or rope.dtype is not torch.float32 or not rope.is_contiguous() \
                    or rope.device != self.device:
                raise ValueError(f"rope must be a contiguous fp32 [positions][rot_dim / 2][2] tensor on {self.device}")
            r.pos, r.rope = _index(pos, "pos", shape, self.device), rope.data_ptr()
            r.rope_rows, r.rot_dim = rope.shape[0], 2 * rope.shape[1]
        r.q_row, r.q_head, r.k_row, r.k_head, r.v_row, r.v_head = qs[0], qs[1], ks[0], ks[1], vs[0], vs[1]
        r.out_row, r.out_head = os[0], os[1]
        r.type, r.rows, r.n_q, r.interleaved = TYPES[q.dtype], n, nq, 1 if interleaved else 0
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
        one = q.dim() == 3
        if not one and q.dim() != 4:
            raise ValueError("q must be [n][rows][query heads][head_dim] or [n][query heads][head_dim]")
        n, nq = q.shape[0], q.shape[-2]
        rows = 1 if one else q.shape[1]
        a = self._a
        if mask is None:
            a.mask = None
        else:
            a.mask = _index(mask, "mask", (n, rows), self.device)
        out, lse = self._attend(q, n, rows, nq, lens, seqs, window, sinks, scale, out, return_lse)
        qs, os = q.stride(), out.stride()
        a.q_seq, a.q_head, a.out_seq, a.out_head = qs[0], qs[-2], os[0], os[-2]
        a.q_row, a.out_row = (0, 0) if one else (qs[1], os[1])
        a.q_start = None
        rc = self.lib.vp_paged_decode(self._cp, self._ap, self._stream())
        if rc:
            check(rc, "vp_paged_decode")
        return (out, lse) if return_lse else out

    def prefill(self, q: torch.Tensor, q_start: torch.Tensor, lens: torch.Tensor, seqs: Optional[torch.Tensor] = None,
                window: int = 0, sinks: int = 0, scale: Optional[float] = None, out: Optional[torch.Tensor] = None,
                return_lse: bool = False):
        """Causal attention of prompt rows: q [rows][query heads][head_dim], rows q_start[i] .. q_start[i + 1] - 1 being the last
        slots of lens[i] (already appended). Other arguments and results as in decode."""
        if q.dim() != 3:
            raise ValueError("q must be [rows][query heads][head_dim]")
        n, a = lens.shape[0], self._a
        a.q_start = _index(q_start, "q_start", (n + 1,), self.device)
        out, lse = self._attend(q, n, q.shape[0], q.shape[1], lens, seqs, window, sinks, scale, out, return_lse)
        qs, os = q.stride(), out.stride()
        a.q_seq = a.out_seq = 0
        a.q_row, a.q_head, a.out_row, a.out_head = qs[0], qs[1], os[0], os[1]
        a.mask = None
        rc = self.lib.vp_paged_prefill(self._cp, self._ap, self._stream())
        if rc:
            check(rc, "vp_paged_prefill")
        return (out, lse) if return_lse else out

    def _attend(self, q, n, rows, nq, lens, seqs, window, sinks, scale, out, return_lse):
        if q.shape[-1] != self.head_dim or q.dtype is not self.dtype or q.device != self.device or q.stride(-1) != 1:
            raise ValueError(f"q must be {self.dtype} heads of {self.head_dim} on {self.device}, elements of a head adjacent")
        a = self._a
        if out is None:
            out = torch.empty(q.shape, dtype=q.dtype, device=self.device)
        elif out.shape != q.shape or out.dtype is not q.dtype or out.device != self.device or out.stride(-1) != 1:
            raise ValueError("out must have q's shape and type, elements of a head adjacent")
        lse = torch.empty(q.shape[:-1], dtype=torch.float32, device=self.device) if return_lse else None
        a.q, a.out, a.lse = q.data_ptr(), out.data_ptr(), lse.data_ptr() if return_lse else None
        a.lens = _index(lens, "lens", (n,), self.device)
        if seqs is None:
            if n > self.table.shape[0]:
                raise ValueError(f"{n} requests, and a table of {self.table.shape[0]}")
            a.seqs = None
        else:
            a.seqs = _index(seqs, "seqs", (n,), self.device)
        need = self.lib.vp_paged_work_bytes(self.head_dim, nq, self.n_kv, rows)
        work = self._work[0]
        if work is None or work.numel() < need:
            work = self._work[0] = torch.empty(max(need, WORK_ZEROED), dtype=torch.uint8, device=self.device)
            work[:WORK_ZEROED].zero_()
        a.work, a.work_bytes = work.data_ptr(), work.numel()
        a.scale = self.head_dim ** -0.5 if scale is None else scale
        a.n, a.rows, a.n_q, a.window, a.sinks = n, rows, nq, window, sinks
        return out, lse

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
