"""The paged key-value cache (include/vpass.h, vp_paged_*; instantllm_b200/paged.py) against the 64-bit oracle: rows
joining the cache with their rotation, attention of the newest rows, attention of prompts; sizes, masks and layouts at which
they can go wrong; refusals.

Tolerances. u is half a unit in the last place of the cache's type (2^-11 fp16, 2^-8 bf16: 11 and 8 significant bits). A rotated element is rounded
once from fp32: u |y| plus 4 ulp of the fp32 products. An attention output rounds its weights (u p each, or half of fp16's
smallest step 2^-24 below its normal range) and itself (u |o|); a score summed over head_dim products in fp32 is off by at most
head_dim 2^-23 sum |q k| scale, which moves a weight by that share, as the exponential's own error (2^-20) does."""
import ctypes
import random

import numpy as np
import pytest
import torch

from instantllm_b200 import _lib, build, paged
from oracle import paged as O

U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


# ------------------------------------------------------------------------------------------------
# host side (no GPU)


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def good_cache(**kw):
    c = dict(k=4096, v=8192, table=256, status=None, page_stride=2 * 64 * 64, head_stride=64 * 64, slot_stride=64,
             table_stride=4, type=0, n_kv=2, head_dim=64, page_size=64, n_pages=8, n_seqs=2, max_pages=4)
    c.update(kw)
    return _lib.VpPaged(**c)


def good_attn(**kw):
    a = dict(q=4096, out=8192, lse=None, lens=256, seqs=None, mask=None, q_start=512, work=1 << 20, work_bytes=1 << 30,
             q_seq=896, q_row=896, q_head=64, out_seq=896, out_row=896, out_head=64, scale=0.125, n=1, rows=1, n_q=14,
             window=0, sinks=0)
    a.update(kw)
    return _lib.VpPagedAttn(**a)


def good_rows(**kw):
    r = dict(q=4096, k=8192, v=12288, q_out=16384, seq=256, slot=512, pos=768, rope=1024, q_row=896, q_head=64, k_row=128,
             k_head=64, v_row=128, v_head=64, out_row=896, out_head=64, type=0, rows=1, n_q=14, rope_rows=16, rot_dim=64,
             interleaved=0)
    r.update(kw)
    return _lib.VpPagedRows(**r)


BAD_CACHE = [dict(type=2), dict(type=7), dict(head_dim=96), dict(head_dim=32), dict(page_size=48), dict(page_size=8),
             dict(page_size=512), dict(n_kv=0), dict(n_pages=0), dict(max_pages=0), dict(k=None), dict(v=4104), dict(table=None),
             dict(page_stride=0), dict(head_stride=-64), dict(slot_stride=66), dict(page_stride=1 << 40), dict(table_stride=3),
             dict(max_pages=1 << 28, table_stride=1 << 28)]
BAD_ATTN = [dict(n=-1), dict(rows=-1), dict(n_q=13), dict(n_q=0), dict(n_q=2 * 65), dict(window=-1), dict(sinks=-1),
            dict(scale=0.0), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=None), dict(out=None), dict(lens=None),
            dict(q=4098), dict(out=8200), dict(q_row=900), dict(out_head=4), dict(work=None), dict(work=1 << 20 | 16)]
BAD_ROWS = [dict(type=1), dict(type=3), dict(rows=-1), dict(n_q=0), dict(rot_dim=8), dict(rot_dim=80), dict(rot_dim=-16),
            dict(rope_rows=0), dict(q=None), dict(k=None), dict(v=None), dict(q_out=None), dict(seq=None), dict(slot=None),
            dict(pos=None), dict(rope=None), dict(rope=1028), dict(q=4100), dict(k_row=132), dict(out_row=900)]


def test_refusals_without_device(lib):
    """Bad arguments are refused before any CUDA call; the addresses are never touched."""
    a, r = good_attn(), good_rows()
    for bad in BAD_CACHE:
        c = good_cache(**bad)
        for call, arg in ((lib.vp_paged_decode, a), (lib.vp_paged_prefill, a), (lib.vp_paged_append, r)):
            assert call(ctypes.addressof(c), ctypes.addressof(arg), None) == -1, bad
    c = good_cache()
    for bad in BAD_ATTN:
        a = good_attn(**bad)
        assert lib.vp_paged_decode(ctypes.addressof(c), ctypes.addressof(a), None) == -1, bad
        assert lib.vp_paged_prefill(ctypes.addressof(c), ctypes.addressof(a), None) == -1, bad
    for bad in BAD_ROWS:
        r = good_rows(**bad)
        assert lib.vp_paged_append(ctypes.addressof(c), ctypes.addressof(r), None) == -1, bad
    a = good_attn(rows=17)
    assert lib.vp_paged_decode(ctypes.addressof(c), ctypes.addressof(a), None) == -1
    assert b"16 rows" in lib.vp_last_error()
    a = good_attn(q_start=None)
    assert lib.vp_paged_prefill(ctypes.addressof(c), ctypes.addressof(a), None) == -1
    a = good_attn(work_bytes=0)
    assert lib.vp_paged_decode(ctypes.addressof(c), ctypes.addressof(a), None) == -1
    assert lib.vp_paged_prefill(ctypes.addressof(c), ctypes.addressof(a), None) == -1
    for call in (lib.vp_paged_decode, lib.vp_paged_prefill, lib.vp_paged_append):
        assert call(None, ctypes.addressof(a), None) == -1
        assert call(ctypes.addressof(c), None, None) == -1


def test_nothing_to_do_without_device(lib):
    c = good_cache()
    for kw in (dict(n=0), dict(rows=0)):
        a = good_attn(q=None, out=None, **kw)
        assert lib.vp_paged_decode(ctypes.addressof(c), ctypes.addressof(a), None) == 0
        assert lib.vp_paged_prefill(ctypes.addressof(c), ctypes.addressof(a), None) == 0
    r = good_rows(rows=0)
    assert lib.vp_paged_append(ctypes.addressof(c), ctypes.addressof(r), None) == 0


def test_work_bytes(lib):
    assert lib.vp_paged_work_bytes(64, 14, 2, 1) > 0
    assert lib.vp_paged_work_bytes(128, 32, 8, 16) >= lib.vp_paged_work_bytes(128, 32, 8, 1)
    for bad in ((96, 14, 2, 1), (64, 13, 2, 1), (64, 14, 0, 1), (64, 0, 2, 1), (64, 130, 2, 1), (64, 14, 2, 0)):
        assert lib.vp_paged_work_bytes(*bad) == 0


def test_layer_wants_cuda_pools():
    k = torch.zeros(2, 2, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError):
        paged.PagedLayer(k, k, torch.zeros(1, 2, dtype=torch.int32))
    with pytest.raises(ValueError):
        paged.PagedLayer(k, k[:, :1], torch.zeros(1, 2, dtype=torch.int32))


def test_extension_builds_and_refuses(lib):
    """The tensor side builds against the installed torch, loads beside the library and refuses a wrong call (no GPU)."""
    build.build_torch()
    from instantllm_b200 import _paged

    for call in (_paged.append, _paged.attend):
        with pytest.raises(ValueError, match="arguments"):
            call(1)


def test_page_pool():
    p = paged.PagePool(6, 16, 3, 4)
    assert p.reserve(0, 17) == (0, [0, 1])
    assert p.reserve(0, 32) == (2, [])
    assert p.reserve(1, 1) == (0, [2])
    assert p.reserve(0, 33) == (2, [3])
    with pytest.raises(_lib.VpError):
        p.reserve(2, 65)  # over the table row
    with pytest.raises(_lib.VpError):
        p.reserve(2, 48)  # two pages are left
    assert p.held[2] == [] and len(p.free) == 2
    assert p.release(0) == [0, 1, 3] and p.release(0) == []
    assert p.reserve(2, 64) == (0, [0, 1, 3, 4])


def test_ancestor_masks():
    t = {"n": 5, "depth": [0, 1, 1, 2, 3], "parent": [-1, 0, 0, 2, 3], "tok": [0] * 5}
    m = paged.ancestor_masks([t, {"n": 1, "depth": [0], "parent": [-1], "tok": [0]}])
    assert m.shape == (2, 16) and m.dtype == torch.int32
    assert m[0, :6].tolist() == [0b1, 0b11, 0b101, 0b1101, 0b11101, 0] and m[1, :2].tolist() == [1, 0]


def test_oracle_visibility():
    """The two forms of visibility agree where a tree is a chain, and a chain is the causal triangle."""
    chain = [(2 << r) - 1 for r in range(5)]
    for n in (3, 5, 9, 30):
        for w, s in ((0, 0), (1, 0), (4, 2), (7, 0)):
            t = O.sees_tree(n, chain, w, s)
            if n >= 5:
                assert (t == O.sees_prompt(n, 5, w, s)).all()
    assert O.sees_tree(3, chain, 0, 0).sum(1).tolist() == [0, 0, 1, 2, 3]


# ------------------------------------------------------------------------------------------------
# GPU


def make_cache(rng, lens, nkv, hd, ps, dtype, layout="hnd", spare=2, fill=None, extra_rows=0):
    """Pools with random pages for requests of these lengths (slots past a length hold `fill`), as (layer, k, v on the host in
    float64 [pages][heads][page_size][head_dim], table rows)."""
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + spare
    shape = (pages, nkv, ps, hd) if layout == "hnd" else (pages, ps, nkv, hd)
    order = list(rng.permutation(pages))
    width = max(need + [1]) + 1
    table = np.full((len(lens) + extra_rows, width), -1, dtype=np.int32)
    for i, n in enumerate(need):
        table[i, :n] = [order.pop() for _ in range(n)]
    pools = []
    for _ in range(2):
        p = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype)
        if fill is not None:
            keep = torch.zeros((pages, ps), dtype=torch.bool)
            for i, n in enumerate(lens):
                for j in range(n):
                    keep[table[i, j // ps], j % ps] = True
            view = p.transpose(1, 2) if layout == "hnd" else p
            view[~keep] = fill
        pools.append(p.cuda() if layout == "hnd" else p.cuda().transpose(1, 2))
    host = [p.cpu().double().numpy() for p in pools]
    t = torch.from_numpy(table).cuda()
    return paged.PagedLayer(pools[0], pools[1], t), host[0], host[1], table


def tolerance(o, spread, smax, n, hd, dtype):
    u = U[dtype]
    step = 2.0 ** -25 if dtype == torch.float16 else 0.0
    delta = hd * 2.0 ** -23 * smax + 2.0 ** -20
    return u * np.abs(o) + (u + 2 * delta) * spread + step * (n * spread.max(initial=0.0) + 1)


def compare(out, lse, want, dtype, hd):
    """out [..][hd], lse [..] against a list of (index, (o, lse, spread, smax), slots seen)."""
    out = out.double().cpu().numpy()
    lse = lse.double().cpu().numpy()
    assert np.isfinite(out).all()
    for at, (o, le, spread, smax), n in want:
        off = np.abs(out[at] - o)
        tol = tolerance(o, spread, smax, n, hd, dtype)
        assert (off <= tol).all(), (at, float(off.max()), float(tol.min()))
        if np.isinf(le):
            assert lse[at] == -np.inf and (out[at] == 0).all(), at
        else:
            assert abs(lse[at] - le) <= hd * 2.0 ** -23 * smax + 2.0 ** -20 + 2.0 ** -22 * abs(le), at


def tree_masks(rng, n, rows):
    m = np.zeros((n, rows), dtype=np.int64)
    for i in range(n):
        for r in range(rows):
            m[i, r] = (m[i, rng.integers(0, r)] if r else 0) | 1 << r
    return m


def want_decode(q, k, v, table, lens, masks, window, sinks, scale, ps, seqs=None, clip=None):
    n, rows, nq, hd = q.shape
    group = nq // k.shape[1]
    want = []
    for i, length in enumerate(lens):
        row = table[i if seqs is None else seqs[i]]
        ks, vs = (O.slots(p, row, length) for p in (k, v))
        seen = O.sees_tree(length, [int(x) for x in masks[i]], window, sinks)
        for r in range(rows):
            for h in range(nq):
                want.append(((i, r, h), O.attend(q[i, r, h], ks[h // group], vs[h // group], seen[r], scale), int(seen[r].sum())))
    return want


SHAPES = [(14, 2, 64, torch.float16, 64, "hnd"), (14, 2, 64, torch.bfloat16, 16, "nhd"), (8, 2, 128, torch.bfloat16, 32, "hnd"),
          (4, 4, 128, torch.float16, 256, "nhd"), (9, 1, 64, torch.float16, 128, "hnd"), (64, 1, 64, torch.float16, 16, "hnd")]


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,hd,dtype,ps,layout", SHAPES)
@pytest.mark.parametrize("rows", [1, 2, 5, 16])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (5, 3), (64, 0), (100, 70)])
def test_decode(nq, nkv, hd, dtype, ps, layout, rows, window, sinks):
    """Lengths of zero, one, around a tile and a page and past several, NaN in every unused slot, requests shorter than their
    rows, random trees."""
    rng = np.random.default_rng(rows * 1000 + window + nq + ps)
    lens = [300, 0, 1, 15, 16, 17, 63, 64, 65, 128, 257, 2 * rows + 1, rows]
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype, layout, fill=float("nan"))
    q = torch.from_numpy(rng.standard_normal((len(lens), rows, nq, hd)).astype(np.float32)).to(dtype)
    masks = tree_masks(rng, len(lens), rows)
    chain = rows == 5
    if chain:
        masks[:] = [(2 << r) - 1 for r in range(rows)]
    out, lse = kv.decode(q.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                         mask=None if chain else torch.from_numpy(masks.astype(np.int32)).cuda(), window=window, sinks=sinks,
                         return_lse=True)
    kv.check()
    compare(out, lse, want_decode(q.double().numpy(), k, v, table, lens, masks, window, sinks, hd ** -0.5, ps), dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,nq,nkv,ps,dtype", [(64, 14, 2, 64, torch.float16), (128, 8, 2, 16, torch.bfloat16)])
def test_decode_long_and_uneven(hd, nq, nkv, ps, dtype):
    """One long request beside short ones (its length is split and joined), single rows given as [n][heads][head_dim] slices of
    one projection, a scale of the caller's, and the same bits when called again."""
    rng = np.random.default_rng(hd)
    lens = [9001, 3, 700, 1, 4097, 0]
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype)
    fused = torch.from_numpy(rng.standard_normal((len(lens), (nq + 2 * nkv) * hd)).astype(np.float32)).to(dtype).cuda()
    q = fused[:, :nq * hd].unflatten(1, (nq, hd))
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = kv.decode(q, ln, scale=0.2, return_lse=True)
    again = kv.decode(q, ln, scale=0.2)
    assert out.shape == (len(lens), nq, hd) and torch.equal(out, again)
    masks = np.ones((len(lens), 1), dtype=np.int64)
    want = want_decode(q.double().cpu().numpy()[:, None], k, v, table, lens, masks, 0, 0, 0.2, ps)
    compare(out[:, None], lse[:, None], want, dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("hd,n,rows", [(64, 90001, 1), (128, 50001, 1), (64, 30011, 4), (64, 20001, 16)])
def test_decode_very_long(hd, n, rows):
    """Runs of many tiles per CTA: every stage of the ring is refilled many times."""
    rng = np.random.default_rng(n)
    nq, nkv, ps, dtype = 14, 2, 64, torch.float16
    kv, k, v, table = make_cache(rng, [n, 70], nkv, hd, ps, dtype)
    q = torch.from_numpy(rng.standard_normal((2, rows, nq, hd)).astype(np.float32)).to(dtype)
    masks = tree_masks(rng, 2, rows)
    out, lse = kv.decode(q.cuda(), torch.tensor([n, 70], dtype=torch.int32).cuda(), mask=torch.from_numpy(masks.astype(np.int32)).cuda(),
                         return_lse=True)
    kv.check()
    want = want_decode(q.double().numpy(), k, v, table, [n, 70], masks, 0, 0, hd ** -0.5, ps)
    compare(out, lse, want, dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,hd,rows,lens", [(1, 1, 64, 1, [60001]), (9, 1, 64, 1, [70003, 5]), (8, 1, 128, 1, [30001, 9, 12001]), (8, 1, 128, 2, [30001]),
                                                 (14, 2, 64, 2, [40001]), (5, 1, 128, 3, [6001, 0, 9001]), (32, 8, 128, 4, [13001]), (12, 4, 64, 4, [2001])])
def test_decode_joins_of_many_parts(nq, nkv, hd, rows, lens):
    """One head's slots over up to all CTAs: records joined at once, by eights, by eights of eights, call after call with
    the same bits."""
    rng = np.random.default_rng(lens[0] + nq)
    dtype, ps, n = torch.float16, 64, len(lens)
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype, fill=float("nan"))
    q = torch.from_numpy(rng.standard_normal((n, rows, nq, hd)).astype(np.float32)).to(dtype)
    masks = tree_masks(rng, n, rows)
    d, m, ln = q.cuda(), torch.from_numpy(masks.astype(np.int32)).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    outs = [kv.decode(d, ln, mask=m, return_lse=True) for _ in range(12)]
    kv.check()
    for o, lse in outs[1:]:
        assert torch.equal(o, outs[0][0]) and torch.equal(lse, outs[0][1])
    compare(*outs[0], want_decode(q.double().numpy(), k, v, table, lens, masks, 0, 0, hd ** -0.5, ps), dtype, hd)


@pytest.mark.gpu
def test_decode_large_scores_and_empty_masks():
    """Scores far past exp's range, rising and falling along the cache; rows whose mask has no bit see the old slots only, and
    nothing when there are none."""
    rng = np.random.default_rng(5)
    lens, hd, nq, nkv = [500, 2, 66], 64, 14, 2
    kv, k, v, table = make_cache(rng, lens, nkv, hd, 64, torch.float16)
    kv.k.mul_(30)
    k = kv.k.double().cpu().numpy()
    q = torch.from_numpy(20 * rng.standard_normal((3, 2, nq, hd)).astype(np.float32)).half()
    masks = np.array([[1, 0], [0, 0], [0, 3]])
    out, lse = kv.decode(q.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), mask=torch.from_numpy(masks.astype(np.int32)).cuda(),
                         return_lse=True)
    assert (out[1] == 0).all()
    compare(out, lse, want_decode(q.double().numpy(), k, v, table, lens, masks, 0, 0, hd ** -0.5, 64), torch.float16, hd)


@pytest.mark.gpu
def test_decode_requests_by_index_and_out_of_range():
    """seqs picks rows of the table; a request, a length or a page outside the cache is told by check(), the other requests
    are served."""
    rng = np.random.default_rng(6)
    lens, hd, nq, nkv, ps = [100, 40, 17], 64, 4, 2, 16
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, torch.float16)
    q = torch.from_numpy(rng.standard_normal((2, 1, nq, hd)).astype(np.float32)).half()
    seqs = [2, 0]
    ln = [lens[s] for s in seqs]

    def run(seqs, ln):
        return kv.decode(q.cuda(), torch.tensor(ln, dtype=torch.int32).cuda(), seqs=torch.tensor(seqs, dtype=torch.int32).cuda(),
                         return_lse=True)

    ones = np.ones((2, 1), dtype=np.int64)
    want = want_decode(q.double().numpy(), k, v, table, ln, ones, 0, 0, hd ** -0.5, ps, seqs)
    out, lse = run(seqs, ln)
    compare(out, lse, want, torch.float16, hd)
    kv.check()
    for bad_seq, bad_len in ((99, ln[1]), (-1, ln[1]), (0, -5)):
        o2, l2 = run([seqs[0], bad_seq], [ln[0], bad_len])
        assert torch.equal(o2[0], out[0]) and (o2[1] == 0).all() and (l2[1] == -np.inf).all()
        with pytest.raises(_lib.VpError, match="slot"):
            kv.check()
        kv.check()
    kv.table[0, 1] = 1 << 20  # a page that does not exist reads as zeros
    k[table[0, 1]], v[table[0, 1]] = 0, 0
    out, lse = run(seqs, ln)
    with pytest.raises(_lib.VpError, match="page"):
        kv.check()
    compare(out, lse, want_decode(q.double().numpy(), k, v, table, ln, ones, 0, 0, hd ** -0.5, ps, seqs), torch.float16, hd)


@pytest.mark.gpu
def test_window_reads_no_page_before_it():
    """Pages that a window has left behind may be anybody's: their table entries are not read."""
    rng = np.random.default_rng(7)
    lens, hd, nq, nkv, ps = [1000, 333], 64, 14, 2, 16
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, torch.float16)
    q = torch.from_numpy(rng.standard_normal((2, 1, nq, hd)).astype(np.float32)).half().cuda()
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    starts = torch.tensor([0, 1, 2], dtype=torch.int32).cuda()
    out = kv.decode(q, ln, window=64, sinks=4)
    pre = kv.prefill(q[:, 0].contiguous(), starts, ln, window=64, sinks=4)
    for i, n in enumerate(lens):
        kv.table[i, 1:(n - 64) // ps] = -7
        first = int(table[i, 0])  # beside the sinks, the first page holds whatever its next owner wrote
        kv.k[first, :, 4:] = float("nan")
        kv.v[first, :, 4:] = float("inf")
        edge = int(table[i, (n - 64) // ps])
        kv.v[edge, :, :(n - 64) % ps] = float("nan")
    assert torch.equal(kv.decode(q, ln, window=64, sinks=4), out)
    assert torch.equal(kv.prefill(q[:, 0].contiguous(), starts, ln, window=64, sinks=4), pre)
    kv.check()


def want_prefill(q, k, v, table, starts, lens, window, sinks, scale):
    group = q.shape[1] // k.shape[1]
    want = []
    for i, length in enumerate(lens):
        a, b = starts[i], starts[i + 1]
        ks, vs = (O.slots(p, table[i], length) for p in (k, v))
        new = b - a
        seen = np.zeros((new, length), dtype=bool)
        have = min(new, length)
        if have:
            seen[new - have:] = O.sees_prompt(length, have, window, sinks)
        for r in range(new):
            for h in range(q.shape[1]):
                want.append(((a + r, h), O.attend(q[a + r, h], ks[h // group], vs[h // group], seen[r], scale), int(seen[r].sum())))
    return want


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,hd,dtype,ps,layout", SHAPES)
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (7, 3), (130, 0), (64, 140)])
def test_prefill(nq, nkv, hd, dtype, ps, layout, window, sinks):
    """Whole prompts, chunks over a cached prefix, requests without rows, without slots, with more rows than slots."""
    rng = np.random.default_rng(window + nq + ps + hd)
    lens = [37, 0, 1, 129, 300, 64, 5, 400]
    new = [37, 0, 1, 129, 40, 3, 9, 1]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype, layout, fill=float("nan"))
    q = torch.from_numpy(rng.standard_normal((int(starts[-1]), nq, hd)).astype(np.float32)).to(dtype)
    out, lse = kv.prefill(q.cuda(), torch.from_numpy(starts.astype(np.int32)).cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                          window=window, sinks=sinks, return_lse=True)
    kv.check()
    compare(out, lse, want_prefill(q.double().numpy(), k, v, table, starts, lens, window, sinks, hd ** -0.5), dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv,hd,dtype", [(14, 2, 64, torch.float16), (4, 1, 128, torch.bfloat16)])
def test_prefill_long(nq, nkv, hd, dtype):
    """A prompt of many tiles, scores that rise along it (the running maximum moves far), and a chunk over a long prefix; the
    same bits when called again. Rows are sampled."""
    rng = np.random.default_rng(nq)
    lens, new = [1500, 3001], [1500, 77]
    starts = np.concatenate([[0], np.cumsum(new)])
    kv, k, v, table = make_cache(rng, lens, nkv, hd, 64, dtype)
    ramp = torch.zeros(kv.k.shape[0], 64, device="cuda")
    for i, n in enumerate(lens):
        for j in range(-(-n // 64)):
            ramp[int(table[i, j])] = 0.2 + 0.15 * j
    kv.k.mul_(ramp[:, None, :, None].to(dtype))
    k = kv.k.double().cpu().numpy()
    q = torch.from_numpy(3 * rng.standard_normal((int(starts[-1]), nq, hd)).astype(np.float32)).to(dtype)
    args = (q.cuda(), torch.from_numpy(starts.astype(np.int32)).cuda(), torch.tensor(lens, dtype=torch.int32).cuda())
    out, lse = kv.prefill(*args, return_lse=True)
    assert torch.equal(out, kv.prefill(*args))
    pick = sorted(rng.choice(int(starts[-1]), 40, replace=False))
    want = []
    for t in pick:
        i = int(np.searchsorted(starts, t, side="right") - 1)
        p = lens[i] - new[i] + t - starts[i]
        ks, vs = (O.slots(x, table[i], p + 1) for x in (k, v))
        for h in range(nq):
            g = h // (nq // nkv)
            want.append(((t, h), O.attend(q[t, h].double().numpy(), ks[g], vs[g], np.ones(p + 1, dtype=bool), hd ** -0.5), p + 1))
    compare(out, lse, want, dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["trees", "prompts", "chunks"])
def test_many_requests(kind):
    """More work than CTAs: every CTA goes through several requests, some of them cut in pieces, calls follow one another
    without a pause and give the same bits each time; rows are sampled."""
    rng = np.random.default_rng(11)
    nq, nkv, hd, ps, dtype = 14, 2, 64, 64, torch.float16
    lens = [int(x) for x in np.exp(rng.uniform(np.log(20), np.log(2500), 70))]
    lens[7], lens[40] = 6000, 0
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype, fill=float("nan"))
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    if kind == "trees":
        q = torch.from_numpy(rng.standard_normal((70, 16, nq, hd)).astype(np.float32)).to(dtype)
        masks = tree_masks(rng, 70, 16)
        d, m = q.cuda(), torch.from_numpy(masks.astype(np.int32)).cuda()
        outs = [kv.decode(d, ln, mask=m, return_lse=True) for _ in range(20)]
        pick = [3, 7, 40, 69]
        want = [((pick[at[0]],) + at[1:], o, n) for at, o, n in
                want_decode(q[pick].double().numpy(), k, v, table[pick], [lens[i] for i in pick], masks[pick], 0, 0, hd ** -0.5, ps)]
    else:
        new = [n if kind == "prompts" else min(n, 50) for n in lens]
        starts = np.concatenate([[0], np.cumsum(new)])
        q = torch.from_numpy(rng.standard_normal((int(starts[-1]), nq, hd)).astype(np.float32)).to(dtype)
        d, qs = q.cuda(), torch.from_numpy(starts.astype(np.int32)).cuda()
        outs = [kv.prefill(d, qs, ln, return_lse=True) for _ in range(20)]
        want = []
        for t in rng.choice(int(starts[-1]), 30, replace=False):
            i = int(np.searchsorted(starts, t, side="right") - 1)
            p = lens[i] - new[i] + t - starts[i]
            ks, vs = (O.slots(x, table[i], p + 1) for x in (k, v))
            for h in (0, 6, 7, 13):
                want.append(((t, h), O.attend(q[t, h].double().numpy(), ks[h // 7], vs[h // 7], np.ones(p + 1, dtype=bool), hd ** -0.5), p + 1))
    kv.check()
    for o, lse in outs[1:]:
        assert torch.equal(o, outs[0][0]) and torch.equal(lse, outs[0][1])
    compare(*outs[0], want, dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("n,length,hd,nkv", [(1, 1500, 64, 2), (3, 2000, 128, 2), (20, 700, 64, 2), (73, 300, 64, 2), (75, 333, 64, 2), (160, 90, 128, 1),
                                              (300, 50, 64, 3)])
def test_decode_of_equally_long_requests(n, length, hd, nkv):
    """About equal lengths: requests cut evenly, one pair of request and head a CTA, several of them."""
    rng = np.random.default_rng(n)
    nq, ps, dtype = 3 * nkv, 16, torch.float16
    lens = [int(x) for x in rng.integers(length - length // 20, length + 1, n)]
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype, fill=float("nan"))
    q = torch.from_numpy(rng.standard_normal((n, 1, nq, hd)).astype(np.float32)).to(dtype)
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    out, lse = kv.decode(q.cuda(), ln, return_lse=True)
    for _ in range(5):
        assert torch.equal(out, kv.decode(q.cuda(), ln))
    kv.check()
    compare(out, lse, want_decode(q.double().numpy(), k, v, table, lens, np.ones((n, 1), dtype=np.int64), 0, 0, hd ** -0.5, ps), dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [200, 1000, 2600])
def test_very_many_short_requests(n):
    """More requests than are sorted, than threads look at one each, than lengths are kept on the chip; every request checked
    by its log sum exp and output at one row."""
    rng = np.random.default_rng(n)
    nq, nkv, hd, ps, dtype = 6, 2, 64, 16, torch.float16
    lens = [int(x) for x in rng.integers(0, 40, n)]
    lens[n // 2], lens[n - 1] = 700, 300
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype, fill=float("nan"))
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    one = torch.from_numpy(rng.standard_normal((n, 1, nq, hd)).astype(np.float32)).to(dtype)
    ones = np.ones((n, 1), dtype=np.int64)

    def near(got, masks, q, rows):
        want = want_decode(q.double().numpy(), k, v, table, lens, masks, 0, 0, hd ** -0.5, ps)
        compare(*got, [w for w in want if w[0][1] == rows - 1 and w[0][2] in (0, 5)], dtype, hd)

    near(kv.decode(one.cuda(), ln, return_lse=True), ones, one, 1)
    trees = torch.from_numpy(rng.standard_normal((n, 7, nq, hd)).astype(np.float32)).to(dtype)
    chain = np.tile([(2 << r) - 1 for r in range(7)], (n, 1))
    near(kv.decode(trees.cuda(), ln, return_lse=True), chain, trees, 7)
    starts = torch.arange(n + 1, dtype=torch.int32).cuda() * 7
    out, lse = kv.prefill(trees.view(-1, nq, hd).cuda(), starts, ln, return_lse=True)
    near((out.view(n, 7, nq, hd), lse.view(n, 7, nq)), chain, trees, 7)
    kv.check()


@pytest.mark.gpu
def test_prompt_rows_that_overlap_are_told():
    """A q_start that runs backwards or past the rows: those requests are dropped or clipped, and check() tells it."""
    rng = np.random.default_rng(2)
    kv, *_ = make_cache(rng, [40, 40, 40], 2, 64, 16, torch.float16)
    q = torch.zeros(40, 4, 64, dtype=torch.float16, device="cuda")
    ln = torch.tensor([40, 40, 40], dtype=torch.int32).cuda()
    for bad in ([0, 30, 20, 40], [0, 10, 20, 90], [-3, 10, 20, 40]):
        kv.prefill(q, torch.tensor(bad, dtype=torch.int32).cuda(), ln)
        with pytest.raises(_lib.VpError, match="slot"):
            kv.check()
    kv.prefill(q, torch.tensor([0, 10, 20, 40], dtype=torch.int32).cuda(), ln)
    kv.check()


@pytest.mark.gpu
@pytest.mark.parametrize("window,sinks", [(2 ** 31 - 1, 2 ** 31 - 1), (2 ** 31 - 1, 0), (3, 2 ** 31 - 1), (2 ** 62, 2 ** 62)])
def test_windows_and_sinks_past_everything(window, sinks):
    """They are as none, and as all, also where a request is shorter than its new rows."""
    rng = np.random.default_rng(9)
    kv, *_ = make_cache(rng, [300, 3, 17], 2, 64, 16, torch.float16, fill=float("nan"))
    ln = torch.tensor([300, 3, 17], dtype=torch.int32).cuda()
    for rows, nq in ((5, 4), (16, 14)):
        q = torch.from_numpy(rng.standard_normal((3, rows, nq, 64)).astype(np.float32)).half().cuda()
        assert torch.equal(kv.decode(q, ln, window=window, sinks=sinks), kv.decode(q, ln))
        starts = torch.arange(4, dtype=torch.int32).cuda() * rows
        flat = q.view(-1, nq, 64)
        assert torch.equal(kv.prefill(flat, starts, ln, window=window, sinks=sinks), kv.prefill(flat, starts, ln))
    kv.check()


@pytest.mark.gpu
def test_c_entry_ignores_what_a_prompt_call_has_not():
    """vp_paged_prefill through the C ABI alone: the fields of a decode call (request strides, masks) hold anything."""
    rng = np.random.default_rng(8)
    kv, k, v, table = make_cache(rng, [50, 20], 2, 64, 16, torch.float16)
    q = torch.from_numpy(rng.standard_normal((60, 4, 64)).astype(np.float32)).half().cuda()
    ln, starts = torch.tensor([50, 20], dtype=torch.int32).cuda(), torch.tensor([0, 45, 60], dtype=torch.int32).cuda()
    want = kv.prefill(q, starts, ln)
    lib, out = _lib.load(), torch.zeros_like(q)
    work = torch.zeros(lib.vp_paged_work_bytes(64, 4, 2, 60), dtype=torch.uint8, device="cuda")
    a = _lib.VpPagedAttn(q.data_ptr(), out.data_ptr(), None, ln.data_ptr(), None, 4096, starts.data_ptr(), work.data_ptr(), work.numel(),
                         8 * 10 ** 9, 256, 64, -8 * 10 ** 9, 256, 64, 0.125, 2, 60, 4, 0, 0)
    _lib.check(lib.vp_paged_prefill(ctypes.addressof(kv._c), ctypes.addressof(a), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.gpu
def test_prompts_left_over_for_a_last_round():
    """As many equal blocks as leave a few over for a last round of the CTAs, against the oracle in sampled rows; the same bits
    each time."""
    rng = np.random.default_rng(12)
    nq, nkv, hd, dtype, rows = 4, 1, 64, torch.float16, 256
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    n = (sms + 5) // 4 + 1  # four blocks of 256 packed rows each
    lens = [int(x) for x in rng.integers(700, 900, n)]
    kv, k, v, table = make_cache(rng, lens, nkv, hd, 64, dtype, fill=float("nan"))
    q = torch.from_numpy(rng.standard_normal((n * rows, nq, hd)).astype(np.float32)).to(dtype)
    starts = torch.arange(n + 1, dtype=torch.int32).cuda() * rows
    args = (q.cuda(), starts, torch.tensor(lens, dtype=torch.int32).cuda())
    out, lse = kv.prefill(*args, return_lse=True)
    for _ in range(5):
        assert torch.equal(out, kv.prefill(*args))
    kv.check()
    want = []
    for i in range(n):
        for r in (0, 63, 64, 130, 255):
            p = lens[i] - rows + r
            ks, vs = (O.slots(x, table[i], p + 1) for x in (k, v))
            for h in (0, 3):
                t = i * rows + r
                want.append(((t, h), O.attend(q[t, h].double().numpy(), ks[0], vs[0], np.ones(p + 1, dtype=bool), hd ** -0.5), p + 1))
    compare(out, lse, want, dtype, hd)


@pytest.mark.gpu
@pytest.mark.parametrize("src,dtype", [(torch.float16, torch.float16), (torch.bfloat16, torch.bfloat16),
                                       (torch.float32, torch.float16), (torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("nq,nkv,hd,rot,interleaved,layout", [(14, 2, 64, 64, False, "hnd"), (8, 2, 128, 128, True, "nhd"),
                                                             (3, 1, 64, 32, False, "nhd"), (5, 5, 128, 48, True, "hnd"),
                                                             (14, 2, 64, 0, False, "hnd")])
def test_append(src, dtype, nq, nkv, hd, rot, interleaved, layout):
    """Slices of one projection, padding rows, rows out of range; slots that no row names keep their bits."""
    rng = np.random.default_rng(hd + rot + nq)
    lens, ps = [40, 1, 130], 16
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, dtype, layout)
    rows = 23
    fused = torch.from_numpy(rng.standard_normal((rows, nq + 2 * nkv, hd)).astype(np.float32)).to(src)
    d = fused.cuda()
    places = [(s, j) for s, n in enumerate(lens) for j in range(n)]
    rng.shuffle(places)
    seq = np.array([p[0] for p in places[:rows]], dtype=np.int32)
    slot = np.array([p[1] for p in places[:rows]], dtype=np.int32)
    pos = rng.integers(0, 200, rows).astype(np.int32)
    seq[4], seq[9] = -1, 77
    slot[11] = 10 ** 6
    pos[13] = 200
    rope = paged.rope_table(200, rot, 1e4) if rot else None
    q = kv.append(d[:, :nq], d[:, nq:nq + nkv], d[:, nq + nkv:], *(torch.from_numpy(x).cuda() for x in (seq, slot, pos)), rope,
                  interleaved=interleaved)
    with pytest.raises(_lib.VpError):
        kv.check()
    f = fused.double().numpy()
    cs = rope.cpu().numpy() if rot else np.zeros((200, 0, 2))
    want_q = np.zeros((rows, nq, hd))
    touched = np.zeros(k.shape[:1] + k.shape[2:3], dtype=bool)
    for t in range(rows):
        if rot and pos[t] >= 200:
            continue
        y = O.rotate(f[t], cs[min(pos[t], 199)], interleaved)
        want_q[t] = y[:nq]
        if 0 <= seq[t] < len(lens) and slot[t] < 1000:
            at = table[seq[t], slot[t] // ps], slot[t] % ps
            touched[at] = True
            k[at[0], :, at[1]], v[at[0], :, at[1]] = y[nq:nq + nkv], f[t, nq + nkv:]
    assert touched.sum() == rows - 4 + (0 if rot else 1)
    u = U[dtype]

    def near(got, want, size):
        got = got.double().cpu().numpy()
        assert (np.abs(got - want) <= u * np.abs(want) + 2.0 ** -22 * size + 2.0 ** -25).all()

    near(q, want_q, 8.0)
    gk, gv = kv.k.cpu(), kv.v.cpu()
    near(gk, k, 8.0)
    near(gv, v, 0.0)
    untouched = torch.from_numpy(~touched)
    for g, w in ((gk, k), (gv, v)):  # bit for bit
        assert np.array_equal(g.double().numpy().swapaxes(1, 2)[untouched.numpy()], w.swapaxes(1, 2)[untouched.numpy()])


@pytest.mark.gpu
def test_append_in_place_and_one_row():
    rng = np.random.default_rng(1)
    kv, k, v, table = make_cache(rng, [70], 2, 64, 64, torch.float16)
    x = torch.from_numpy(rng.standard_normal((1, 18, 64)).astype(np.float32)).half().cuda()
    idx = [torch.tensor([i], dtype=torch.int32).cuda() for i in (0, 69, 69)]
    rope = paged.rope_table(70)
    q = kv.append(x[:, :14], x[:, 14:16], x[:, 16:], *idx, rope)
    same = x[:, :14]
    assert kv.append(same, x[:, 14:16], x[:, 16:], *idx, rope, out=same) is same
    assert torch.equal(same, q)


@pytest.mark.gpu
@pytest.mark.parametrize("src", [torch.float16, torch.float32])
def test_append_large_call_equals_small_ones(src):
    """A call too large for L2 (it runs in another shape) writes the bits of the same rows in small calls."""
    nq, nkv, hd, ps, n = 32, 8, 128, 64, 3500
    g = torch.Generator(device="cuda").manual_seed(5)
    x = torch.randn((n, nq + 2 * nkv, hd), generator=g, device="cuda").to(src)
    pages = -(-n // ps)
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None]
    seq, slot = torch.zeros(n, dtype=torch.int32, device="cuda"), torch.arange(n, dtype=torch.int32, device="cuda")
    rope = paged.rope_table(n, hd)
    got = []
    for step in (n, 500):
        kv = paged.PagedLayer(*torch.zeros((2, pages, nkv, ps, hd), dtype=torch.float16, device="cuda"), table)
        q = [kv.append(x[a:a + step, :nq], x[a:a + step, nq:nq + nkv], x[a:a + step, nq + nkv:], seq[a:a + step], slot[a:a + step],
                       slot[a:a + step], rope) for a in range(0, n, step)]
        got.append((torch.cat(q), kv.k, kv.v))
    for a, b in zip(*got):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_past_32_bits():
    """A pool of more than 2^32 elements: its last page is written and read like its first."""
    hd, ps, nkv, nq = 64, 64, 2, 14
    pages = (1 << 32) // (hd * ps * nkv) + 40
    pool = torch.zeros((pages, nkv, ps, hd), dtype=torch.float16, device="cuda")
    rng = np.random.default_rng(2)
    n = 130
    ids = [pages - 1, 3, pages - 30]
    table = torch.tensor([ids], dtype=torch.int32).cuda()
    kv = paged.PagedLayer(pool, pool, table)  # keys and values in one pool: both read what is written last, the values
    x = torch.from_numpy(rng.standard_normal((n, nq + 2 * nkv, hd)).astype(np.float32)).half()
    d = x.cuda()
    zero = torch.zeros(n, dtype=torch.int32).cuda()
    slot = torch.arange(n, dtype=torch.int32).cuda()
    vals = d[:, nq:nq + nkv]
    q = kv.append(d[:, :nq], vals, vals, zero, slot, None, None)
    kv.check()
    k = np.zeros((3, nkv, ps, hd))
    for j in range(n):
        k[j // ps, :, j % ps] = x[j, nq:nq + nkv].double().numpy()
    assert torch.equal(pool[ids[2], :, 1].cpu(), x[n - 1, nq:nq + nkv])
    lens = torch.tensor([n], dtype=torch.int32).cuda()
    out, lse = kv.decode(q[-1:], lens, return_lse=True)
    qh = q.double().cpu().numpy()
    want = want_decode(qh[None, -1:], k, k, np.array([[0, 1, 2]]), [n], np.ones((1, 1), dtype=np.int64), 0, 0, hd ** -0.5, ps)
    compare(out[None], lse[None], want, torch.float16, hd)
    starts = torch.tensor([0, n], dtype=torch.int32).cuda()
    out, lse = kv.prefill(q, starts, lens, return_lse=True)
    compare(out, lse, want_prefill(qh, k, k, np.array([[0, 1, 2]]), [0, n], [n], 0, 0, hd ** -0.5), torch.float16, hd)


@pytest.mark.gpu
def test_refusals():
    rng = np.random.default_rng(3)
    kv, *_ = make_cache(rng, [20, 20], 2, 64, 16, torch.float16)
    q = torch.zeros(2, 1, 14, 64, dtype=torch.float16, device="cuda")
    ln = torch.tensor([20, 20], dtype=torch.int32).cuda()
    for bad in (dict(q=q.float()), dict(q=q.cpu()), dict(q=q[..., :32]), dict(lens=ln.long()), dict(lens=ln[:1]), dict(lens=ln.cpu()),
                dict(mask=torch.zeros(2, 2, dtype=torch.int32).cuda()), dict(out=q[:1]), dict(q=q[0, 0]),
                dict(q=torch.zeros(3, 1, 14, 64).half().cuda(), lens=torch.tensor([1, 1, 1], dtype=torch.int32).cuda())):
        with pytest.raises(ValueError):
            kv.decode(**{**dict(q=q, lens=ln), **bad})
    for bad in (dict(q=q[:, :, :13]), dict(window=-1), dict(sinks=-1), dict(scale=0.0),
                dict(q=torch.zeros(2, 17, 14, 64).half().cuda()),
                dict(q=torch.zeros(2 * 14 * 64 + 4).half().cuda()[4:].view(2, 1, 14, 64))):
        with pytest.raises(_lib.VpError):
            kv.decode(**{**dict(q=q, lens=ln), **bad})
    with pytest.raises(ValueError):
        kv.prefill(q[:, 0], torch.tensor([0, 1], dtype=torch.int32).cuda(), ln)
    with pytest.raises(ValueError):
        kv.prefill(q, torch.tensor([0, 1, 2], dtype=torch.int32).cuda(), ln)
    x = torch.zeros(2, 18, 64, dtype=torch.float16, device="cuda")
    i = torch.zeros(2, dtype=torch.int32, device="cuda")
    good = dict(q=x[:, :14], k=x[:, 14:16], v=x[:, 16:], seq=i, slot=i, pos=i, rope=paged.rope_table(8))
    for bad in (dict(k=x[:, 14:15]), dict(v=x[:, 14:15]), dict(q=x[:, :14].bfloat16()), dict(pos=None), dict(seq=i[:1]),
                dict(rope=paged.rope_table(8).half()), dict(q=x[:, :14, :32])):
        with pytest.raises(ValueError):
            kv.append(**{**good, **bad})
    with pytest.raises(_lib.VpError):
        kv.append(**{**good, "rope": paged.rope_table(8, 8)})
    with pytest.raises(ValueError):
        paged.PagedLayer(kv.k, kv.v, kv.table.long())
    with pytest.raises(ValueError):
        paged.PagedLayer(kv.k, kv.v.bfloat16(), kv.table)


@pytest.mark.gpu
def test_pool_of_a_model():
    """PagedKV: pages given, grown and returned; the table follows, and other requests' pages stay."""
    kv = paged.PagedKV(n_layers=2, n_pages=8, page_size=16, max_seqs=3, max_len=64)
    kv.reserve(0, 20)
    kv.reserve(1, 16)
    kv.reserve(0, 33)
    assert kv.table[0, :4].tolist() == [0, 1, 3, -1] and kv.table[1, 0].item() == 2 and kv.free_pages == 4
    kv.release(0)
    assert kv.table[0].tolist() == [-1] * 4 and kv.free_pages == 7 and kv.table[1, 0].item() == 2
    with pytest.raises(_lib.VpError):
        kv.reserve(2, 65)
    assert len(kv) == 2 and kv[1].k.data_ptr() == kv.k[1].data_ptr()
    kv.check()


@pytest.mark.gpu
def test_other_stream_and_graph():
    """Calls follow torch's current stream, and a captured append + decode step replays on new inputs."""
    rng = np.random.default_rng(4)
    lens, nq, nkv, hd = [200, 31], 14, 2, 64
    kv, k, v, table = make_cache(rng, lens, nkv, hd, 64, torch.float16)
    x = torch.from_numpy(rng.standard_normal((2, nq + 2 * nkv, hd)).astype(np.float32)).half().cuda()
    seq = torch.tensor([0, 1], dtype=torch.int32).cuda()
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    last = ln - 1
    rope = paged.rope_table(256)

    def step():
        q = kv.append(x[:, :nq], x[:, nq:nq + nkv], x[:, nq + nkv:], seq, last, last, rope)
        return kv.decode(q, ln)

    first = step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = step()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            third = step()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, second)
    x.copy_(x.flip(0))
    torch.cuda.synchronize()
    g.replay()
    torch.cuda.synchronize()
    replayed = third.clone()
    assert torch.equal(replayed, step()) and not torch.equal(replayed, first)


def test_workspace_serves_every_call(lib):
    """The workspace that a layer makes when it is built is the largest that any call asks for."""
    for hd in (64, 128):
        most = lib.vp_paged_work_bytes(hd, 64, 1, paged.MAX_ROWS)
        for nq, nkv in ((14, 2), (32, 8), (12, 12), (64, 1), (256, 4), (9, 1)):
            for rows in (1, 2, 3, 7, 15, 16, 17, 37, 64, 256, 5000, 1 << 24):
                assert 0 < lib.vp_paged_work_bytes(hd, nq, nkv, rows) <= most
    work = [None]
    paged._workspace(work, 64, "cpu")
    first = work[0]
    assert first.nbytes == lib.vp_paged_work_bytes(64, 64, 1, 16) and not first[:paged.WORK_ZEROED].any()
    paged._workspace(work, 64, "cpu")
    assert len(work) == 1 and work[0] is first
    paged._workspace(work, 128, "cpu")  # a layer of larger heads on the same list: the first one stays alive behind the new
    assert len(work) == 2 and work[1] is first and work[0].nbytes > first.nbytes


@pytest.mark.gpu
def test_graph_outlives_larger_calls():
    """A decode captured as the layer's very first call, then calls of every size before its first replay and between
    replays: the graph's results are the eager ones, no tensor of others is written, and eager calls before the first
    replay are right too."""
    rng = np.random.default_rng(21)
    lens, nq, nkv, hd = [9001, 3, 700], 14, 2, 64  # the first request is split and joined
    kv, k, v, table = make_cache(rng, lens, nkv, hd, 64, torch.float16)
    q = torch.from_numpy(rng.standard_normal((3, 1, nq, hd)).astype(np.float32)).half()
    d, ln = q.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    many = torch.from_numpy(rng.standard_normal((710, nq, hd)).astype(np.float32)).half().cuda()
    starts = torch.tensor([0, 400, 401, 710], dtype=torch.int32).cuda()
    tree = torch.from_numpy(rng.standard_normal((3, 16, nq, hd)).astype(np.float32)).half().cuda()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out, lse = kv.decode(d, ln, return_lse=True)
    eager = kv.decode(d, ln, return_lse=True)
    compare(*eager, want_decode(q.double().numpy(), k, v, table, lens, np.ones((3, 1), dtype=np.int64), 0, 0, hd ** -0.5, 64),
            torch.float16, hd)
    big = kv.prefill(many, starts, ln), kv.decode(tree, ln)
    others = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in (1 << 20, 1 << 21, 1 << 22, 1 << 24, 5 << 23) for _ in range(4)]
    for _ in range(3):
        out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
        assert torch.equal(kv.prefill(many, starts, ln), big[0]) and torch.equal(kv.decode(tree, ln), big[1])
    assert all(bool((x == 7).all()) for x in others)
    kv.check()
    with pytest.raises(_lib.VpError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            d + 1
            paged.PagedLayer(kv.k, kv.v, kv.table)
    g2 = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g2):  # another view of the cache, on the status and workspace that are there
        late = paged.PagedLayer(kv.k, kv.v, kv.table, kv.status, kv._work).decode(d, ln)
    g2.replay()
    torch.cuda.synchronize()
    assert torch.equal(late, eager[0])


@pytest.mark.gpu
def test_workspace_is_the_layers_own():
    """A workspace that somebody put in the place of the layer's is refused, not replaced."""
    rng = np.random.default_rng(22)
    kv, *_ = make_cache(rng, [20], 2, 64, 16, torch.float16)
    q, ln = torch.zeros(1, 1, 14, 64, dtype=torch.float16, device="cuda"), torch.tensor([20], dtype=torch.int32).cuda()
    mine = kv._work[0]
    kv._work[0] = mine[:1 << 16]
    with pytest.raises(ValueError, match="workspace"):
        kv.decode(q, ln)
    kv._work[0] = None
    with pytest.raises(ValueError, match="work"):
        kv.decode(q, ln)
    kv._work[0] = mine
    kv.decode(q, ln)
    kv.check()


def kernel_source(name):
    return (build.PKG / "csrc" / name).read_text()


def test_tile_kernel_goes_through_its_pieces_to_the_end():
    """A wait that runs out must end in a status. The tile kernel's softmax warps meet at named barriers, which have no limit and
    want all of them, so no role may leave by a flag that another has not seen yet: only the scheduler looks at it, and
    everybody leaves at the piece that says so, whose hand-over is always waited for. Copies that were not waited for land
    before the CTA ends. Told from the source: on a sound kernel no wait can be made to run out."""
    src = kernel_source("vp_paged_prefill.cuh")
    parts = [src.index(x) for x in ("---- softmax", "---- the CTA's pieces", "---- K and V tiles", "---- products")] + [len(src)]
    softmax, scheduler, producer, issuer = (src[a:b] for a, b in zip(parts, parts[1:]))
    assert "dead" not in softmax + issuer
    for role in (softmax, producer, issuer):
        loop = role[role.index("for (int r = 0;; ++r) {"):]
        assert [x.strip() for x in loop.splitlines() if "seq < 0" in x and "break" in x] == ["if (seq < 0) break;"]
        assert "wait_piece(&info_full" in role and "wait_warp(&info_full" not in role
        assert "pg_arrive(&info_empty" in role[role.index("if (seq < 0) break;"):]
    assert "wait_piece(&info_empty" in scheduler and "__any_sync(0xffffffffu, piece < 0 || *(volatile int*)&dead)" in scheduler
    waits = src[src.index("auto wait_piece"):src.index("if (warp >= 8) asm")]
    assert "pg_wait" not in waits and waits.count("dead") == 1  # it sets the flag, and does not look at it
    assert producer.count("gone = !wait_warp") == 2 and "if (gone) break;" in producer
    assert "mbar_wait_warp(&edge" in producer


def test_decode_refills_nothing_after_a_wait_that_ran_out():
    """A decode warp whose wait for a stage ran out asks for no more tiles (the copy may still arrive in the stage, and its barrier
    counts one at a time), and waits once more for what is in flight before the CTA may end. Told from the source."""
    src = kernel_source("vp_paged_decode.cuh")
    warps = src[src.index("---- consumers"):src.index("---- joiners")]
    at = warps.index("if (!wait(&full[warp][st]")
    block = warps[at:warps.index("const uint32_t kb", at)]
    assert "coming.any = false;" in block and "ahead.t = t1;" in block and "gave_up[warp] = k_th" in block
    end = warps[warps.index("w.advance(n);"):]
    assert "gave_up[warp]" in end and "mbar_wait_warp(&full[warp][k % DC_STAGES], (k / DC_STAGES) & 1)" in end
    assert "pg_wait(bar, parity, &dead)" in src and "!*(volatile int*)&dead" not in src  # lanes agree on the flag


@pytest.mark.gpu
def test_check_after_a_timeout_leaves_the_counters_zero():
    """What a call that gave up leaves behind (its status bit, counters that are not back at zero) is gone after check(), on
    every workspace that the layer has had; later calls are right."""
    rng = np.random.default_rng(23)
    lens, nq, nkv, hd = [9001, 3, 700], 14, 2, 64
    kv, k, v, table = make_cache(rng, lens, nkv, hd, 64, torch.float16)
    one = torch.from_numpy(rng.standard_normal((3, 1, nq, hd)).astype(np.float32)).half().cuda()
    tree = torch.from_numpy(rng.standard_normal((3, 16, nq, hd)).astype(np.float32)).half().cuda()
    ln = torch.tensor(lens, dtype=torch.int32).cuda()
    want = kv.decode(one, ln), kv.decode(tree, ln)
    kv.check()
    kv._work.append(torch.zeros(paged.WORK_ZEROED, dtype=torch.uint8, device="cuda"))
    for w in kv._work:  # set by hand, with no call under way
        w[:paged.WORK_ZEROED].fill_(1)
    kv.status.fill_(paged.DEV_ERR_TIMEOUT)
    with pytest.raises(_lib.VpError, match="void"):
        kv.check()
    assert not any(bool(w[:paged.WORK_ZEROED].any()) for w in kv._work)
    assert torch.equal(kv.decode(one, ln), want[0]) and torch.equal(kv.decode(tree, ln), want[1])
    kv.check()


def test_tensor_memory_is_taken_after_the_kernel_before():
    """A kernel whose prologue overlaps the one before it must hold nothing that that one could wait for. From the source."""
    src = kernel_source("vp_paged_prefill.cuh")
    body = src[src.index("k_paged_tiles(const"):]
    assert body.index("pdl_wait();") < body.index("tcgen05.alloc")


@pytest.mark.gpu
def test_overlapping_rows_past_a_count_of_32_bits():
    """Requests that all claim the same 2^30 rows have 2^32 pieces between them: told, and nothing is written."""
    rng = np.random.default_rng(24)
    n, rows = 1024, 1 << 30
    kv, *_ = make_cache(rng, [40] * 2, 2, 64, 16, torch.float16, extra_rows=n - 2)
    q = torch.zeros(1, 2, 64, dtype=torch.float16, device="cuda").expand(rows, 2, 64)
    out = torch.full((1, 2, 64), 7.0, dtype=torch.float16, device="cuda")
    starts = torch.tensor([0, rows] * (n // 2) + [0], dtype=torch.int32).cuda()
    kv.prefill(q, starts, torch.full((n,), 40, dtype=torch.int32, device="cuda"), out=out.expand(rows, 2, 64))
    with pytest.raises(_lib.VpError, match="slot"):
        kv.check()
    assert bool((out == 7).all())
    one, ln = torch.ones(40, 4, 64, dtype=torch.float16, device="cuda"), torch.tensor([40], dtype=torch.int32).cuda()
    kv.prefill(one, torch.tensor([0, 40], dtype=torch.int32).cuda(), ln)
    kv.check()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("kind,lift", [("one", 14), ("tree", 7), ("prompt", 7)])
def test_small_weights_of_many_slots(kind, lift, hd, dtype):
    """One slot far above 60,000 others whose weights, 2^-26.7 of its own each, carry all of the output: the weights that fp16
    rounds are taken 2^lift higher, so what is lost of each is at most half of 2^(-24 - lift)."""
    rng = np.random.default_rng(25)
    n, nq, ps, rows = 60001, 4, 64, {"one": 1, "tree": 5, "prompt": 5}[kind]
    kv, _, _, table = make_cache(rng, [n], 1, hd, ps, dtype)
    kv.k.zero_()
    kv.k[..., 0] = -18.5
    kv.v.copy_(1000 + torch.randint(-8, 9, kv.v.shape, device="cuda") * 4)
    top = int(table[0, 0])
    kv.k[top, 0, 3, 0] = 0
    kv.v[top, 0, 3] = 0
    k, v = kv.k.cpu().double().numpy(), kv.v.cpu().double().numpy()
    q = torch.zeros(1, rows, nq, hd, dtype=dtype)
    q[..., 0] = 1
    q[..., 1] = torch.arange(rows * nq).view(1, rows, nq)  # meets zeros
    ln = torch.tensor([n], dtype=torch.int32).cuda()
    if kind == "prompt":
        out, lse = (x[None] for x in kv.prefill(q[0].cuda(), torch.tensor([0, rows], dtype=torch.int32).cuda(), ln, scale=1.0, return_lse=True))
    else:
        out, lse = kv.decode(q.cuda(), ln, scale=1.0, return_lse=True)
    kv.check()
    out, lse = out.double().cpu().numpy(), lse.double().cpu().numpy()
    u, step = U[dtype], 2.0 ** (-25 - lift) if dtype == torch.float16 else 0.0
    ks, vs = (O.slots(p, table[0], n) for p in (k, v))
    for r in range(rows):
        seen = np.arange(n) <= n - rows + r
        o, le, spread, smax = O.attend(q[0, r, 0].double().numpy(), ks[0], vs[0], seen, 1.0)
        assert 0.5 < o.min()
        tol = u * np.abs(o) + (u + 2 * (hd * 2.0 ** -23 * smax + 2.0 ** -20)) * spread + step * n * np.abs(vs).max()
        assert (np.abs(out[0, r] - o) <= tol).all(), (r, float(np.abs(out[0, r] - o).max()), float(tol.min()))
        assert (np.abs(lse[0, r] - le) <= hd * 2.0 ** -23 * smax + 2.0 ** -20 + 2.0 ** -22 * abs(le)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("nq,nkv", [(4, 2), (14, 2)])  # both attention kernels
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (3, 2), (40, 0)])
def test_slots_that_no_row_sees_hold_anything(nq, nkv, window, sinks):
    """NaN and infinities in every slot that no row of the call sees: new slots outside all masks, new slots in a mask that the
    window has left behind, new slots that only rows before the first slot name, old slots just before every row's window."""
    rng = np.random.default_rng(26 + window)
    hd, ps, rows = 64, 16, 5
    lens = [300, 3, 77, 5, 140]
    masks = np.array([[0b00001, 0b00000, 0b00101, 0b00110, 0b00111], [0b11111] * 2 + [0b00100, 0b01000, 0b01100], [0b11111] * 5,
                      [0] * 5, [0b00011, 0b00011, 0b00111, 0b01110, 0b10110]])
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, torch.float16, fill=float("nan"))
    hidden = 0
    for i, n in enumerate(lens):
        seen = O.sees_tree(n, [int(m) for m in masks[i]], window, sinks).any(0)
        for j in np.flatnonzero(~seen):
            at = int(table[i, j // ps]), slice(None), j % ps
            kv.k[at], kv.v[at] = float("nan"), float("inf") if j % 2 else float("nan")
            k[at], v[at] = 0, 0
            hidden += 1
    assert hidden > 0
    q = torch.from_numpy(rng.standard_normal((len(lens), rows, nq, hd)).astype(np.float32)).half()
    out, lse = kv.decode(q.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), mask=torch.from_numpy(masks.astype(np.int32)).cuda(),
                         window=window, sinks=sinks, return_lse=True)
    kv.check()
    compare(out, lse, want_decode(q.double().numpy(), k, v, table, lens, masks, window, sinks, hd ** -0.5, ps), torch.float16, hd)


def test_prompt_calls_look_at_no_request_strides(lib):
    """Request strides of any value pass a prompt call's checks (here up to the next refusal, that of q_start) and are refused
    by a decode call; no device is needed."""
    c = good_cache()
    for kw in (dict(q_seq=3), dict(out_seq=-5), dict(q_seq=2 ** 63 - 1, out_seq=-(2 ** 63) + 1)):
        a = good_attn(q_start=None, **kw)
        assert lib.vp_paged_prefill(ctypes.addressof(c), ctypes.addressof(a), None) == -1
        assert b"q_start" in lib.vp_last_error()
        a = good_attn(n=2, **kw)
        assert lib.vp_paged_decode(ctypes.addressof(c), ctypes.addressof(a), None) == -1
        assert b"strides" in lib.vp_last_error()


@pytest.mark.gpu
def test_c_prompt_call_with_odd_request_strides():
    """The same through the C ABI: the outputs are those of the Python call."""
    rng = np.random.default_rng(27)
    kv, *_ = make_cache(rng, [50, 20], 2, 64, 16, torch.float16)
    q = torch.from_numpy(rng.standard_normal((60, 4, 64)).astype(np.float32)).half().cuda()
    ln, starts = torch.tensor([50, 20], dtype=torch.int32).cuda(), torch.tensor([0, 45, 60], dtype=torch.int32).cuda()
    want = kv.prefill(q, starts, ln)
    lib, out = _lib.load(), torch.zeros_like(q)
    work = torch.zeros(lib.vp_paged_work_bytes(64, 4, 2, 60), dtype=torch.uint8, device="cuda")
    a = _lib.VpPagedAttn(q.data_ptr(), out.data_ptr(), None, ln.data_ptr(), None, 0, starts.data_ptr(), work.data_ptr(), work.numel(),
                         12345, 256, 64, -3, 256, 64, 0.125, 2, 60, 4, 0, 0)
    _lib.check(lib.vp_paged_prefill(ctypes.addressof(kv._c), ctypes.addressof(a), torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def odd(t, dims):
    """t in memory of its own whose strides in these dimensions, all of one element, are odd numbers."""
    shape = list(t.shape)
    assert all(shape[d] == 1 for d in dims)
    strides = [7 + 2 * d if d in dims else x for d, x in enumerate(t.stride())]
    return t.as_strided(t.shape, strides)


@pytest.mark.gpu
def test_strides_of_extents_of_one_mean_nothing():
    """One row, one request, one head: whatever torch holds as their strides, the call is the contiguous one's."""
    rng = np.random.default_rng(28)
    kv, *_ = make_cache(rng, [50], 1, 64, 16, torch.float16)
    ln, starts = torch.tensor([50], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    idx = [torch.tensor([i], dtype=torch.int32).cuda() for i in (0, 49, 49)]
    rope = paged.rope_table(50)
    for nq, dims in ((1, (0, 1, 2)), (4, (0, 1))):
        q = torch.from_numpy(rng.standard_normal((1, 1, nq, 64)).astype(np.float32)).half().cuda()
        want = kv.decode(q, ln)
        assert torch.equal(kv.decode(odd(q, dims), ln, out=odd(torch.zeros_like(q), dims)), want)
        flat = tuple(d - 1 for d in dims if d)
        assert torch.equal(kv.decode(odd(q[0], flat), ln), want[0])
        assert torch.equal(kv.prefill(odd(q[0], flat), starts, ln, out=odd(torch.zeros_like(q[0]), flat)), kv.prefill(q[0], starts, ln))
        k, v = (torch.from_numpy(rng.standard_normal((1, 1, 64)).astype(np.float32)).half().cuda() for _ in range(2))
        turned = kv.append(q[0], k, v, *idx, rope)
        held = kv.k.clone(), kv.v.clone()
        got = kv.append(odd(q[0], flat), odd(k, (0, 1)), odd(v, (0, 1)), *idx, rope, out=odd(torch.zeros_like(q[0]), flat))
        assert torch.equal(got, turned) and torch.equal(kv.k, held[0]) and torch.equal(kv.v, held[1])
    kv.check()


@pytest.mark.gpu
@pytest.mark.parametrize("nq", [4, 14])
def test_results_into_given_tensors_and_strided_queries(nq):
    """out= with strides of its own, four-dimensional queries that are slices, pools whose heads lie further apart than their
    slots: the bits of the contiguous call, and nothing beside them."""
    rng = np.random.default_rng(29)
    n, rows, hd, nkv, ps, lens = 3, 5, 64, 2, 16, [300, 40, 77]
    kv, k, v, table = make_cache(rng, lens, nkv, hd, ps, torch.float16)
    wide = torch.full((2, kv.pages, nkv + 1, ps + 3, hd + 8), 5.0, dtype=torch.float16, device="cuda")
    for x, y in zip(wide, (kv.k, kv.v)):
        x[:, :nkv, :ps, :hd] = y
    far = paged.PagedLayer(wide[0, :, :nkv, :ps, :hd], wide[1, :, :nkv, :ps, :hd], kv.table)
    big = torch.from_numpy(rng.standard_normal((n, rows + 2, nq + 3, hd + 8)).astype(np.float32)).half().cuda()
    q = big[:, 1:rows + 1, 2:nq + 2, 8:]
    ln, starts = torch.tensor(lens, dtype=torch.int32).cuda(), torch.arange(n + 1, dtype=torch.int32).cuda() * rows

    def given(*shape):
        x = torch.full((*shape[:-2], shape[-2] + 1, shape[-1] + 8), 9.0, dtype=torch.float16, device="cuda")
        return x, x[..., :shape[-2], :shape[-1]]

    want, wl = kv.decode(q.contiguous(), ln, return_lse=True)
    for c in (kv, far):
        whole, out = given(n, rows, nq, hd)
        got, gl = c.decode(q, ln, out=out, return_lse=True)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want) and torch.equal(gl, wl)
        out.fill_(9)
        assert bool((whole == 9).all())
        whole, out = given(n * rows, nq, hd)
        flat = q.contiguous().view(n * rows, nq, hd)
        c.prefill(flat, starts, ln, out=out)
        assert torch.equal(out, kv.prefill(flat, starts, ln))
        out.fill_(9)
        assert bool((whole == 9).all())
        c.check()
    x = torch.from_numpy(rng.standard_normal((n, 2 * nkv, hd)).astype(np.float32)).half().cuda()
    seq, last = torch.arange(n, dtype=torch.int32).cuda(), ln - 1
    a = kv.append(q[:, 0].contiguous(), x[:, :nkv], x[:, nkv:], seq, last, last, paged.rope_table(400))
    whole, out = given(n, nq, hd)
    far.append(q[:, 0], x[:, :nkv], x[:, nkv:], seq, last, last, paged.rope_table(400), out=out)
    assert torch.equal(out, a) and torch.equal(far.k, kv.k) and torch.equal(far.v, kv.v)
    out.fill_(9)
    far.k.fill_(5), far.v.fill_(5)
    assert bool((whole == 9).all()) and bool((wide == 5).all())


@pytest.mark.gpu
def test_tensors_that_want_a_gradient_are_refused():
    """The operators have no backward, so they say so instead of returning a result without one."""
    rng = np.random.default_rng(30)
    kv, *_ = make_cache(rng, [20], 2, 64, 16, torch.float16)
    q = torch.from_numpy(rng.standard_normal((1, 14, 64)).astype(np.float32)).half().cuda()
    x = torch.from_numpy(rng.standard_normal((1, 4, 64)).astype(np.float32)).half().cuda()
    ln, starts = torch.tensor([20], dtype=torch.int32).cuda(), torch.tensor([0, 1], dtype=torch.int32).cuda()
    idx = [torch.tensor([i], dtype=torch.int32).cuda() for i in (0, 19, 19)]
    rope = paged.rope_table(20)
    g, y = q.clone().requires_grad_(), x.clone().requires_grad_()
    calls = [lambda q, x: kv.decode(q, ln), lambda q, x: kv.prefill(q, starts, ln),
             lambda q, x: kv.append(q, x[:, :2], x[:, 2:], *idx, rope)]
    for call in calls:
        with pytest.raises(ValueError, match="gradient"):
            call(g, y)
        want = call(q, x)
        with torch.no_grad():
            assert torch.equal(call(g, y), want)
        assert torch.equal(call(g.detach(), y.detach()), want)
    with pytest.raises(ValueError, match="gradient"):
        calls[2](q, y)
    kv.check()


def test_page_pool_knows_its_requests():
    """A request below zero is none: it does not stand for one counted from the end."""
    p = paged.PagePool(6, 16, 3, 4)
    p.reserve(2, 20)
    for seq in (-1, -3, 3):
        with pytest.raises(IndexError, match="request"):
            p.reserve(seq, 64)
        with pytest.raises(IndexError, match="request"):
            p.release(seq)
    assert p.held == [[], [], [0, 1]] and len(p.free) == 4
