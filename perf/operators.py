"""The paged-cache operators as they are timed: appending rotated keys and values, attention of the newest rows of many
requests, and attention of prompts, over one paged key-value cache.

`run` computes an operator in its plain form (elementary torch operations in 32 bits) or, with `own`, through
instantllm_b200.paged. Shapes are those of the framework's model (14 query and 2 key-value heads of 64, trees of 16 rows,
64 requests with prefixes of 128 to 2,048 tokens) and one generic wider one (32 and 8 heads of 128).
"""
import math
import random

import torch

own = False

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16}


def listed():
    model = {"nq": 14, "nkv": 2, "hd": 64, "dtype": "f16"}
    wide = {"nq": 32, "nkv": 8, "hd": 128, "dtype": "bf16"}
    return [
        # one request's next token joins its cache: the smallest call of a decode step
        dict(model, name="append_one", op="append", seqs=1, rows=1, lo=256, hi=256, page=64, layout="hnd", half=True),
        # the draft trees of 64 requests, 16 rows each, sliced out of one fused projection
        dict(model, name="append_trees", op="append", seqs=64, rows=16, lo=128, hi=2048, page=64, layout="hnd", half=True),
        # a batch of prompts (rows = 0: every slot of the request is new), slot-major pages
        dict(wide, name="append_prompts", op="append", seqs=13, rows=0, lo=257, hi=4099, page=16, layout="nhd", half=False),
        # one request's next token over a 256-token prefix
        dict(model, name="decode_one", op="decode", seqs=1, rows=1, lo=257, hi=257, page=64, layout="hnd", window=0, sinks=0),
        # 64 requests of uneven length, one token each
        dict(model, name="decode_many", op="decode", seqs=64, rows=1, lo=128, hi=2048, page=64, layout="hnd", window=0, sinks=0),
        # the same requests, each verifying a draft tree of 16 rows
        dict(model, name="decode_trees", op="decode", seqs=64, rows=16, lo=144, hi=2064, page=64, layout="hnd", window=0, sinks=0),
        # a few very long contexts: the bytes of the cache are all that counts
        dict(wide, name="decode_long", op="decode", seqs=4, rows=1, lo=60001, hi=131072, page=128, layout="hnd", window=0, sinks=0),
        # many long requests that see a window and the first four tokens
        dict(model, name="decode_window", op="decode", seqs=128, rows=1, lo=900, hi=16384, page=16, layout="nhd", window=1024, sinks=4),
        # one prompt of 256 tokens
        dict(model, name="prefill_one", op="prefill", seqs=1, rows=0, lo=256, hi=256, page=64, layout="hnd", window=0, sinks=0),
        # a ragged batch of prompts
        dict(model, name="prefill_ragged", op="prefill", seqs=16, rows=0, lo=128, hi=2048, page=64, layout="hnd", window=0, sinks=0),
        # one long prompt of the wider shape
        dict(wide, name="prefill_long", op="prefill", seqs=1, rows=0, lo=8192, hi=8192, page=128, layout="hnd", window=0, sinks=0),
        # the next 2,048 tokens of long prompts that see a window and the first four tokens
        dict(model, name="prefill_window", op="prefill", seqs=4, rows=2048, lo=6001, hi=8191, page=16, layout="nhd", window=1024, sinks=4),
    ]


def draw(rng):
    def log(a, b):
        return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))

    op = rng.choice(["append", "decode", "prefill"])
    nq, nkv, hd = rng.choice([(14, 2, 64), (14, 2, 64), (32, 8, 128), (12, 12, 64), (16, 4, 128), (9, 1, 64), (8, 1, 128)])
    c = {"op": op, "nq": nq, "nkv": nkv, "hd": hd, "dtype": rng.choice(["f16", "bf16"]),
         "page": rng.choice([16, 32, 64, 128]), "layout": rng.choice(["hnd", "nhd"])}
    if op == "append":
        rows = rng.choice([0, 1, 1, rng.randint(2, 16)])
        hi = log(64, 4096)
        most = 13 * 4099 * 48 * 128 // ((nq + 2 * nkv) * hd)  # elements of the largest listed call
        seqs = log(1, max(1, min(128, most // (3 * hi if rows == 0 else 16))))
        return dict(c, seqs=seqs, rows=rows, lo=max(16, hi // rng.randint(1, 8)), hi=hi, half=rng.random() < 0.7)
    window = rng.choice([0, 0, log(64, 2048)])
    c.update(window=window, sinks=rng.choice([0, 1, 4, 64]) if window else 0)
    if op == "decode":
        rows = rng.choice([1, 1, 1, 4, 16, rng.randint(2, 15)])
        hi = log(64, 131072)
        seqs = log(1, max(1, min(256, 300000 * 8 * 128 // (hi * nkv * hd * rows))))
        return dict(c, seqs=seqs, rows=rows, lo=max(rows, hi // rng.randint(1, 8)), hi=hi)
    hi = log(48, 8192)
    rows = rng.choice([0, 0, max(1, hi // rng.randint(2, 9))])
    seqs = log(1, max(1, min(32, 32 * 8192 * 8192 // (2 * nq * hi * hi))))
    return dict(c, seqs=seqs, rows=rows, lo=max(16, hi // rng.randint(1, 8)), hi=hi)


def lengths(case):
    """Slots in use per request (the new rows included), and new rows per request: fixed by the case alone."""
    rng = random.Random("%d %d %d" % (case["seqs"], case["lo"], case["hi"]))
    lens = [int(round(math.exp(rng.uniform(math.log(case["lo"]), math.log(case["hi"]))))) for _ in range(case["seqs"])]
    lens[0] = case["hi"]
    if case["op"] == "append" and case["rows"]:
        lens = [n + case["rows"] for n in lens]
    new = [min(case["rows"] or n, n) if case["op"] == "prefill" else case["rows"] or n for n in lens]
    return lens, new


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    nq, nkv, hd, ps, op = case["nq"], case["nkv"], case["hd"], case["page"], case["op"]
    dt = DTYPES[case["dtype"]]
    lens, new = lengths(case)
    need = [-(-n // ps) for n in lens]
    pages = sum(need) + 3
    shape = (pages, nkv, ps, hd) if case["layout"] == "hnd" else (pages, ps, nkv, hd)
    pools = [torch.randn(shape, generator=g, dtype=dt, device=dev) for _ in range(2)]
    k, v = (p if case["layout"] == "hnd" else p.transpose(1, 2) for p in pools)
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32)
    width = max(need)
    starts = torch.tensor([0] + need[:-1], device=dev).cumsum(0)
    at = starts[:, None] + torch.arange(width, device=dev)[None, :]
    used = torch.arange(width, device=dev)[None, :] < torch.tensor(need, device=dev)[:, None]
    table = torch.where(used, order[at.clamp(max=pages - 1)], -1).to(torch.int32)
    rows = sum(new)
    s = {"op": op, "k": k, "v": v, "table": table, "max_len": max(lens), "nq": nq, "window": case.get("window", 0),
         "sinks": case.get("sinks", 0), "lens": torch.tensor(lens, dtype=torch.int32, device=dev)}
    if op == "append":
        qkv = torch.randn((rows, nq + 2 * nkv, hd), generator=g, dtype=dt, device=dev)
        s["q"], s["kn"], s["vn"] = qkv[:, :nq], qkv[:, nq:nq + nkv], qkv[:, nq + nkv:]
        seq = torch.tensor([i for i, n in enumerate(new) for _ in range(n)], dtype=torch.int32, device=dev)
        row = torch.cat([torch.arange(n, dtype=torch.int32) for n in new]).to(dev)
        base = torch.tensor([a - b for a, b in zip(lens, new)], dtype=torch.int32, device=dev)[seq.long()]
        s["seq"], s["slot"] = seq, base + row
        # drafts of a tree share depths: the position runs behind the slot
        s["pos"] = s["slot"] if case["rows"] in (0, 1) else base + torch.div(row + 1, 2, rounding_mode="floor")
        f = 1e6 ** (-torch.arange(hd // 2, dtype=torch.float64, device=dev) * 2 / hd)
        a = torch.arange(max(lens) + 16, dtype=torch.float64, device=dev)[:, None] * f[None, :]
        s["rope"], s["half"] = torch.stack([a.cos(), a.sin()], -1).float().contiguous(), case["half"]
    elif op == "decode":
        r = case["rows"]
        s["q"] = torch.randn((case["seqs"], r, nq, hd), generator=g, dtype=dt, device=dev)
        s["mask"] = None
        if r > 1:  # random trees: row i hangs below one of the rows before it
            par = [None] + [torch.randint(0, i, (case["seqs"],), generator=g, device=dev) for i in range(1, r)]
            anc = torch.ones((case["seqs"], r), dtype=torch.int64, device=dev)
            for i in range(1, r):
                anc[:, i] = anc.gather(1, par[i][:, None])[:, 0] | (1 << i)
            s["mask"] = anc.to(torch.int32)
    else:
        s["q"] = torch.randn((rows, nq, hd), generator=g, dtype=dt, device=dev)
        s["q_start"] = torch.tensor([0] + new, device=dev).cumsum(0).to(torch.int32)
        s["max_new"] = max(new)
    if own:
        from instantllm_b200.paged import PagedLayer

        s["layer"] = PagedLayer(k, v, table)
    return s


def run(state):
    s = state
    if own:
        kv = s["layer"]
        if s["op"] == "append":
            q = kv.append(s["q"], s["kn"], s["vn"], s["seq"], s["slot"], s["pos"], s["rope"], interleaved=not s["half"])
            return {"q": q, "k": s["k"], "v": s["v"]}
        if s["op"] == "decode":
            out, lse = kv.decode(s["q"], s["lens"], mask=s["mask"], window=s["window"], sinks=s["sinks"], return_lse=True)
            return {"out": out, "lse": lse}
        return {"out": kv.prefill(s["q"], s["q_start"], s["lens"], window=s["window"], sinks=s["sinks"])}
    return {"append": plain_append, "decode": plain_decode, "prefill": plain_prefill}[s["op"]](s)


def rotate(x, cs, half):
    x = x.float()
    c, sn = cs[:, None, :, 0], cs[:, None, :, 1]
    if half:
        a, b = x.chunk(2, -1)
        return torch.cat([a * c - b * sn, b * c + a * sn], -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * c - b * sn, b * c + a * sn], -1).flatten(-2)


def plain_append(s):
    k, v = s["k"], s["v"]
    ps = k.shape[2]
    cs = s["rope"][s["pos"].long()]
    slot = s["slot"].long()
    page = s["table"][s["seq"].long(), slot // ps].long()
    k[page, :, slot % ps] = rotate(s["kn"], cs, s["half"]).to(k.dtype)
    v[page, :, slot % ps] = s["vn"].to(v.dtype)
    return {"q": rotate(s["q"], cs, s["half"]).to(k.dtype), "k": k, "v": v}


def gathered(s):
    """The requests' keys and values in slot order, [requests][heads][slots][hd] in 32 bits, zero past each request's end."""
    n, ps = s["table"].shape[0], s["k"].shape[2]
    pages = s["table"][:, :-(-s["max_len"] // ps)].clamp(min=0).long()
    inside = torch.arange(pages.shape[1] * ps, device=pages.device)[None, :] < s["lens"][:, None]
    kv = [p[pages].float().transpose(1, 2).flatten(2, 3) for p in (s["k"], s["v"])]
    return [x.masked_fill_(~inside[:, None, :, None], 0.0) for x in kv]


def softmax_product(scores, hidden, v):
    """softmax over what is not hidden, times v, and the log of its sum; rows without any are zero."""
    scores.masked_fill_(hidden, -math.inf)
    m = scores.amax(-1, keepdim=True)
    scores.sub_(m.masked_fill(m == -math.inf, 0.0)).exp_()
    total = scores.sum(-1, keepdim=True)
    lse = (m + total.log())[..., 0]
    out = scores.flatten(2, -2) @ v
    return out.view(scores.shape[:-1] + v.shape[-1:]) / total.masked_fill(total == 0, 1.0), lse


def plain_decode(s):
    q, lens = s["q"], s["lens"].long()
    n, r, nq, hd = q.shape
    k, v = gathered(s)
    nkv, length = k.shape[1], k.shape[2]
    x = q.float().view(n, r, nkv, nq // nkv, hd).transpose(1, 2)  # [n][nkv][r][g][hd]
    scores = (x.flatten(2, 3) @ k.transpose(2, 3)).mul_(hd ** -0.5).view(n, nkv, r, nq // nkv, length)
    j = torch.arange(length, device=q.device)
    base = (lens - r)[:, None, None]
    rows = torch.arange(r, device=q.device)
    anc = s["mask"] if s["mask"] is not None else ((2 << rows) - 1)[None, :].expand(n, r)
    bits = (anc[:, :, None].long() >> rows) & 1  # [n][r][r]
    depth = bits.sum(-1) - 1
    draft = (j[None, None, :] - base).clamp(0, r - 1).expand(n, r, length)
    old = j < base
    seen = old | ((bits.gather(2, draft) > 0) & (j < lens[:, None, None]))
    if s["window"]:
        place = torch.where(old, j, base + depth[:, None, :].expand(n, r, r).gather(2, draft))
        seen &= (base + depth[:, :, None] - place < s["window"]) | (place < s["sinks"])
    out, lse = softmax_product(scores, ~seen[:, None, :, None, :], v)
    return {"out": out.transpose(1, 2).reshape(n, r, nq, hd).to(q.dtype), "lse": lse.transpose(1, 2).reshape(n, r, nq)}


def plain_prefill(s):
    q, start, lens = s["q"], s["q_start"].long(), s["lens"].long()
    rows, nq, hd = q.shape
    n, most = lens.shape[0], s["max_new"]
    k, v = gathered(s)
    nkv, length = k.shape[1], k.shape[2]
    i = torch.arange(most, device=q.device)
    new = start[1:] - start[:-1]
    padded = q.float()[(start[:-1, None] + i).clamp(max=rows - 1)].view(n, most, nkv, nq // nkv, hd).transpose(1, 2)
    scores = (padded.flatten(2, 3) @ k.transpose(2, 3)).mul_(hd ** -0.5).view(n, nkv, most, nq // nkv, length)
    place = ((lens - new)[:, None] + i)[:, :, None]
    j = torch.arange(length, device=q.device)
    hidden = j > place
    if s["window"]:
        hidden |= (place - j >= s["window"]) & (j >= s["sinks"])
    out, _ = softmax_product(scores, hidden[:, None, :, None, :], v)
    at = torch.arange(rows, device=q.device)
    seq = torch.bucketize(at, start[1:], right=True)
    return {"out": out.transpose(1, 2).reshape(n, most, nq, hd)[seq, at - start[seq]].to(q.dtype)}


def exact(case, seed):
    """The operator's definition in 64 bits, one request and one head at a time."""
    s = prepare(case, seed)
    lens, new = lengths(case)
    ps, hd = s["k"].shape[2], case["hd"]
    group = case["nq"] // case["nkv"]
    if case["op"] == "append":
        z = torch.view_as_complex(s["rope"].double()[s["pos"].long()])  # [rows][hd / 2]

        def turned(x):
            x = x.double()
            if case["half"]:
                y = torch.complex(x[..., :hd // 2].contiguous(), x[..., hd // 2:].contiguous()) * z[:, None]
                return torch.cat([y.real, y.imag], -1)
            return torch.view_as_real(torch.view_as_complex(x.reshape(*x.shape[:-1], -1, 2).contiguous()) * z[:, None]).flatten(-2)

        kv = []
        for pool, x in ((s["k"], turned(s["kn"])), (s["v"], s["vn"].double())):
            whole = pool.double()
            flat = whole.transpose(1, 2).reshape(-1, case["nkv"], hd)
            flat[s["table"].long()[s["seq"].long(), s["slot"].long() // ps] * ps + s["slot"].long() % ps] = x
            kv.append(flat.view(-1, ps, case["nkv"], hd).transpose(1, 2))
        return {"q": turned(s["q"]), "k": kv[0], "v": kv[1]}
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=s["q"].device)
    lse = torch.full(s["q"].shape[:-1], -math.inf, dtype=torch.float64, device=out.device)
    first = 0
    for i, (n, m) in enumerate(zip(lens, new)):
        pages = s["table"][i, :-(-n // ps)].long()
        j = torch.arange(n, device=out.device)
        if case["op"] == "decode":
            q, o, le = s["q"][i], out[i], lse[i]
            seen = torch.zeros((m, n), dtype=torch.bool, device=out.device)
            place = j.clone()
            masks = s["mask"][i].tolist() if s["mask"] is not None else [(2 << r) - 1 for r in range(m)]
            for r, bits in enumerate(masks):
                place[n - m + r] = n - m + bin(bits).count("1") - 1
                seen[r, :n - m] = True
                for t in range(m):
                    seen[r, n - m + t] = bool(bits >> t & 1)
            at = place[n - m:]
        else:
            q, o, le = s["q"][first:first + m], out[first:first + m], lse[first:first + m]
            place, at = j, j[n - m:]
            seen = j[None, :] <= at[:, None]
        first += m
        if case["window"]:
            seen &= (at[:, None] - place[None, :] < case["window"]) | (place[None, :] < case["sinks"])
        for h in range(case["nq"]):
            kk, vv = (p[pages, h // group].reshape(-1, hd)[:n].double() for p in (s["k"], s["v"]))
            sc = torch.where(seen, q[:, h].double() @ kk.T / math.sqrt(hd), torch.tensor(-math.inf, dtype=torch.float64, device=out.device))
            le[:, h] = torch.logsumexp(sc, -1)
            o[:, h] = torch.nan_to_num(torch.softmax(sc, -1)) @ vv
    return {"out": out, "lse": lse} if case["op"] == "decode" else {"out": out}


def work(case):
    lens, new = lengths(case)
    nq, nkv, hd = case["nq"], case["nkv"], case["hd"]
    rows = sum(new)
    if case["op"] == "append":
        # each row in and out in 16 bits, its rotation, its three indexes and its page
        return {"bytes": rows * (2 * 2 * (nq + 2 * nkv) * hd + 4 * hd + 16), "flops": 3 * rows * (nq + nkv) * hd}
    w, sinks = case["window"], case["sinks"]
    slots = pairs = 0
    for n, m in zip(lens, new):
        first = n - m
        if case["op"] == "decode":
            # the cached slots some row sees; a row of a tree of m rows sees itself and its ancestors, at most m
            old = first if not w else min(first, sinks + max(0, min(w, first - sinks)))
            slots += old + m
            pairs += m * (old + 1)
        else:
            slots += n if not w else min(n, sinks + max(0, min(n - sinks, m + w - 1)))
            # sum over positions p = first .. n - 1 of what p sees
            pairs += sum(p + 1 if not w else min(p + 1, w + max(0, min(sinks, p + 1 - w))) for p in range(first, n))
    return {"bytes": 2 * (2 * slots * nkv * hd + 2 * rows * nq * hd) + (4 * rows * nq if case["op"] == "decode" else 0),
            "flops": 4 * pairs * nq * hd}
