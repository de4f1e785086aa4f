"""The model over a paged key-value cache, for as many requests at once as the cache holds: prompts of a batch in one go
(`prefill`), one token each (`decode`), or a draft tree each (`verify`), with greedy acceptance as in the verify pass.

The attention and the cache are the paged operators (instantllm_b200.paged); the projections are plain library matrix
products on fp16 weights, dequantised once. VerifyEngine's persistent kernel serves up to four requests with less latency;
this serves a batch, where the projections' weights are read once for all of it. The reference serves one request
(Engine.generate, Engine.swift:922-1038; prefill :588-601; accept and commit, Shaders.swift:254-365).

    python -m instantllm_b200.paged_engine --requests 64 --prompt 256 --new 64
"""
from __future__ import annotations

from typing import Callable, Optional

import numpy as np
import torch
import torch.nn.functional as F

from ._lib import VpError
from .paged import PagedKV, ancestor_masks, rope_table
from .synth import FFN, HIDDEN, STOP_IDS

N_Q, N_KV, HEAD = 14, 2, 64
EPS = 1e-6


def _dense(m: dict, device) -> torch.Tensor:
    """A matrix of the standard layouts (include/vpass.h) in fp16."""
    if m["fmt"] in ("f16", "f32"):
        return torch.from_numpy(np.asarray(m["w"])).to(device).half()
    codes = torch.from_numpy(np.array(m["codes"])).to(device)
    scales = torch.from_numpy(np.asarray(m["scales"]).astype(np.float32)).to(device)
    if m["fmt"] == "q4":
        q = torch.stack([codes & 15, codes >> 4], -1).flatten(1).float().unflatten(1, (-1, 64))
        return (q * scales[..., :1] + scales[..., 1:]).flatten(1).half()
    q = codes.float().unflatten(1, (scales.shape[1], -1))
    return (q * scales[..., None]).flatten(1).half()


class PagedEngine:
    def __init__(self, weights: dict, n_pages: int = 1024, page_size: int = 64, max_seqs: int = 64, max_len: int = 4096,
                 window: int = 0, sinks: int = 0, device: int = 0):
        self.device = torch.device("cuda", device)
        self.vocab, self.window, self.sinks = weights["vocab"], window, sinks
        dev = self.device

        def vec(x):
            return torch.from_numpy(np.asarray(x, dtype=np.float32)).to(dev)

        self.embed = _dense(weights["embed"], dev)
        self.norm = vec(weights["final_norm"])
        self.layers = [{"wqkv": _dense(L["wqkv"], dev), "bqkv": vec(L["bqkv"]).half(), "wo": _dense(L["wo"], dev),
                        "wgu": _dense(L["wgu"], dev), "wd": _dense(L["wd"], dev), "ln1": vec(L["ln1"]), "ln2": vec(L["ln2"])}
                       for L in weights["layers"]]
        self.kv = PagedKV(len(self.layers), n_pages, page_size, max_seqs, max_len, N_KV, HEAD, torch.float16, device)
        self.rope = rope_table(max_len + 16, HEAD, device=dev)
        self.lens = [0] * max_seqs  # committed slots of each request

    def _i32(self, x) -> torch.Tensor:
        return torch.as_tensor(np.asarray(x, dtype=np.int32)).to(self.device)

    def _rows(self, tokens, seq, slot, pos, attend: Callable) -> torch.Tensor:
        """Rows through the layers; attend(layer of the cache, rotated queries) -> attention output. Residual rows fp32."""
        tokens, seq, slot, pos = (self._i32(v) for v in (tokens, seq, slot, pos))
        x = self.embed[tokens.long()].float()
        for L, kv in zip(self.layers, self.kv.layers):
            qkv = F.linear(F.rms_norm(x, (HIDDEN,), L["ln1"], EPS).half(), L["wqkv"], L["bqkv"]).view(-1, N_Q + 2 * N_KV, HEAD)
            q = kv.append(qkv[:, :N_Q], qkv[:, N_Q:N_Q + N_KV], qkv[:, N_Q + N_KV:], seq, slot, pos, self.rope)
            x = x + F.linear(attend(kv, q).reshape(-1, HIDDEN), L["wo"])
            gu = F.linear(F.rms_norm(x, (HIDDEN,), L["ln2"], EPS).half(), L["wgu"])
            x = x + F.linear(F.silu(gu[:, :FFN]) * gu[:, FFN:], L["wd"])
        return x

    def _logits(self, x: torch.Tensor) -> torch.Tensor:
        return F.linear(F.rms_norm(x, (HIDDEN,), self.norm, EPS).half(), self.embed).float()

    def prefill(self, prompts: dict) -> torch.Tensor:
        """{request: token ids} appended to the requests (their first tokens, or the next chunk of them) in one batch;
        logits fp32 [requests][vocab] of each one's last token."""
        seqs = list(prompts)
        n = [len(prompts[s]) for s in seqs]
        if min(n) < 1:
            raise ValueError("a prompt has at least one token")
        self.kv.reserve_all({s: self.lens[s] + k for s, k in zip(seqs, n)})
        slot = np.concatenate([self.lens[s] + np.arange(k) for s, k in zip(seqs, n)])
        starts = np.concatenate([[0], np.cumsum(n)])
        ids, lens = self._i32(seqs), self._i32([self.lens[s] + k for s, k in zip(seqs, n)])
        q_start = self._i32(starts)
        x = self._rows(np.concatenate([prompts[s] for s in seqs]), np.repeat(seqs, n), slot, slot,
                       lambda kv, q: kv.prefill(q, q_start, lens, seqs=ids, window=self.window, sinks=self.sinks))
        for s, k in zip(seqs, n):
            self.lens[s] += k
        return self._logits(x[self._i32(starts[1:] - 1).long()])

    def decode(self, tokens: dict) -> torch.Tensor:
        """{request: its last token}: one step of every request; logits fp32 [requests][vocab]."""
        return self.verify({s: {"n": 1, "parent": [-1], "depth": [0], "tok": [0]} for s in tokens}, tokens, commit=False, keep=1)[0][:, 0]

    def verify(self, trees: dict, roots: dict, commit: bool = True, keep: int = 0):
        """{request: draft tree} (dicts as in synth.seeded_tree; row 0 is the root, the request's last token): logits fp32
        [requests][rows][vocab] of a pass over all trees, rows of the largest, and with commit the tokens that each
        request commits: the longest path whose drafts equal their parents' argmax, then one more. The accepted rows'
        keys and values move up behind the root (the commit's compaction). keep: rows that stay without commit."""
        seqs = list(trees)
        n = np.array([trees[s]["n"] for s in seqs])
        rows = int(n.max())
        self.kv.reserve_all({s: self.lens[s] + k for s, k in zip(seqs, n.tolist())})
        base, pad = np.array([self.lens[s] for s in seqs]), rows - n
        # All requests of a call have as many rows, the last slots of each: a smaller tree stands behind padding rows, which are
        # its last old slots (not stored again), so that it takes no slot beyond its own.
        at = np.arange(rows) - pad[:, None]  # row of the tree, negative for padding
        real, tree_row = at >= 0, np.maximum(at, 0)
        tok = np.array([[roots[s]] + [trees[s]["tok"][r] if 0 < r < trees[s]["n"] else 0 for r in range(1, rows)] for s in seqs])
        depth = np.array([[trees[s]["depth"][r] if r < trees[s]["n"] else 0 for r in range(rows)] for s in seqs])
        tok, depth = np.take_along_axis(tok, tree_row, 1), np.take_along_axis(depth, tree_row, 1)
        anc = ancestor_masks([trees[s] for s in seqs]).numpy()[:, :rows].astype(np.int64)
        below = (1 << pad)[:, None] - 1  # the old slots among the call's rows
        anc = np.where(real, np.take_along_axis(anc, tree_row, 1) << pad[:, None] | below, (2 << np.arange(rows)) - 1)
        masks, ids, lens = self._i32(anc), self._i32(seqs), self._i32(base + n)
        x = self._rows(tok.ravel(), np.where(real, np.array(seqs)[:, None], -1).ravel(), (base[:, None] + tree_row).ravel(),
                       (base[:, None] + depth).ravel(),
                       lambda kv, q: kv.decode(q.view(len(seqs), rows, N_Q, HEAD), lens, mask=masks, seqs=ids, window=self.window,
                                               sinks=self.sinks))
        if pad.any():  # back in the trees' order; rows past a tree are its root again
            order = np.arange(len(seqs))[:, None] * rows + pad[:, None] + np.where(np.arange(rows) < n[:, None], np.arange(rows), 0)
            x = x[self._i32(order.ravel()).long()]
        logits = self._logits(x).view(len(seqs), rows, -1)
        if not commit:
            for s in seqs:
                self.lens[s] += keep
            return logits, None
        best = logits.argmax(-1).cpu().numpy()
        out, src, dst = {}, [], []
        for i, s in enumerate(seqs):
            t, path = trees[s], [0]
            while True:
                child = [c for c in range(1, t["n"]) if t["parent"][c] == path[-1] and t["tok"][c] == best[i, path[-1]]]
                if not child:
                    break
                path.append(child[0])
            out[s] = [int(best[i, r]) for r in path]
            for d, r in enumerate(path):
                if r != d:
                    src.append((s, self.lens[s] + r))
                    dst.append((s, self.lens[s] + d))
            self.lens[s] += len(path)
        self._move(src, dst)
        return logits, out

    def _move(self, src, dst) -> None:
        if not src:
            return
        ps = self.kv.page_size
        (a, i), (b, j) = (self._i32(list(zip(*x))).long() for x in (src, dst))
        pa, pb = self.kv.table[a, i // ps].long(), self.kv.table[b, j // ps].long()
        for pool in (self.kv.k, self.kv.v):
            pool[:, pb, :, j % ps] = pool[:, pa, :, i % ps]  # the right side is a copy: a slot may be read and written

    def release(self, seq: int) -> None:
        self.kv.release(seq)
        self.lens[seq] = 0

    def generate(self, prompts: list, max_new: int, tree_fn: Optional[Callable] = None, eos=STOP_IDS) -> list:
        """Greedy token lists of all prompts (up to max_new each, a stop token included). tree_fn(request, committed tokens) ->
        draft tree whose root is the last of them; without it, one token a step. Requests 0 .. len(prompts) - 1 must be free,
        and are again afterwards, also when it fails."""
        if max_new < 1:
            return [[] for _ in prompts]
        held = [s for s, n in enumerate(self.lens[:len(prompts)]) if n]
        if held:
            raise VpError(f"requests {held} hold a context: release them first")
        out = {s: [] for s in range(len(prompts))}
        live = dict(enumerate(prompts))
        try:
            first = self.prefill(live).argmax(-1).tolist() if live else []
            new = {s: [t] for s, t in zip(live, first)}
            while live:
                for s in list(new):
                    for t in new[s]:
                        out[s].append(t)
                        if t in eos or len(out[s]) == max_new:
                            self.release(s)
                            del live[s]
                            break
                if not live:
                    break
                roots = {s: out[s][-1] for s in live}
                if tree_fn is None:
                    new = {s: [t] for s, t in zip(live, self.decode(roots).argmax(-1).tolist())}
                else:
                    new = self.verify({s: tree_fn(s, list(prompts[s]) + out[s]) for s in live}, roots)[1]
            self.kv.check()
        finally:  # what a step that failed leaves
            for s in live:
                if s < len(self.lens):
                    self.release(s)
        return list(out.values())


def main() -> None:
    import argparse
    import time

    from . import synth

    ap = argparse.ArgumentParser(description="greedy decoding of many requests over a paged cache, on seeded synthetic weights")
    ap.add_argument("--requests", type=int, default=64)
    ap.add_argument("--prompt", type=int, default=256)
    ap.add_argument("--new", type=int, default=64)
    ap.add_argument("--format", default="q4", choices=("q4", "q8", "q8g32", "f16"))
    a = ap.parse_args()
    length = a.prompt + a.new + 16
    eng = PagedEngine(synth.make_weights(a.format), n_pages=a.requests * (-(-length // 64)), max_seqs=a.requests, max_len=length)
    prompts = [synth.make_prompt(a.prompt, seed=i).tolist() for i in range(a.requests)]
    eng.generate(prompts, 4)
    torch.cuda.synchronize()
    t = time.perf_counter()
    out = eng.generate(prompts, a.new)
    torch.cuda.synchronize()
    t = time.perf_counter() - t
    n = sum(map(len, out))
    print(f"{a.requests} requests of {a.prompt} + {a.new} tokens: {n} tokens in {t * 1e3:.1f} ms, {n / t:,.0f} tok/s")


if __name__ == "__main__":
    main()
