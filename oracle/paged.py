"""The paged-cache operators from their definitions, in float64 (tests only): rotation, visibility, attention of one row."""
from __future__ import annotations

import numpy as np


def rotate(x: np.ndarray, cs: np.ndarray, interleaved: bool) -> np.ndarray:
    """x [heads][head_dim] turned by cs [rot_dim / 2][2] (cos, sin)."""
    y = np.array(x, dtype=np.float64)
    r = cs.shape[0]
    for i in range(r):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + r)
        c, s = float(cs[i, 0]), float(cs[i, 1])
        y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    return y


def slots(pool: np.ndarray, table_row, n: int) -> np.ndarray:
    """[heads][n][head_dim] of a request from its pages; pool [pages][heads][page_size][head_dim]."""
    ps = pool.shape[2]
    j = np.arange(n)
    return np.asarray(pool[np.asarray(table_row)[j // ps], :, j % ps].swapaxes(0, 1), dtype=np.float64)


def sees_prompt(length: int, new: int, window: int, sinks: int) -> np.ndarray:
    """bool [new][length]: row r is the slot length - new + r."""
    out = np.zeros((new, length), dtype=bool)
    for r in range(new):
        p = length - new + r
        for j in range(p + 1):
            out[r, j] = window == 0 or p - j < window or j < sinks
    return out


def sees_tree(length: int, masks, window: int, sinks: int) -> np.ndarray:
    """bool [rows][length]: row r sees the slots before the rows, and new slot j where bit j of masks[r] is set."""
    rows = len(masks)
    base = length - rows
    place = list(range(max(0, base))) + [base + bin(m).count("1") - 1 for m in masks]
    out = np.zeros((rows, length), dtype=bool)
    for r in range(rows):
        if base + r < 0:
            continue
        p = base + bin(masks[r]).count("1") - 1
        for j in range(length):
            if j >= base and not masks[r] >> (j - base) & 1:
                continue
            at = place[j] if base >= 0 else place[j - base]
            out[r, j] = window == 0 or p - at < window or at < sinks
    return out


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, seen: np.ndarray, scale: float):
    """(out [head_dim], lse, sum of p |v| / l, largest sum of |q k| scale) of one row and head over k, v [slots][head_dim]."""
    hd = q.shape[0]
    if not seen.any():
        return np.zeros(hd), -np.inf, np.zeros(hd), 0.0
    k, v = k[seen], v[seen]
    s = k @ q * scale
    m = s.max()
    p = np.exp(s - m)
    l = p.sum()
    return p @ v / l, m + np.log(l), p @ np.abs(v) / l, float((np.abs(k) @ np.abs(q)).max() * scale)
