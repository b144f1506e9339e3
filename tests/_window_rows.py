"""Attention within a sliding window in float64, with a bound of what each query row's own rows allow."""

from __future__ import annotations

import numpy as np
import torch

from _rows import DECODE, Softmax


def code_rows(cache: np.ndarray, table: np.ndarray, b: int, rows: int, h: int):
    """float64 codes [rows, D] and row scales [rows] of KV head h of request b, and which rows lie in the cache."""
    nb, bs, _, _ = cache.shape
    t = np.arange(rows)
    blk = table[b, t // bs].astype(np.int64)
    there = (blk >= 0) & (blk < nb)
    raw = np.ascontiguousarray(cache[np.where(there, blk, 0), t % bs, h])
    return DECODE[raw[:, :-4]], np.ascontiguousarray(raw[:, -4:]).view(np.float32)[:, 0].astype(np.float64), there


def window_by_row(q, kc, vc, table, lens, qlens, window, sinks, scale, dtype):
    """(out, bound) float64 [T, Hq, Dv]; numpy arrays in, what some row sees has to be finite.

    P = p s 2^k (s: the V row's scale) has 11 significant bits (2^-11 of p |V|), or 2^-25 absolutely where it is
    subnormal.  k puts the largest p |s| of the rows that this query row sees at 2^6 at least, so that is 2^-31
    max(p |s|) |code|.  What a query row does not see is in no term."""
    hq, hkv, group = q.shape[1], kc.shape[2], q.shape[1] // kc.shape[2]
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    out = np.zeros((q.shape[0], hq, vc.shape[3] - 4))
    bound = np.zeros_like(out)
    row = 0
    for b, (size, n) in enumerate(zip(lens, qlens)):
        at, t = size - n + np.arange(n)[:, None], np.arange(size)[None, :]
        inside = (t <= at) & ((t > at - window) | (t < sinks))
        for h in range(hkv):
            k, ks, there = code_rows(kc, table, b, size, h)
            v, vs, _ = code_rows(vc, table, b, size, h)
            sees = inside & there
            some = sees.any(axis=0)
            key = np.where(some[:, None], k, 0.0) * np.where(some, ks, 0.0)[:, None]
            v, vs = np.where(some[:, None], v, 0.0), np.where(some, vs, 0.0)
            value = v * vs[:, None]
            for head in range(h * group, (h + 1) * group):
                sm = Softmax(q[row:row + n, head], key, sees, scale)
                y = sm.p @ value
                most = (sm.p * np.abs(vs)).max(axis=1, initial=0.0)[:, None]
                out[row:row + n, head] = y
                bound[row:row + n, head] = half * np.abs(y) + (2.0 ** -11 + sm.rel) * (sm.p @ np.abs(value)) + tiny + \
                    2.0 ** -31 * most * (sees.astype(np.float64) @ np.abs(v))
        row += n
    return out, bound
