"""Plain float64 forms of the operators that look at the HiF8 cache row by row,
and the error bounds that their kernels are held to."""

from __future__ import annotations

import math

import numpy as np
import torch

from oracle import hif8_oracle as o

DECODE = np.asarray(o.DECODE, dtype=np.float64)


def decoded_rows(cache: np.ndarray, table: np.ndarray, b: int, rows: int, h: int) -> tuple[np.ndarray, np.ndarray]:
    """float64 rows [rows, D] of KV head h of request b, and which of them lie in a block of the cache."""
    nb, bs, _, width = cache.shape
    out = np.zeros((rows, width - 4))
    there = np.zeros(rows, dtype=bool)
    for t in range(rows):
        blk = int(table[b, t // bs])
        if not 0 <= blk < nb:
            continue
        raw = cache[blk, t % bs, h]
        with np.errstate(invalid="ignore"):
            out[t] = DECODE[raw[:-4]] * np.float64(raw[-4:].copy().view(np.float32)[0])
        there[t] = True
    return out, there


class Softmax:
    """One (request, KV head): weights of its query rows and how exactly float32 arithmetic keeps them.

    A logit is a sum of D products of 16-bit values accumulated in float32, times
    two float32 factors: off by at most delta = (D + 8) 2^-24 sum|q k| scale.  A
    weight is then off by at most a factor 1 +- 2 (delta_max + n 2^-24) and a
    few units of exp2, which 2^-20 covers."""

    def __init__(self, q: np.ndarray, key: np.ndarray, sees: np.ndarray, scale: float):
        n, d = key.shape
        x = np.where(sees, 0.0, -np.inf)
        used = sees.any(axis=0)
        with np.errstate(invalid="ignore", over="ignore"):
            x[:, used] = np.where(sees[:, used], (q @ key[used].T) * scale, -np.inf)
            size = (np.abs(q) @ np.abs(key[used]).T) * abs(scale)
        top = x.max(axis=1, initial=-np.inf, keepdims=True)
        top = np.where(np.isfinite(top), top, 0.0)
        with np.errstate(invalid="ignore"):
            p = np.exp(x - top)
            total = p.sum(axis=1, keepdims=True)
            self.p = np.where(total > 0, p / np.where(total > 0, total, 1.0), np.where(np.isnan(total), np.nan, 0.0))
        size = np.where(sees[:, used], size, 0.0)
        size = size[np.isfinite(size)]
        delta = (d + 8) * 2.0 ** -24 * (size.max() if size.size else 0.0)
        self.rel = 2 * (delta + n * 2.0 ** -24) + 2.0 ** -20


def attention_with_bound(sm: Softmax, value: np.ndarray, dtype: torch.dtype) -> tuple[np.ndarray, np.ndarray]:
    """(out, how far a kernel may be off).  The weights go through the product with
    V in 16 bits with 11 significant ones (2^-11 each, 2^-25 absolute against the
    largest where they are subnormal), and the output is rounded once."""
    used = (sm.p != 0).any(axis=0)
    p, v = sm.p[:, used], value[used]
    good = np.isfinite(v).all(axis=1)
    with np.errstate(invalid="ignore"):
        out = p[:, good] @ v[good]
        mag = p[:, good] @ np.abs(v[good])
        for t in np.flatnonzero(~good):      # a row that does not see it has no part in it
            out += np.where(p[:, t, None] != 0, p[:, t, None] * v[t], 0.0)
    top = np.abs(v[good]).max(initial=0.0)
    half = torch.finfo(dtype).eps / 2
    tiny = torch.finfo(dtype).smallest_normal * half
    # The rounding to the output's type takes what lies half a step past its largest value to infinity.
    most = torch.finfo(dtype).max * (1 + half / 2)
    out = np.where(np.abs(out) >= most, np.copysign(np.inf, out), out)
    bound_of = np.where(np.isfinite(out), np.abs(out), 0.0)
    return out, half * bound_of + (2.0 ** -11 + sm.rel) * mag + len(v) * 2.0 ** -25 * top + tiny


def tree_reference(q, kc, vc, table, ctx, qlens, mask, scale, dtype):
    """(out, bound) float64 [T, Hq, Dv] of tree attention."""
    total, hq, _ = q.shape
    hkv = kc.shape[2]
    out = np.zeros((total, hq, vc.shape[3] - 4))
    bound = np.zeros_like(out)
    row = 0
    for b, (c, n) in enumerate(zip(ctx, qlens)):
        for h in range(hkv):
            key, there = decoded_rows(kc, table, b, c + n, h)
            value, _ = decoded_rows(vc, table, b, c + n, h)
            sees = np.concatenate([np.ones((n, c), bool), mask[row:row + n, :n].astype(bool)], axis=1) & there
            for g in range(hq // hkv):
                sm = Softmax(q[row:row + n, h * (hq // hkv) + g], key, sees, scale)
                y, e = attention_with_bound(sm, value, dtype)
                out[row:row + n, h * (hq // hkv) + g], bound[row:row + n, h * (hq // hkv) + g] = y, e
        row += n
    return out, bound


def weights_reference(q, kc, table, lens, qlens, scale, causal=True):
    """(sums, bound) float64 [B, Hkv, max(lens)]: softmax weight of every cached row over rows and heads."""
    hq, hkv = q.shape[1], kc.shape[2]
    sums = np.zeros((len(lens), hkv, max(max(lens), 1)))
    bound = np.zeros_like(sums)
    row = 0
    for b, (size, n) in enumerate(zip(lens, qlens)):
        i, t = np.arange(n)[:, None], np.arange(size)[None, :]
        sees = (t <= size - n + i) if causal else np.ones((n, size), bool)
        for h in range(hkv):
            key, there = decoded_rows(kc, table, b, size, h)
            for g in range(hq // hkv):
                sm = Softmax(q[row:row + n, h * (hq // hkv) + g], key, sees & there, scale)
                total = sm.p.sum(axis=0)
                sums[b, h, :size] += total
                bound[b, h, :size] += (sm.rel + 2.0 ** -24 * n * (hq // hkv)) * total
        row += n
    return sums, bound


def evict_reference(kc, vc, table, lens, weights, keep, positions=None, sinks=0, protect_from=None):
    """Eviction on numpy copies: (key cache, value cache, weights, positions, new lengths)."""
    kc, vc, weights = kc.copy(), vc.copy(), weights.copy()
    positions = None if positions is None else positions.copy()
    nb, bs = kc.shape[:2]
    new = []

    def slot(b, t):
        blk = int(table[b, t // bs])
        return (blk, t % bs) if 0 <= blk < nb else None

    for b, size in enumerate(lens):
        n = min(size, keep[b])
        new.append(n)
        for h in range(kc.shape[2]):
            at = positions[b, h, :size] if positions is not None else np.arange(size)
            safe = (at < sinks) | ((at >= protect_from[b]) if protect_from is not None else False)
            w = weights[b, h, :size].astype(np.float64)
            order = sorted(range(size), key=lambda t: (0 if safe[t] else 2 if math.isnan(w[t]) else 1,
                                                       0.0 if safe[t] or math.isnan(w[t]) else -w[t], t))
            kept = set(order[:n])
            holes = [t for t in range(n) if t not in kept]
            movers = [t for t in range(n, size) if t in kept]
            assert len(holes) == len(movers)
            for to, frm in zip(holes, movers):
                d, s = slot(b, to), slot(b, frm)
                if d is not None and s is not None:
                    kc[d][h], vc[d][h] = kc[s][h], vc[s][h]
                weights[b, h, to] = weights[b, h, frm]
                if positions is not None:
                    positions[b, h, to] = positions[b, h, frm]
            if n < size:
                weights[b, h, n:size] = 0.0
    return kc, vc, weights, positions, new


def ancestors(parents: list[int]) -> np.ndarray:
    """Mask [n, n] of a tree given by parents (-1: the context): a node sees its ancestors and itself."""
    n = len(parents)
    mask = np.zeros((n, n), dtype=bool)
    for i, parent in enumerate(parents):
        if parent >= 0:
            mask[i] = mask[parent]
        mask[i, i] = True
    return mask
