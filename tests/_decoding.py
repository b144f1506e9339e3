"""Plain float64 forms of the operators around a decoding step: attention within a
sliding window, verification of drafts, pages taken and given back."""

from __future__ import annotations

import numpy as np

from _rows import DECODE, Softmax, attention_with_bound


def cached_rows(cache: np.ndarray, table: np.ndarray, b: int, rows: int, h: int):
    """float64 rows [rows, D] of KV head h of request b, and which of them lie in a block of the cache."""
    nb, bs, _, width = cache.shape
    t = np.arange(rows)
    blk = table[b, t // bs].astype(np.int64)
    there = (blk >= 0) & (blk < nb)
    raw = np.ascontiguousarray(cache[np.where(there, blk, 0), t % bs, h])
    with np.errstate(invalid="ignore"):
        out = DECODE[raw[:, :-4]] * np.ascontiguousarray(raw[:, -4:]).view(np.float32).astype(np.float64)
    out[~there] = 0.0
    return out, there


def window_reference(q, kc, vc, table, lens, qlens, window, sinks, scale, dtype):
    """(out, bound) float64 [T, Hq, Dv] of windowed attention, bounds as in tests/_rows.py:
    both kernels keep logits and weights in float32 and give the weights 16 bits beside V."""
    hq, hkv = q.shape[1], kc.shape[2]
    out = np.zeros((q.shape[0], hq, vc.shape[3] - 4))
    bound = np.zeros_like(out)
    row = 0
    for b, (size, n) in enumerate(zip(lens, qlens)):
        at, t = size - n + np.arange(n)[:, None], np.arange(size)[None, :]
        inside = (t <= at) & ((t > at - window) | (t < sinks))
        for h in range(hkv):
            key, there = cached_rows(kc, table, b, size, h)
            value, _ = cached_rows(vc, table, b, size, h)
            sees = inside & there
            for head in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                sm = Softmax(q[row:row + n, head], key, sees, scale)
                out[row:row + n, head], bound[row:row + n, head] = attention_with_bound(sm, value, dtype)
        row += n
    return out, bound


def verify_reference(probs, draft, tokens, parents, uniforms, qlens, width):
    """(accepted, counts, next tokens), each request by itself; float32 numpy arrays in."""
    accepted = np.full((len(qlens), width), -1, dtype=np.int32)
    counts, drawn, row = [], [], 0
    vocab = probs.shape[1]

    def weight_of(values):
        return np.where(np.isfinite(values) & (values > 0), values, 0.0)

    for b, n in enumerate(qlens):
        if n == 0:
            counts.append(0)
            drawn.append(-1)
            continue
        u = uniforms[row:row + n].astype(np.float64)
        x = tokens[row:row + n]
        up = parents[row:row + n] if parents is not None else np.arange(n) - 1
        now, path = 0, [0]
        while True:
            with np.errstate(invalid="ignore"):
                p = probs[row + now].astype(np.float64)
                rest, taken, gone, residual = 1.0, None, [], p
                for j in range(now + 1, n):
                    if up[j] != now:
                        continue
                    mass = p[x[j]] if 0 <= x[j] < vocab and x[j] not in gone else 0.0
                    mass = mass if mass > 0 else 0.0
                    if draft is not None:
                        q = draft[row + j].astype(np.float64)
                        residual = p - q
                        if mass > 0 and u[j] * q[x[j]] < mass:
                            taken = j
                    elif mass > 0 and u[j] * rest < mass:
                        taken = j
                    if taken is not None:
                        break
                    rest -= mass
                    gone.append(x[j])
            if taken is None:
                break
            now = taken
            path.append(now)
        weight = weight_of(residual)
        if draft is None:
            weight[[v for v in gone if 0 <= v < vocab]] = 0.0
        if not weight.sum() > 0:
            weight = weight_of(p)
        upto = np.cumsum(weight)
        some = np.flatnonzero(weight)
        past = np.flatnonzero((upto > u[0] * upto[-1]) & (weight > 0))
        drawn.append(int(past[0]) if past.size else int(some[-1]) if some.size else -1)
        counts.append(len(path))
        accepted[b, :len(path)] = path
        row += n
    return accepted, np.array(counts, dtype=np.int32), np.array(drawn, dtype=np.int64)


def extend_reference(table, free, count, ctx, qlens, page, total):
    """(slots, positions, lens, missing, table, count) of lists and numpy copies."""
    table = table.copy()
    slots, at, missing = np.full(total, -1, dtype=np.int64), np.full(total, -1, dtype=np.int64), []
    row = 0
    for b, (c, n) in enumerate(zip(ctx, qlens)):
        lack = 0
        for j in range(c // page, -(-(c + n) // page) if n else c // page):
            if j >= table.shape[1]:
                lack += 1
            elif table[b, j] < 0:
                if count:
                    count -= 1
                    table[b, j] = free[count]
                else:
                    lack += 1
        missing.append(lack)
        for p in range(c, c + n):
            j = p // page
            at[row] = p
            if j < table.shape[1] and table[b, j] >= 0:
                slots[row] = int(table[b, j]) * page + p % page
            row += 1
    return slots, at, [c + n for c, n in zip(ctx, qlens)], missing, table, count


def release_reference(table, free, count, lens, page, window=None, sinks=0):
    table, free = table.copy(), free.copy()
    for b in range(table.shape[0]):
        for j in range(table.shape[1]):
            needed = j * page < lens[b] and (window is None or j * page < sinks or (j + 1) * page > lens[b] + 1 - window)
            if table[b, j] >= 0 and not needed and count < len(free):
                free[count], table[b, j] = table[b, j], -1
                count += 1
    return table, free, count
