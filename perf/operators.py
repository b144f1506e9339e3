"""Timed calls of the operators that edit the HiF8 paged KV cache or look at it row by row.

Five operators: attention of a tree of drafted tokens over the cache
(``tree``), the acceptance of a drafted path (``accept``), decode attention
that accumulates each cached row's softmax weight (``decode``), the same
weights of many query rows at once (``weights``), and eviction of the rows of
least weight (``evict``).  Where ``own`` is false each runs in its plain form:
rows gathered through the block table and decoded to float32, products,
exponentials, sorting and indexing in torch.

Caches are uint8 ``[num_blocks, page, kv_heads, dim + 4]``: HiF8 codes and the
row's float32 scale.  Head counts and sizes are those of the hybrid model
(16 query / 4 KV heads of 256, 128-token pages) and generic ones.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = Path(__file__).resolve().parent.parent / "gcc-hif8-quantized-from-qwen3.5-9b_amd"
_DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------- cases
def listed() -> list[dict]:
    model = {"heads": 16, "kv_heads": 4, "dim": 256, "page": 128, "dtype": "bf16", "row_scales": False}
    return [
        # One short request that verifies eight drafted tokens: latency.
        {"name": "tree_1x512", "kind": "tree", "batch": 1, "ctx": 512, "drafts": 8, **model},
        # Eight long requests with trees of up to 32 nodes: the cache stream.
        {"name": "tree_8x16k", "kind": "tree", "batch": 8, "ctx": 16384, "drafts": 32, **model},
        # Three query heads per KV head, 16-token pages, odd lengths, fp16, a scale per row.
        {"name": "tree_ragged", "kind": "tree", "batch": 3, "ctx": 4099, "drafts": 61, "heads": 24, "kv_heads": 8,
         "dim": 128, "page": 16, "dtype": "fp16", "row_scales": True},
        # Acceptance after the verification of one request in a model of eight attention layers.
        {"name": "accept_1x8", "kind": "accept", "batch": 1, "ctx": 300, "drafts": 32, "layers": 8, **model},
        # The same for 32 requests decoding together.
        {"name": "accept_32x8", "kind": "accept", "batch": 32, "ctx": 200, "drafts": 64, "layers": 8, **model},
        # One decode step of one short request that keeps its key weights.
        {"name": "decode_1x512", "kind": "decode", "batch": 1, "ctx": 512, **model},
        # One decode step of eight requests of 8k to 16k cached tokens.
        {"name": "decode_8x16k", "kind": "decode", "batch": 8, "ctx": 16384, **model},
        # Key weights of the last 32 prompt tokens of four requests: what a prompt is thinned by.
        {"name": "weights_window", "kind": "weights", "batch": 4, "ctx": 8192, "rows": 32, **model},
        # Key weights of a whole 4096-token prompt.
        {"name": "weights_prompt", "kind": "weights", "batch": 1, "ctx": 4096, "rows": 4096, **model},
        # Heads of 64, 32-token pages, odd lengths, fp16, a scale per row.
        {"name": "weights_ragged", "kind": "weights", "batch": 5, "ctx": 1537, "rows": 129, "heads": 12,
         "kv_heads": 4, "dim": 64, "page": 32, "dtype": "fp16", "row_scales": True},
        # One request's cache of 600 rows cut to 512, rows never moved before.
        {"name": "evict_1x600", "kind": "evict", "batch": 1, "ctx": 600, "keep": 512, "positions": False, **model},
        # Eight caches of 8k to 16k rows cut to 4096, rows out of order from earlier cuts.
        {"name": "evict_8x16k", "kind": "evict", "batch": 8, "ctx": 16384, "keep": 4096, "positions": True, **model},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["tree", "tree", "decode", "weights", "evict", "accept"])
    heads, kv_heads, dim = rng.choice([(16, 4, 256), (16, 4, 256), (24, 8, 128), (32, 4, 128), (8, 2, 128), (12, 4, 64),
                                       (8, 8, 64), (20, 2, 256)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim,
            "page": rng.choice([16, 32, 64, 128, 144]), "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "row_scales": rng.random() < 0.3, "batch": _log_int(rng, 1, 16)}
    case["ctx"] = _log_int(rng, 33, max(64, min(32768, 100000 // case["batch"])))
    if kind == "tree":
        case["drafts"] = _log_int(rng, 1, 64)
    elif kind == "accept":
        case.update(drafts=_log_int(rng, 2, 64), layers=rng.choice([1, 3, 8]), ctx=_log_int(rng, 1, 400))
    elif kind == "weights":
        most = 200_000_000 // (heads * case["batch"] * case["ctx"])
        case["rows"] = min(case["ctx"], _log_int(rng, 2, max(2, min(2048, most))))
    elif kind == "evict":
        case.update(keep=max(1, int(case["ctx"] * rng.uniform(0.1, 0.95))), positions=rng.random() < 0.5)
    return case


def _ragged(most: int, batch: int) -> list[int]:
    """Lengths between half of ``most`` and ``most``, the first of them ``most``."""
    return [most - (b * 7919) % (most // 2 + 1) for b in range(batch)]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(rows cached before this call's own tokens, this call's tokens) of each request."""
    ctx = _ragged(case["ctx"], case["batch"])
    if case["kind"] in ("tree", "accept"):
        return ctx, _ragged(case["drafts"], case["batch"])
    if case["kind"] == "decode":
        return [c - 1 for c in ctx], [1] * case["batch"]
    if case["kind"] == "weights":
        rows = [min(c, r) for c, r in zip(ctx, _ragged(case["rows"], case["batch"]))]
        return [c - r for c, r in zip(ctx, rows)], rows
    return ctx, [0] * case["batch"]


def _accepted(case: dict) -> list[int]:
    """Length of each request's accepted path."""
    return [min(1 + (3 * b + 4) % 7, (n + 1) // 2) for b, n in enumerate(_lengths(case)[1])]


def work(case: dict) -> dict:
    ctx, new = _lengths(case)
    heads, kv, dim, elem = case["heads"], case["kv_heads"], case["dim"], 2
    rows = sum(c + n for c, n in zip(ctx, new))
    if case["kind"] == "accept":
        moved = sum(_accepted(case)) * case["layers"] * kv * 2 * (dim + 4)
        return {"bytes": 2 * moved + 8 * case["batch"], "flops": 0}
    if case["kind"] == "evict":
        moved = sum(case["keep"] * (c - case["keep"]) // c for c in ctx if c > case["keep"]) * kv
        per = 8 if case["positions"] else 4
        return {"bytes": rows * kv * (per + 4) + 2 * moved * (2 * (dim + 4) + per), "flops": 0}
    pairs = sum(n * c + (n * (n + 1)) // 2 for c, n in zip(ctx, new))
    qo = sum(new) * heads * dim * elem
    if case["kind"] == "tree":
        return {"bytes": rows * kv * 2 * (dim + 4) + 2 * qo + sum(n * n for n in new), "flops": 4 * pairs * heads * dim}
    if case["kind"] == "decode":
        return {"bytes": rows * kv * (2 * (dim + 4) + 8) + 2 * qo, "flops": 4 * pairs * heads * dim}
    return {"bytes": rows * kv * (dim + 4 + 4) + qo, "flops": 2 * pairs * heads * dim}


# ------------------------------------------------------------------ inputs
def _code_values(dtype) -> torch.Tensor:
    """The value of each HiF8 byte."""
    c = torch.arange(256, dtype=torch.int64)
    m = c & 127
    small = torch.tensor([0, 0, 1, -1, 2, 3, -2, -3])[(m >> 3) & 7]
    flip = 1 - 2 * ((m >> 4) & 1)
    two, far = torch.tensor(2.0, dtype=torch.float64), m.double()
    v = (1 + (m & 1).double() / 2) * two ** (flip * (8 + ((m >> 1) & 7)))
    v = torch.where(m < 0x60, (1 + (m & 3).double() / 4) * two ** (flip * (4 + ((m >> 2) & 3))), v)
    v = torch.where(m < 0x40, (1 + (m & 7).double() / 8) * two ** small, v)
    v = torch.where(m < 8, two ** (far - 23), v)
    v = torch.where(m == 0, torch.zeros_like(v), v)
    v = torch.where(m == 0x6F, torch.full_like(v, math.inf), v)
    v = torch.where(c == 0x80, torch.full_like(v, math.nan), torch.where(c > 0x80, -v, v))
    return v.to(dtype)


def _cache(case: dict, blocks: int, mul: float, g: torch.Generator) -> torch.Tensor:
    """Pages of normal values, quantised with a scale per head or per row."""
    dev, kv, dim = g.device, case["kv_heads"], case["dim"]
    values = _code_values(torch.float32)
    grid, code = torch.sort(values[:0x6F])
    border, code = ((grid[1:] + grid[:-1]) / 2).to(dev), code.to(dev, torch.uint8)
    rows = blocks * case["page"]
    scale = 0.3 + 0.8 * torch.rand(rows if case["row_scales"] else 1, kv, generator=g, device=dev)
    scale = scale.expand(rows, kv).contiguous()
    out = torch.empty(rows, kv, dim + 4, dtype=torch.uint8, device=dev)
    x = torch.randn(rows, kv, dim, generator=g, device=dev) * mul / scale[..., None]
    mag = code[torch.bucketize(x.abs(), border)]
    out[..., :dim] = torch.where((x < 0) & (mag > 0), mag | 0x80, mag)
    out[..., dim:] = scale[..., None].view(torch.uint8)
    return out.view(blocks, case["page"], kv, dim + 4)


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    ctx, new = _lengths(case)
    batch, page, kv, dim = case["batch"], case["page"], case["kv_heads"], case["dim"]
    need = [-(-(c + n) // page) for c, n in zip(ctx, new)]
    width, blocks = max(need) + 1, sum(need) + 2
    pages = torch.randperm(blocks, generator=g, device=dev).to(torch.int32)
    table = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
    first = 0
    for b, n in enumerate(need):
        table[b, :n] = pages[first:first + n]
        first += n
    stacks = [torch.stack([_cache(case, blocks, mul, g) for _ in range(case.get("layers", 1))]) for mul in (3.0, 1.5)]
    state = {
        "kind": case["kind"], "value_of": _code_values(torch.float32).to(dev), "table": table,
        "scale": 1.0 / math.sqrt(dim), "page": page, "dim": dim,
        "stacks": stacks, "keys": list(stacks[0].unbind()), "values": list(stacks[1].unbind()),
        "ctx": torch.tensor(ctx, dtype=torch.int32, device=dev),
        "lens": torch.tensor([c + n for c, n in zip(ctx, new)], dtype=torch.int32, device=dev),
        "max_len": max(c + n for c, n in zip(ctx, new)), "max_new": max(new), "total": sum(new),
    }
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device=dev)
    if state["total"]:
        state["query"] = torch.randn(state["total"], case["heads"], dim, generator=g, device=dev).to(
            _DTYPES[case["dtype"]])
    if case["kind"] == "tree":
        # A random tree per request: each node's parent is one of the eight before it, or the context.
        n = case["drafts"]
        back = torch.randint(1, 9, (batch, n), generator=g, device=dev)
        parent = torch.arange(n, device=dev) - back
        hop = torch.zeros(batch, n, n, dtype=torch.float64, device=dev)
        hop.scatter_(2, parent.clamp_min(0)[..., None], (parent >= 0).double()[..., None])
        seen = torch.linalg.matrix_power(hop + torch.eye(n, dtype=torch.float64, device=dev), n) > 0
        state["mask"] = torch.cat([seen[b, :k] for b, k in enumerate(new)])
    elif case["kind"] == "accept":
        # The path's nodes lie behind its own length, as in trees that are wide at the root: the pass can be repeated.
        counts = _accepted(case)
        path = torch.zeros(batch, max(counts), dtype=torch.int32, device=dev)
        for b, (k, n) in enumerate(zip(counts, new)):
            some = torch.randperm(n - k, generator=g, device=dev)[:k] + k if n >= 2 * k else torch.arange(k, device=dev)
            path[b, :k] = torch.sort(some)[0].to(torch.int32)
        state.update(path=path, counts=torch.tensor(counts, dtype=torch.int32, device=dev))
    elif case["kind"] in ("decode", "weights", "evict"):
        rows = width * page
        w = torch.exp(2 * torch.randn(batch, kv, rows, generator=g, device=dev))
        # Rows that nothing attended to have weight zero: ties.
        w[torch.rand(batch, kv, rows, generator=g, device=dev) < 0.1] = 0.0
        w[torch.arange(rows, device=dev) >= state["lens"][:, None, None].expand(batch, kv, rows)] = 0.0
        state["weights"] = w
        if case["kind"] == "evict":
            state.update(keep=case["keep"], sinks=4, recent=state["lens"] - min(32, case["keep"] // 2))
            state["positions"] = None
            if case["positions"]:
                order = torch.rand(batch, kv, rows, generator=g, device=dev)
                order[torch.arange(rows, device=dev) >= state["lens"][:, None, None].expand(batch, kv, rows)] = 2.0
                at = torch.argsort(torch.argsort(order, dim=-1), dim=-1)
                state["positions"] = at.to(torch.int32)
    return state


# --------------------------------------------------------------- plain form
def _rows(s: dict, cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Decoded rows [B, Hkv, L, D] of slots [B, L], float32."""
    dim = s["dim"]
    raw = cache.view(-1, cache.shape[2], dim + 4)[slots].transpose(1, 2)
    scale = raw[..., dim:].contiguous().view(torch.float32)
    return s["value_of"][raw[..., :dim].int()] * scale


def _slots(s: dict, rows: int) -> torch.Tensor:
    t = torch.arange(rows, device=s["table"].device)
    block = s["table"][:, torch.clamp(t // s["page"], max=s["table"].shape[1] - 1)].long().clamp_min(0)
    return block * s["page"] + t % s["page"]


def _weights_plain(s: dict):
    """Softmax weights [B, Hkv, G * n, L] of the padded query rows and their place in the query."""
    starts = s["starts"].long()
    new = starts[1:] - starts[:-1]
    i = torch.arange(s["max_new"], device=starts.device)
    there = i < new[:, None]                                                   # [B, n]
    at = torch.where(there, starts[:-1, None] + i, 0)
    t = torch.arange(s["max_len"], device=starts.device)
    ctx, lens = s["ctx"].long(), s["lens"].long()
    if s["kind"] == "tree":
        draft = t - ctx[:, None]                                               # [B, L]
        among = s["mask"][at].gather(2, draft.clamp(0, s["mask"].shape[1] - 1)[:, None, :].expand(-1, len(i), -1))
        sees = (draft < 0)[:, None, :] | (among & (draft < new[:, None])[:, None, :])
    else:
        sees = t <= ctx[:, None, None] + i[:, None]
    sees = sees & (t < lens[:, None])[:, None, :] & there[..., None]           # [B, n, L]
    q = s["query"][at].float()                                                 # [B, n, Hq, D]
    batch, n, heads, dim = q.shape
    key = _rows(s, s["keys"][0], _slots(s, s["max_len"]))               # [B, Hkv, L, D]
    kv = key.shape[1]
    q = q.transpose(1, 2).reshape(batch, kv, heads // kv * n, dim)
    x = torch.matmul(q, key.transpose(2, 3).contiguous()) * s["scale"]
    sees = sees[:, None, None].expand(-1, kv, heads // kv, -1, -1).reshape(batch, kv, -1, s["max_len"])
    x = x.masked_fill(~sees, -math.inf)
    top = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    return torch.where(total > 0, p / total, 0.0), at, there


def _attention_plain(s: dict, p, there) -> torch.Tensor:
    value = _rows(s, s["values"][0], _slots(s, s["max_len"]))
    o = torch.matmul(p, value)                                                 # [B, Hkv, G * n, D]
    batch, n = there.shape
    o = o.reshape(batch, -1, n, s["dim"]).transpose(1, 2)                      # [B, n, Hq, D]
    return o[there].to(s["query"].dtype)


def _evict_plain(s: dict, weights, positions):
    batch, kv, rows = weights.shape
    t = torch.arange(rows, device=weights.device)
    lens = s["lens"].long()
    after = torch.clamp(lens, max=s["keep"])
    at = positions.long() if positions is not None else t.expand(batch, kv, rows)
    here = (t < lens[:, None])[:, None, :].expand(batch, kv, rows)
    safe = (at < s["sinks"]) | (at >= s["recent"].long()[:, None, None])
    rank = torch.where(here, torch.where(safe, math.inf, weights), -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True)[1]
    place = torch.empty_like(order).scatter_(2, order, t.expand(batch, kv, rows))
    stays = here & (place < after[:, None, None])
    before = (t < after[:, None])[:, None, :]
    hole, mover = (before & ~stays).nonzero().unbind(1), (stays & ~before).nonzero().unbind(1)
    slots = _slots(s, rows)
    to, frm = slots[hole[0], hole[2]], slots[mover[0], mover[2]]
    flat = [c.view(-1, kv, c.shape[-1]) for c in (s["keys"][0], s["values"][0])]
    flat[0][to, hole[1]] = flat[0][frm, mover[1]]
    flat[1][to, hole[1]] = flat[1][frm, mover[1]]
    weights[hole] = weights[mover]
    weights.masked_fill_(here & ~before, 0.0)
    if positions is not None:
        positions[hole] = positions[mover]
    return after.to(torch.int32)


def _accept_plain(s: dict):
    i = torch.arange(s["path"].shape[1], device=s["path"].device)
    taken = i < s["counts"][:, None]
    slots = _slots(s, s["table"].shape[1] * s["page"])
    ctx = s["ctx"].long()[:, None]
    to = slots.gather(1, ctx + torch.where(taken, i, 0))[taken]
    frm = slots.gather(1, ctx + torch.where(taken, s["path"], 0))[taken]
    keys, values = (c.flatten(1, 2) for c in s["stacks"])                      # [layers, slots, Hkv, D + 4]
    keys[:, to], values[:, to] = keys[:, frm], values[:, frm]
    return s["ctx"] + s["counts"]


# --------------------------------------------------------------------- run
def run(state: dict):
    s = state
    if own:
        return _run_own(s)
    if s["kind"] == "accept":
        return {"lens": _accept_plain(s), "keys": s["keys"], "values": s["values"]}
    if s["kind"] == "evict":
        weights = s["weights"].clone()   # a pass starts from the same weights and positions each time
        positions = s["positions"].clone() if s["positions"] is not None else None
        lens = _evict_plain(s, weights, positions)
        return {"lens": lens, "weights": weights, "positions": positions, "keys": s["keys"], "values": s["values"]}
    p, _, there = _weights_plain(s)
    if s["kind"] == "tree":
        return _attention_plain(s, p, there)
    sums = p.sum(2)                                                            # [B, Hkv, L]
    weights = s["weights"].clone()
    if s["kind"] == "decode":
        weights[..., :s["max_len"]] += sums
        return {"out": _attention_plain(s, p, there), "weights": weights}
    seen = (torch.arange(s["max_len"], device=sums.device) < s["lens"][:, None])[:, None, :]
    weights[..., :s["max_len"]] = torch.where(seen, sums, weights[..., :s["max_len"]])
    return weights


def _run_own(s: dict):
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    from hif8_rocm import kv_cache

    keys, values, table = s["keys"], s["values"], s["table"]
    if s["kind"] == "tree":
        return kv_cache.tree_attention(s["query"], keys[0], values[0], table, s["ctx"], s["mask"], scale=s["scale"],
                                       query_start_loc=s["starts"], max_query_len=s["max_new"],
                                       max_seq_len=s["max_len"], validate=False)
    if s["kind"] == "accept":
        lens = kv_cache.accept_drafts(keys, values, table, s["ctx"], s["path"], s["counts"], validate=False)
        return {"lens": lens, "keys": keys, "values": values}
    weights = s["weights"].clone()
    if s["kind"] == "decode":
        out = kv_cache.paged_decode_attention_weights(s["query"], keys[0], values[0], table, s["lens"], weights,
                                                      scale=s["scale"], max_seq_len=s["max_len"], validate=False)
        return {"out": out, "weights": weights}
    if s["kind"] == "weights":
        kv_cache.accumulate_key_weights(s["query"], keys[0], table, s["lens"], weights, scale=s["scale"],
                                        query_start_loc=s["starts"], max_query_len=s["max_new"],
                                        max_seq_len=s["max_len"], accumulate=False, validate=False)
        return weights
    positions = s["positions"].clone() if s["positions"] is not None else None
    lens = kv_cache.evict_kv_rows(keys[0], values[0], table, s["lens"], weights, s["keep"], positions=positions,
                                  sinks=s["sinks"], protect_from=s["recent"], max_seq_len=s["max_len"],
                                  validate=False)
    return {"lens": lens, "weights": weights, "positions": positions, "keys": keys, "values": values}


# ------------------------------------------------------------------- exact
def exact(case: dict, seed: int):
    """Each request by itself in float64."""
    if case["kind"] in ("accept", "evict"):
        return None
    s = prepare(case, seed)
    dev, dim, kv = s["table"].device, case["dim"], case["kv_heads"]
    group = case["heads"] // kv
    ctx, new = _lengths(case)
    value_of = _code_values(torch.float64).to(dev)
    out = torch.zeros(s["total"], case["heads"], dim, dtype=torch.float64, device=dev)
    weights = s["weights"].double() if "weights" in s else None
    row = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        size = c + n
        pages = s["table"][b, :-(-size // case["page"])].long()
        for h in range(kv):
            def decoded(cache):
                raw = cache[pages, :, h].reshape(-1, dim + 4)[:size]
                return value_of[raw[:, :dim].long()] * raw[:, dim:].contiguous().view(torch.float32).double()

            key, total = decoded(s["keys"][0]), torch.zeros(size, dtype=torch.float64, device=dev)
            for g in range(group):
                head = h * group + g
                x = s["query"][row:row + n, head].double() @ key.T / math.sqrt(dim)
                sees = torch.ones(n, size, dtype=torch.bool, device=dev)
                sees[:, c:] = s["mask"][row:row + n, :n] if case["kind"] == "tree" else \
                    torch.ones(n, n, dtype=torch.bool, device=dev).tril()
                p = torch.softmax(x.masked_fill(~sees, -math.inf), dim=-1)
                total += p.sum(0)
                if case["kind"] != "weights":
                    out[row:row + n, head] = p @ decoded(s["values"][0])
            if case["kind"] == "decode":
                weights[b, h, :size] += total
            elif case["kind"] == "weights":
                weights[b, h, :size] = total
        row += n
    if case["kind"] == "tree":
        return out
    return {"out": out, "weights": weights} if case["kind"] == "decode" else weights
