"""Timed calls of the operators around a decoding step over the HiF8 paged KV cache.

Four operators: pages taken for new tokens and the tokens' slots
(``extend``), pages given back (``release``), attention with a sliding window
and first tokens that stay visible (``window``), and verification of drafted
tokens against the target model's probabilities (``verify``).  Where ``own``
is false each runs in its plain form: indexing, sorting, products, exponentials
and sums in torch, in float32, the verification and its sums in float64.

Caches are uint8 ``[num_blocks, page, kv_heads, dim + 4]``: HiF8 codes and the
row's float32 scale.  Head counts and sizes, page and vocabulary are those of
the hybrid model (16 query / 4 KV heads of 256, 128-token pages, 151936
tokens) and generic ones.
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
        # A decode step of eight requests: most need no new page. Latency.
        {"name": "extend_8x1", "kind": "extend", "batch": 8, "ctx": 3000, "new": 1, "page": 128},
        # 48 prompts of 2k to 4k tokens admitted together onto 16-token pages.
        {"name": "extend_48x4k", "kind": "extend", "batch": 48, "ctx": 0, "new": 4096, "page": 16},
        # Eight requests after a rejected chain of drafts: a page or none each.
        {"name": "release_8", "kind": "release", "batch": 8, "ctx": 3000, "behind": 9, "page": 128, "window": 0,
         "sinks": 0},
        # 256 requests of 16k to 32k tokens on 16-token pages whose layers look back 4096: most pages go.
        {"name": "release_256x32k", "kind": "release", "batch": 256, "ctx": 32768, "behind": 16, "page": 16,
         "window": 4096, "sinks": 4},
        # One decode step of one request that has just outgrown its window.
        {"name": "decode_1x1k", "kind": "window", "batch": 1, "ctx": 1500, "new": 1, "window": 1024, "sinks": 4,
         "released": False, **model},
        # One decode step of 32 requests of 16k to 32k tokens, pages outside the window given back.
        {"name": "decode_32x4k", "kind": "window", "batch": 32, "ctx": 32768, "new": 1, "window": 4096, "sinks": 4,
         "released": True, **model},
        # Chains of up to five drafts: three query heads per KV head, 16-token pages, odd lengths, fp16, row scales.
        {"name": "drafts_ragged", "kind": "window", "batch": 11, "ctx": 5003, "new": 5, "window": 1000, "sinks": 21,
         "released": True, "heads": 24, "kv_heads": 8, "dim": 128, "page": 16, "dtype": "fp16", "row_scales": True},
        # A step of chunked prefill: up to 512 new tokens each of four requests.
        {"name": "chunk_4x512", "kind": "window", "batch": 4, "ctx": 16384, "new": 512, "window": 4096, "sinks": 4,
         "released": True, **model},
        # A whole prompt of 8192 tokens.
        {"name": "prompt_8k", "kind": "window", "batch": 1, "ctx": 8192, "new": 8192, "window": 2048, "sinks": 64,
         "released": False, **model},
        # One request that verifies four sampled drafts: latency.
        {"name": "verify_1x5", "kind": "verify", "batch": 1, "new": 5, "vocab": 151_936, "sampled": True, "tree": False},
        # 64 requests with chains of up to seven sampled drafts.
        {"name": "verify_64x8", "kind": "verify", "batch": 64, "new": 8, "vocab": 151_936, "sampled": True,
         "tree": False},
        # Trees of up to 32 nodes of given (not sampled) tokens, an odd vocabulary.
        {"name": "verify_tree", "kind": "verify", "batch": 16, "new": 32, "vocab": 50_257, "sampled": False,
         "tree": True},
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng) -> dict:
    kind = rng.choice(["window", "window", "window", "verify", "verify", "extend", "release"])
    if kind == "verify":
        case = {"kind": kind, "batch": _log_int(rng, 1, 64), "vocab": _log_int(rng, 1000, 160_000),
                "tree": rng.random() < 0.4}
        case["new"] = _log_int(rng, 1, max(2, min(48, 80_000_000 // (case["batch"] * case["vocab"]))))
        case["sampled"] = not case["tree"] and rng.random() < 0.6
        return case
    page = rng.choice([16, 16, 32, 64, 128, 144])
    if kind in ("extend", "release"):
        case = {"kind": kind, "batch": _log_int(rng, 1, 256), "page": page}
        case["ctx"] = _log_int(rng, 1, min(32768, 2_000_000 // case["batch"]))
        if kind == "extend":
            case["new"] = _log_int(rng, 1, max(2, min(8192, 190_000 // case["batch"])))
        else:
            case.update(behind=_log_int(rng, 1, 200), window=rng.choice([0, _log_int(rng, 1, 8192)]))
            case["sinks"] = rng.choice([0, 4, 130]) if case["window"] else 0
        return case
    heads, kv_heads, dim = rng.choice([(16, 4, 256), (16, 4, 256), (24, 8, 128), (32, 4, 128), (8, 2, 128), (12, 4, 64),
                                       (8, 8, 64), (20, 2, 256)])
    case = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page,
            "dtype": rng.choice(["bf16", "bf16", "fp16"]), "row_scales": rng.random() < 0.3,
            "released": rng.random() < 0.5, "batch": _log_int(rng, 1, 24), "window": _log_int(rng, 1, 8192),
            "sinks": rng.choice([0, 1, 4, 4, 64, 300])}
    case["ctx"] = _log_int(rng, 33, max(64, min(32768, 150_000 // case["batch"])))
    case["new"] = 1
    if rng.random() < 0.6:
        reach = min(case["ctx"], case["window"] + case["sinks"])
        most = 300_000_000_000 // (4 * heads * dim * case["batch"] * reach)
        case["new"] = min(case["ctx"], _log_int(rng, 2, max(2, min(4096, most))))
    return case


def _ragged(most: int, batch: int) -> list[int]:
    """Lengths between half of ``most`` and ``most``, the first of them ``most``."""
    return [most - (b * 7919) % (most // 2 + 1) for b in range(batch)]


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """(tokens cached before this call's own, this call's own) of each request."""
    batch = case["batch"]
    if case["kind"] == "verify":
        return [0] * batch, _ragged(case["new"], batch)
    ctx = _ragged(case["ctx"], batch) if case["ctx"] else [0] * batch
    if case["kind"] == "release":
        return ctx, [0] * batch
    new = _ragged(case["new"], batch)
    if case["kind"] == "window":  # ctx counts this call's tokens
        new = [min(c, n) for c, n in zip(ctx, new)]
        ctx = [c - n for c, n in zip(ctx, new)]
    return ctx, new


def _held(case: dict) -> list[int]:
    """Pages that each request of a release holds, those of rejected tokens among them."""
    ctx, _ = _lengths(case)
    return [-(-(c + (b * 5) % (case["behind"] + 1)) // case["page"]) for b, c in enumerate(ctx)]


def _columns(case: dict) -> int:
    ctx, new = _lengths(case)
    need = _held(case) if case["kind"] == "release" else [-(-(c + n) // case["page"]) for c, n in zip(ctx, new)]
    return max(need) + 1


def _seen(case: dict, c: int, n: int) -> tuple[int, int]:
    """(cached rows that some query of a request sees, (query, row) pairs) under the window."""
    window, sinks = case["window"], case["sinks"]
    first = max(0, c + 1 - window)
    rows = c + n - first + min(sinks, first)
    # The query at position P sees min(P + 1, window + sinks) rows.
    reach = window + sinks
    full = max(0, c + n - max(c, reach))
    part = n - full
    pairs = full * reach + part * c + part * (part + 1) // 2
    return rows, pairs


def work(case: dict) -> dict:
    ctx, new = _lengths(case)
    if case["kind"] == "verify":
        rows = case["batch"] * (2 if case["sampled"] else 1)
        return {"bytes": rows * case["vocab"] * 4 + sum(new) * 20, "flops": 0}
    if case["kind"] == "extend":
        pages = sum(-(-(c + n) // case["page"]) - c // case["page"] for c, n in zip(ctx, new))
        return {"bytes": sum(new) * 16 + pages * 12 + case["batch"] * 16, "flops": 0}
    if case["kind"] == "release":
        gone = sum(held - sum(_stays(case, c, j) for j in range(held)) for c, held in zip(ctx, _held(case)))
        return {"bytes": case["batch"] * _columns(case) * 4 + gone * 8, "flops": 0}
    heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
    rows, pairs = (sum(v) for v in zip(*(_seen(case, c, n) for c, n in zip(ctx, new))))
    return {"bytes": rows * kv * 2 * (dim + 4) + 2 * sum(new) * heads * dim * 2, "flops": 4 * pairs * heads * dim}


def _stays(case: dict, length: int, j: int) -> bool:
    """Whether a request of ``length`` tokens goes on needing its page j."""
    page, window = case["page"], case["window"]
    return j * page < length and (not window or j * page < case["sinks"] or (j + 1) * page > length + 1 - window)


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


def _int32(values, dev) -> torch.Tensor:
    return torch.tensor(values, dtype=torch.int32, device=dev)


def _table(case: dict, held: list[list[int]], columns: int, spare: int, g: torch.Generator):
    """(block table of the pages held, ids that are left, number of pages in all)."""
    blocks = sum(map(len, held)) + spare
    pages = torch.randperm(blocks, generator=g, device=g.device).to(torch.int32)
    where = torch.tensor([b * columns + j for b, row in enumerate(held) for j in row], dtype=torch.int64, device=g.device)
    table = torch.full((len(held) * columns,), -1, dtype=torch.int32, device=g.device)
    table[where] = pages[:where.numel()]
    return table.view(len(held), columns), pages[where.numel():], blocks


def prepare(case: dict, seed: int) -> dict:
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)
    ctx, new = _lengths(case)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {"kind": case["kind"], "case": case, "starts": _int32(starts, dev), "total": starts[-1], "max_new": max(new)}
    if case["kind"] == "verify":
        return _prepare_verify(case, new, state, g)
    page, columns = case["page"], _columns(case)
    state.update(page=page, ctx=_int32(ctx, dev), lens=_int32([c + n for c, n in zip(ctx, new)], dev))
    if case["kind"] == "extend":
        held = [list(range(-(-c // page))) for c in ctx]
        fresh = sum(-(-(c + n) // page) - len(h) for c, n, h in zip(ctx, new, held))
        state["table"], left, blocks = _table(case, held, columns, fresh + 7, g)
        state["free"] = torch.full((blocks,), -1, dtype=torch.int32, device=dev)
        state["free"][:left.numel()] = left
        state["count"] = _int32([left.numel()], dev)
        return state
    if case["kind"] == "release":
        state["table"], left, blocks = _table(case, [list(range(h)) for h in _held(case)], columns, 7, g)
        state["free"] = torch.full((blocks,), -1, dtype=torch.int32, device=dev)
        state["free"][:left.numel()] = left
        state["count"] = _int32([left.numel()], dev)
        return state
    held = []
    for c, n in zip(ctx, new):
        low = max(0, c + 1 - case["window"])
        held.append([j for j in range(-(-(c + n) // page))
                     if not case["released"] or j * page < case["sinks"] or (j + 1) * page > low])
    state["table"], _, blocks = _table(case, held, columns, 2, g)
    state.update(value_of=_code_values(torch.float32).to(dev), dim=case["dim"], scale=1.0 / math.sqrt(case["dim"]),
                 keys=_cache(case, blocks, 3.0, g), values=_cache(case, blocks, 1.5, g), window=case["window"],
                 sinks=case["sinks"], max_len=max(c + n for c, n in zip(ctx, new)))
    state["query"] = torch.randn(state["total"], case["heads"], case["dim"], generator=g, device=dev).to(
        _DTYPES[case["dtype"]])
    return state


def _prepare_verify(case: dict, new: list[int], state: dict, g: torch.Generator) -> dict:
    """Target rows, drafts drawn near them, one uniform number per row."""
    dev, vocab, rows = g.device, case["vocab"], state["total"]
    # Logits as a vocabulary head gives them: a few likely tokens, a long tail.
    def likely():
        logits = torch.randn(rows, vocab, generator=g, device=dev)
        logits.scatter_add_(1, torch.randint(0, vocab, (rows, 12), generator=g, device=dev),
                            9 + 5 * torch.rand(rows, 12, generator=g, device=dev))
        return logits

    logits = likely()
    state["probs"] = torch.softmax(logits, dim=-1)
    # The row that row i of the drafts continues: the one before it, or (in a tree) one of the eight before it.
    row, first = torch.arange(rows, device=dev), torch.zeros(rows, dtype=torch.int64, device=dev)
    for s, n in zip(state["starts"].tolist(), new):
        first[s:s + n] = s
    back = torch.randint(1, 9, (rows,), generator=g, device=dev) if case["tree"] else torch.ones_like(row)
    parent = torch.maximum(row - back, first)
    # The draft model's distribution of row i's token, after its parent: the target's, disturbed.
    draft = logits[parent] + 0.8 * torch.randn(rows, vocab, generator=g, device=dev)
    del logits
    draft = torch.softmax(draft, dim=-1)
    if case["sampled"]:
        tokens = torch.multinomial(draft, 1, generator=g)[:, 0]
        state["draft"] = draft
    else:
        best = torch.topk(draft, 4, dim=-1)[1]
        tokens = best.gather(1, torch.randint(0, 4, (rows, 1), generator=g, device=dev))[:, 0]
        state["draft"] = None
    state["tokens"] = tokens.to(torch.int32)
    state["parents"] = torch.where(row > first, parent - first, -1).to(torch.int32) if case["tree"] else None
    state["uniforms"] = torch.rand(rows, generator=g, device=dev)
    return state


# --------------------------------------------------------------- plain form
def _extend_plain(s: dict, table, count):
    page, batch, columns = s["page"], *table.shape
    starts, ctx = s["starts"].long(), s["ctx"].long()
    new = starts[1:] - starts[:-1]
    j = torch.arange(columns, device=table.device)
    wants = (j >= (ctx // page)[:, None]) & (j * page < (ctx + new)[:, None]) & (new > 0)[:, None] & (table < 0)
    rank = torch.cumsum(wants.reshape(-1).to(torch.int64), 0).view(batch, columns) - 1
    gets = wants & (rank < count)
    ids = s["free"][(count - 1 - rank).clamp(0, s["free"].numel() - 1)]
    table.copy_(torch.where(gets, ids, table))
    missing = (wants & ~gets).sum(1).to(torch.int32)
    count.sub_(gets.sum().to(torch.int32))
    row = torch.arange(s["total"], device=table.device)
    b = torch.searchsorted(starts, row, right=True) - 1
    at = ctx[b] + row - starts[b]
    block = table[b, at // page].long()
    return torch.where(block < 0, -1, block * page + at % page), at, s["ctx"] + new.to(torch.int32), missing


def _release_plain(s: dict, table, free, count):
    page, window = s["page"], s["case"]["window"]
    j = torch.arange(table.shape[1], device=table.device)
    size = s["ctx"].long()[:, None]
    stays = j * page < size
    if window:
        stays = stays & ((j * page < s["case"]["sinks"]) | ((j + 1) * page > size + 1 - window))
    goes = (table >= 0) & ~stays
    place = torch.cumsum(goes.reshape(-1).to(torch.int64), 0).view_as(goes) - 1 + count
    end = free.numel()                                    # one place more takes what stays
    longer = torch.cat([free, free.new_zeros(1)])
    longer[torch.where(goes, place, end).reshape(-1)] = table.reshape(-1)
    free.copy_(longer[:end])
    count.add_(goes.sum().to(torch.int32))
    table.masked_fill_(goes, -1)


def _decoded(s: dict, cache: torch.Tensor, slots: torch.Tensor) -> torch.Tensor:
    """Decoded rows [Hkv, L, D] of slots [L], float32."""
    dim = s["dim"]
    raw = cache.view(-1, cache.shape[2], dim + 4)[slots].transpose(0, 1)
    return s["value_of"][raw[..., :dim].int()] * raw[..., dim:].contiguous().view(torch.float32)


def _window_plain(s: dict) -> torch.Tensor:
    """Requests one by one (their lengths are known), 512 query rows at a time over the rows that those see."""
    ctx, new = _lengths(s["case"])
    window, sinks, page, heads = s["window"], s["sinks"], s["page"], s["query"].shape[1]
    kv, dim, dev = s["keys"].shape[2], s["dim"], s["query"].device
    out, row = torch.empty_like(s["query"]), 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        for i in range(0, n, 512):
            k = min(512, n - i)
            low = max(0, c + i + 1 - window)
            t = torch.cat([torch.arange(0, min(sinks, low), device=dev), torch.arange(low, c + i + k, device=dev)])
            slots = s["table"][b, t // page].long() * page + t % page
            key, value = _decoded(s, s["keys"], slots), _decoded(s, s["values"], slots)
            at = c + i + torch.arange(k, device=dev)[:, None]
            sees = (t <= at) & ((t > at - window) | (t < sinks))                          # [k, L]
            q = s["query"][row + i:row + i + k].float().view(k, kv, heads // kv, dim)
            q = q.permute(1, 2, 0, 3).reshape(kv, -1, dim)                                # [Hkv, G k, D]
            x = torch.matmul(q, key.transpose(1, 2).contiguous()) * s["scale"]
            x = x.view(kv, -1, k, t.numel()).masked_fill(~sees, -math.inf)
            p = torch.exp(x - x.amax(-1, keepdim=True))
            p = p / p.sum(-1, keepdim=True)
            o = torch.matmul(p.view(kv, -1, t.numel()), value).view(kv, heads // kv, k, dim)
            out[row + i:row + i + k] = o.permute(2, 0, 1, 3).reshape(k, heads, dim).to(out.dtype)
        row += n
    return out


def _verify_plain(s: dict):
    probs, starts = s["probs"], s["starts"].long()
    first, new = starts[:-1], starts[1:] - starts[:-1]
    batch, width, dev = new.numel(), s["max_new"], probs.device
    i = torch.arange(width, device=dev)
    there = i < new[:, None]
    at = torch.where(there, first[:, None] + i, 0)
    tokens, u = s["tokens"][at].long(), s["uniforms"][at].double()
    parent = s["parents"][at].long() if s["parents"] is not None else (i - 1).expand(batch, width)
    accepted = torch.full((batch, width), -1, dtype=torch.int32, device=dev)
    accepted[:, 0] = 0
    count = torch.ones(batch, dtype=torch.int64, device=dev)
    now = torch.zeros(batch, dtype=torch.int64, device=dev)
    rest = torch.ones(batch, dtype=torch.float64, device=dev)
    each = torch.arange(batch, device=dev)
    for k in range(1, width):
        child = there[:, k] & (parent[:, k] == now)
        x = tokens[:, k]
        p = probs[first + now, x].double()
        if s["draft"] is not None:
            q = s["draft"][at[:, k], x].double()
            takes = child & (u[:, k] * q < p)
            # A chain ends at its first rejection: no later row continues row `now`.
        else:
            again = ((parent[:, 1:k] == now[:, None]) & (tokens[:, 1:k] == x[:, None])).any(1)
            p = torch.where(again, 0.0, p)
            takes = child & ~again & (u[:, k] * rest < p)
            rest = torch.where(takes, 1.0, torch.where(child, rest - p, rest))
        accepted[each, torch.where(takes, count, 0)] = torch.where(takes, k, 0).to(torch.int32)
        now = torch.where(takes, k, now)
        count = count + takes
    weight = probs[first + now].double()
    if s["draft"] is not None:
        other = s["draft"][torch.clamp(first + now + 1, max=s["total"] - 1)].double()
        weight = torch.where((now + 1 < new)[:, None], (weight - other).clamp_min(0.0), weight)
    else:
        gone = there & (parent == now[:, None]) & (i > 0)
        # One column more takes what is no rejected child.
        keep = torch.ones(batch, weight.shape[1] + 1, dtype=torch.float64, device=dev)
        keep.scatter_(1, torch.where(gone, tokens, weight.shape[1]), 0.0)
        weight = weight * keep[:, :-1]
    upto = torch.cumsum(weight, dim=1)
    drawn = torch.searchsorted(upto, u[:, :1] * upto[:, -1:], right=True)[:, 0]
    return accepted, count.to(torch.int32), drawn.clamp_max(probs.shape[1] - 1)


# --------------------------------------------------------------------- run
def run(state: dict):
    s = state
    if own:
        return _run_own(s)
    if s["kind"] == "window":
        return _window_plain(s)
    if s["kind"] == "verify":
        return _verify_plain(s)
    table, count = s["table"].clone(), s["count"].clone()   # a pass starts from the same pages each time
    if s["kind"] == "extend":
        return (*_extend_plain(s, table, count), table, count)
    free = s["free"].clone()
    _release_plain(s, table, free, count)
    return table, free, count


def _run_own(s: dict):
    if str(_PACKAGE) not in sys.path:
        sys.path.insert(0, str(_PACKAGE))
    from hif8_rocm import kv_cache

    if s["kind"] == "window":
        seen = {"window": s["window"], "sinks": s["sinks"], "scale": s["scale"], "max_seq_len": s["max_len"],
                "validate": False}
        if s["max_new"] == 1:
            return kv_cache.paged_decode_attention(s["query"], s["keys"], s["values"], s["table"], s["lens"], **seen)
        return kv_cache.paged_attention(s["query"], s["keys"], s["values"], s["table"], s["lens"],
                                        query_start_loc=s["starts"], max_query_len=s["max_new"], **seen)
    if s["kind"] == "verify":
        return kv_cache.verify_drafts(s["probs"], s["tokens"], s["uniforms"], draft_probs=s["draft"],
                                      parents=s["parents"], query_start_loc=s["starts"], max_query_len=s["max_new"],
                                      validate=False)
    table, count = s["table"].clone(), s["count"].clone()
    if s["kind"] == "extend":
        got = kv_cache.extend_block_tables(table, s["free"], count, s["ctx"], block_size=s["page"],
                                           query_start_loc=s["starts"], total_query_tokens=s["total"], validate=False)
        return (*got, table, count)
    free = s["free"].clone()
    kv_cache.release_blocks(table, free, count, s["ctx"], block_size=s["page"], window=s["case"]["window"] or None,
                            sinks=s["case"]["sinks"], validate=False)
    return table, free, count


# ------------------------------------------------------------------- exact
def exact(case: dict, seed: int):
    """Each request by itself, page by page and in float64."""
    s = prepare(case, seed)
    ctx, new = _lengths(case)
    dev = s["starts"].device
    if case["kind"] == "window":
        return _window_exact(case, s, ctx, new)
    if case["kind"] == "verify":
        return _verify_exact(s, new)
    page = case["page"]
    table, free, count = s["table"].tolist(), s["free"].tolist(), int(s["count"][0])
    if case["kind"] == "release":
        for row, size in zip(table, ctx):
            for j, block in enumerate(row):
                if block >= 0 and not _stays(case, size, j):
                    free[count], row[j] = block, -1
                    count += 1
        return _int32(table, dev), _int32(free, dev), _int32([count], dev)
    slots, at, missing = [], [], []
    for row, c, n in zip(table, ctx, new):
        missing.append(0)
        for p in range(c, c + n):
            j = p // page
            if row[j] < 0:
                if count:
                    count -= 1
                    row[j] = free[count]
                elif p == c or p % page == 0:
                    missing[-1] += 1
            slots.append(row[j] * page + p % page if row[j] >= 0 else -1)
            at.append(p)
    return (torch.tensor(slots, device=dev), torch.tensor(at, device=dev), s["lens"], _int32(missing, dev),
            _int32(table, dev), _int32([count], dev))


def _window_exact(case: dict, s: dict, ctx: list[int], new: list[int]) -> torch.Tensor:
    dev, dim, kv = s["query"].device, case["dim"], case["kv_heads"]
    group, page = case["heads"] // kv, case["page"]
    value_of = _code_values(torch.float64).to(dev)
    out = torch.zeros(s["total"], case["heads"], dim, dtype=torch.float64, device=dev)
    row = 0
    for b, (c, n) in enumerate(zip(ctx, new)):
        pages = s["table"][b, :-(-(c + n) // page)].long()
        for h in range(kv):
            def decoded(cache):
                raw = cache[pages.clamp_min(0), :, h].reshape(-1, dim + 4)[:c + n]
                return value_of[raw[:, :dim].long()] * raw[:, dim:].contiguous().view(torch.float32).double()

            key, value = decoded(s["keys"]), decoded(s["values"])
            for i in range(0, n, 1024):
                k = min(1024, n - i)
                # Rows that none of these queries can see lie before `low`, the first tokens apart.
                low = max(0, c + i + 1 - case["window"])
                near = torch.arange(low, c + i + k, device=dev)
                t = torch.cat([torch.arange(min(case["sinks"], low), device=dev), near])
                at = torch.arange(c + i, c + i + k, device=dev)[:, None]
                hidden = (t > at) | ((at - t >= case["window"]) & (t >= case["sinks"]))
                for head in range(h * group, (h + 1) * group):
                    x = s["query"][row + i:row + i + k, head].double() @ key[t].T / math.sqrt(dim)
                    out[row + i:row + i + k, head] = torch.softmax(x.masked_fill(hidden, -math.inf), dim=-1) @ value[t]
        row += n
    return out


def _verify_exact(s: dict, new: list[int]):
    accepted, counts, drawn, row = [], [], [], 0
    for n in new:
        tokens, u = s["tokens"][row:row + n].tolist(), s["uniforms"][row:row + n].double().tolist()
        parents = s["parents"][row:row + n].tolist() if s["parents"] is not None else list(range(-1, n - 1))
        path = [0]
        while True:
            p = s["probs"][row + path[-1]].double()
            weight, left, taken = p.clone(), 1.0, None
            for k in (k for k in range(1, n) if parents[k] == path[-1]):
                x = tokens[k]
                if s["draft"] is not None:
                    q = s["draft"][row + k].double()
                    if u[k] * float(q[x]) < float(p[x]):
                        taken = k
                        break
                    weight = torch.clamp(p - q, min=0.0)
                else:
                    mass = float(weight[x])
                    if mass > 0 and u[k] * left < mass:
                        taken = k
                        break
                    left, weight[x] = left - mass, 0.0
            if taken is None:
                break
            path.append(taken)
        upto = torch.cumsum(weight, 0)
        drawn.append(int((upto <= u[0] * upto[-1]).sum().clamp_max(upto.numel() - 1)))
        counts.append(len(path))
        accepted.append(path + [-1] * (s["max_new"] - len(path)))
        row += n
    dev = s["probs"].device
    return _int32(accepted, dev), _int32(counts, dev), torch.tensor(drawn, device=dev)
