"""HiFloat8 paged KV cache: layout, the fused static write and decode attention.

Mirrors the reference's ``vllm_ascend_hif8.kv_cache`` layout API
(kv_cache.py:22-184) and replaces its adapter's write and attention sequences
(kv_runtime.py:1168-1339 and 1375-1563) with two native operators:

* :func:`write_kv_cache` - static quant with per-head checkpoint scales, row
  packing and slot scatter in one kernel (bytes identical to
  ``static_quant -> pack_kv_rows -> index_copy_``);
* :func:`paged_decode_attention` - one query token per request; the kernel reads
  only the pages in the block table and decodes them on chip, instead of
  gathering and materialising bf16 K/V for a fused-attention call.

Beside them stand operators without a counterpart in the reference.  A step of a
server, in their order: :func:`extend_block_tables`, :func:`write_kv_cache`,
:func:`paged_attention` (with a window or without) or :func:`tree_attention`,
:func:`verify_drafts`, :func:`accept_drafts`, :func:`release_blocks`; and
:func:`evict_kv_rows`, which holds a cache to a size.

K and V are separate uint8 tensors ``[num_blocks, block_size, num_kv_heads,
head_size + 4]``; a row is HiF8 codes followed by a little-endian FP32 scale.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Sequence

import torch

from . import native

HIF8_SCALE_BYTES = 4
HIF8_CACHE_DTYPE = "fp8_per_token_head"


@dataclass(frozen=True)
class Hif8KVCacheLayout:
    """Physical layout of one K/V cache pair (kv_cache.py:26-88)."""

    num_blocks: int
    block_size: int
    num_kv_heads: int
    head_size: int
    head_size_v: int | None = None

    def __post_init__(self) -> None:
        head_size_v = self.head_size if self.head_size_v is None else self.head_size_v
        values = (self.num_blocks, self.block_size, self.num_kv_heads, self.head_size, head_size_v)
        if any(not isinstance(value, int) or value <= 0 for value in values):
            raise ValueError(f"HIF8 KV dimensions must be positive integers, got {values}")
        if self.head_size % HIF8_SCALE_BYTES:
            raise ValueError(
                "HIF8 KV head_size must be divisible by four so the inline FP32 "
                f"scale is aligned, got {self.head_size}"
            )
        if head_size_v % HIF8_SCALE_BYTES:
            raise ValueError(
                "HIF8 KV head_size_v must be divisible by four so the inline FP32 "
                f"scale is aligned, got {head_size_v}"
            )

    @property
    def resolved_head_size_v(self) -> int:
        return self.head_size if self.head_size_v is None else self.head_size_v

    @property
    def key_width(self) -> int:
        return self.head_size + HIF8_SCALE_BYTES

    @property
    def value_width(self) -> int:
        return self.resolved_head_size_v + HIF8_SCALE_BYTES

    @property
    def page_size_bytes(self) -> int:
        return self.block_size * self.num_kv_heads * (self.key_width + self.value_width)

    @property
    def key_page_size_bytes(self) -> int:
        return self.block_size * self.num_kv_heads * self.key_width

    @property
    def value_page_size_bytes(self) -> int:
        return self.block_size * self.num_kv_heads * self.value_width

    def key_shape(self) -> tuple[int, int, int, int]:
        return (self.num_blocks, self.block_size, self.num_kv_heads, self.key_width)

    def value_shape(self) -> tuple[int, int, int, int]:
        return (self.num_blocks, self.block_size, self.num_kv_heads, self.value_width)

    def allocate(self, device: torch.device | str) -> tuple[torch.Tensor, torch.Tensor]:
        """Zero-filled K and V caches of this layout on ``device``."""
        return (
            torch.zeros(self.key_shape(), dtype=torch.uint8, device=device),
            torch.zeros(self.value_shape(), dtype=torch.uint8, device=device),
        )


def pack_kv_rows(data: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """Pack ``[T, H, D]`` codes and ``[T, H]`` FP32 scales into ``[T, H, D + 4]`` rows (kv_cache.py:151-170)."""
    if data.dtype != torch.uint8 or data.ndim != 3:
        raise TypeError("data must be a 3-D torch.uint8 tensor")
    if scale.dtype != torch.float32 or scale.shape != data.shape[:2]:
        raise TypeError("scale must be float32 with shape [tokens, heads]")
    if data.shape[-1] % HIF8_SCALE_BYTES:
        raise ValueError("head dimension must be divisible by four for inline scales")
    packed = torch.empty((*data.shape[:-1], data.shape[-1] + HIF8_SCALE_BYTES), dtype=torch.uint8,
                         device=data.device)
    packed[..., :-HIF8_SCALE_BYTES].copy_(data)
    packed[..., -HIF8_SCALE_BYTES:].copy_(
        scale.contiguous().view(torch.uint8).reshape(*scale.shape, HIF8_SCALE_BYTES))
    return packed


def unpack_kv_rows(packed: torch.Tensor, head_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Split ``[T, H, D + 4]`` rows into codes and FP32 scales (kv_cache.py:173-184)."""
    if packed.dtype != torch.uint8 or packed.ndim != 3:
        raise TypeError("packed must be a 3-D torch.uint8 tensor")
    expected = head_size + HIF8_SCALE_BYTES
    if packed.shape[-1] != expected:
        raise ValueError(f"packed last dimension must be {expected}, got {packed.shape[-1]}")
    data = packed[..., :head_size]
    scale = packed[..., head_size:].contiguous().view(torch.float32).reshape(*packed.shape[:2])
    return data, scale


def _check_caches(key_cache: torch.Tensor, value_cache: torch.Tensor) -> None:
    for name, cache in (("key_cache", key_cache), ("value_cache", value_cache)):
        if cache.dtype != torch.uint8 or cache.ndim != 4:
            raise TypeError(f"{name} must be a 4-D uint8 tensor")
        if not cache.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
    if key_cache.shape[:3] != value_cache.shape[:3]:
        raise ValueError("key_cache and value_cache must have the same blocks and heads")


def _check_window(window: int | None, sinks: int) -> tuple[int | None, int]:
    """Both as the operators take them: integers of 64 bits, past every length where they were larger."""
    if window is None:
        if sinks:
            raise ValueError("sinks need a window")
        return None, 0
    if isinstance(window, bool) or not isinstance(window, int) or window < 1:
        raise ValueError(f"window must be a positive integer, got {window}")
    if isinstance(sinks, bool) or not isinstance(sinks, int) or sinks < 0:
        raise ValueError(f"sinks must be a non-negative integer, got {sinks}")
    return min(window, 1 << 62), min(sinks, 1 << 62)


def _pages_in_window(lens: torch.Tensor, query_lens, columns: int, block_size: int, window: int, sinks: int):
    """Which table columns the query rows of each request look at, ``[B, columns]`` (lengths apart)."""
    first = torch.arange(columns, device=lens.device)[None, :] * block_size
    rows = torch.as_tensor(query_lens, device=lens.device).expand(lens.shape)
    low = (lens.to(torch.int64) - rows + 1 - window)[:, None]
    return ((first + block_size > low) | (first < sinks)) & (rows > 0)[:, None]


def write_kv_cache(
    key: torch.Tensor,
    value: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    slot_mapping: torch.Tensor,
    key_scale: torch.Tensor,
    value_scale: torch.Tensor,
    *,
    num_actual_tokens: int | None = None,
    validate: bool = True,
) -> None:
    """Quantise ``key``/``value`` ``[T, Hkv, D]`` with per-head scales into the caches, in place.

    Static branch of ``_write_hif8_cache`` (kv_runtime.py:1222-1339): row (t, h)
    becomes ``static_encode(x / scale[h])`` plus the sidecar ``scale[h]`` at
    slot ``slot_mapping[t]``; negative slots are padding and are skipped.  With
    ``validate`` a slot beyond the cache raises IndexError before anything is
    written (one host synchronisation, as in the reference); without it such
    tokens are skipped on the device.
    """
    if key is None or value is None:
        raise ValueError("HIF8 KV cache update requires both key and value")
    _check_caches(key_cache, value_cache)
    if key.ndim != 3 or value.ndim != 3:
        raise ValueError(f"expected K/V [tokens, heads, dim], got {tuple(key.shape)} / {tuple(value.shape)}")
    if key.shape[-1] + HIF8_SCALE_BYTES != key_cache.shape[-1] or \
            value.shape[-1] + HIF8_SCALE_BYTES != value_cache.shape[-1]:
        raise ValueError(
            "HIF8 KV input dimensions do not match the cache rows: "
            f"K={key.shape[-1]}+4/{key_cache.shape[-1]}, V={value.shape[-1]}+4/{value_cache.shape[-1]}"
        )
    tokens = key.shape[0] if num_actual_tokens is None else int(num_actual_tokens)
    if tokens < 0 or tokens > key.shape[0] or tokens > value.shape[0]:
        raise ValueError(f"invalid num_actual_tokens={tokens} for K/V rows {key.shape[0]}/{value.shape[0]}")
    slots = slot_mapping[:tokens]
    if slots.dtype not in (torch.int32, torch.int64):
        slots = slots.to(torch.int64)
    slots = native._as_native_operand(slots.to(key_cache.device))
    if validate and tokens:
        capacity = key_cache.shape[0] * key_cache.shape[1]
        if bool((slots >= capacity).any()):
            raise IndexError("HIF8 KV slot mapping references an invalid block")
    extension = native.load_extension()
    native._operator("hif8_kv_cache_write", extension)(
        key[:tokens].contiguous(), value[:tokens].contiguous(), key_cache, value_cache, slots,
        key_scale.to(torch.float32).contiguous(), value_scale.to(torch.float32).contiguous(), None)


def paged_decode_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int] | torch.Tensor,
    *,
    scale: float,
    max_seq_len: int | None = None,
    window: int | None = None,
    sinks: int = 0,
    validate: bool = True,
) -> torch.Tensor:
    """Decode attention over HiF8 pages: ``query`` ``[B, Hq, D]`` -> ``[B, Hq, Dv]``.

    One query token per request (the last position, so the causal mask admits
    every cached token); the contract is ``paged_attention_reference``
    (kv_cache.py:314-372) with ``query_lens`` all 1.  ``seq_lens`` may be a host
    sequence (as the reference's ``seq_lens_list``) or an int32 device tensor;
    with a tensor, pass ``max_seq_len`` to avoid a host synchronisation.
    ``validate`` checks the block ids that the lengths reach (kv_cache.py:247-249).

    With ``window`` the token sees the last ``window`` cached tokens (itself among
    them) and the first ``sinks`` alone, as in :func:`paged_attention`.
    """
    _check_caches(key_cache, value_cache)
    window, sinks = _check_window(window, sinks)
    if query.ndim != 3:
        raise ValueError("query must have shape [tokens, num_heads, head_size]")
    batch = query.shape[0]
    if query.shape[1] % key_cache.shape[2]:
        raise ValueError("num_heads must be divisible by num_kv_heads")
    if block_table.ndim != 2 or block_table.shape[0] < batch:
        raise ValueError("block_table must have shape [batch, max_blocks]")
    block_size = key_cache.shape[1]
    if isinstance(seq_lens, torch.Tensor):
        lens_dev = seq_lens.to(device=query.device, dtype=torch.int32).contiguous()
        if max_seq_len is None:
            max_seq_len = int(lens_dev.max().item()) if batch else 0
        lengths = None
    else:
        lengths = [int(v) for v in seq_lens]
        if len(lengths) != batch:
            raise ValueError("one sequence length is required per request")
        if any(v < 0 for v in lengths):
            raise ValueError("sequence lengths must be non-negative")
        lens_dev = torch.tensor(lengths, dtype=torch.int32).to(query.device)
        if max_seq_len is None:
            max_seq_len = max(lengths, default=0)
    if max_seq_len > block_table.shape[1] * block_size:
        raise ValueError("block_table has too few entries for a sequence length")
    table = block_table[:batch]
    if table.dtype not in (torch.int32, torch.int64):
        table = table.to(torch.int64)
    table = table.to(query.device).contiguous()
    if validate and batch and max_seq_len > 0:
        if bool((lens_dev > max_seq_len).any()):
            raise ValueError("max_seq_len is smaller than a sequence length")
        needed = (max_seq_len + block_size - 1) // block_size
        used = torch.arange(needed, device=query.device)[None, :] * block_size < lens_dev[:, None].to(torch.int64)
        if window is not None:
            used &= _pages_in_window(lens_dev, 1, needed, block_size, window, sinks)
        ids = table[:, :needed].to(torch.int64)
        if bool(((ids < 0) | (ids >= key_cache.shape[0]))[used].any()):
            raise IndexError("block_table references a block outside the cache")
    extension = native.load_extension()
    if window is not None:
        return native._operator("hif8_window_attention", extension)(
            query.contiguous(), key_cache, value_cache, table, None, lens_dev, float(scale), window, sinks, 1,
            int(max_seq_len))
    return native._operator("hif8_paged_decode_attention", extension)(
        query.contiguous(), key_cache, value_cache, table, lens_dev, float(scale), int(max_seq_len))


def paged_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int] | torch.Tensor,
    *,
    scale: float,
    query_lens: Sequence[int] | None = None,
    query_start_loc: torch.Tensor | None = None,
    causal: bool = True,
    max_query_len: int | None = None,
    max_seq_len: int | None = None,
    window: int | None = None,
    sinks: int = 0,
    validate: bool = True,
) -> torch.Tensor:
    """Attention over HiF8 pages for any number of query tokens per request.

    ``query`` is ``[T, Hq, D]`` in the TND layout; request b owns the next
    ``query_lens[b]`` rows, which are the last positions of its
    ``seq_lens[b]`` cached tokens (this step's cache write included), and with
    ``causal`` row i sees keys ``0 .. seq_lens[b] - query_lens[b] + i`` - the
    contract of ``paged_attention_reference`` with ``query_lens``
    (kv_cache.py:314-372) and of the reference's TND attention call
    (kv_runtime.py:1470-1563).  Returns ``[T, Hq, Dv]``.

    The request split comes from ``query_lens`` (host integers, as the
    reference's oracle takes them; rows must add up to T) or from
    ``query_start_loc`` (an int32 device tensor ``[B + 1]``, the cumulative
    form of the reference's ``actual_seq_lengths_q`` with a leading 0; pass
    ``max_query_len`` to avoid a host synchronisation, and ``validate=False``
    as well, since validation checks it against ``query_start_loc``).  One
    query row per request runs the decode kernel; otherwise the multi-token
    kernel.

    ``window`` (no counterpart in the reference; causal calls) makes the row at
    position P see the rows ``t <= P`` with ``t > P - window`` or ``t < sinks``
    alone: a sliding window, and first tokens that stay visible.  Pages that no row
    sees are not read, so :func:`release_blocks` may have taken them.  K and V are
    then ``dec(code) * row scale`` without a rounding to the query dtype, what a
    row does not see has no influence on it, NaN and infinities included, and a
    row that sees nothing gets zeros, as do rows that ``query_start_loc`` gives to
    no request.  Small weights beside an infinite V, and the shapes that are
    fast, are those of :func:`tree_attention`.
    """
    _check_caches(key_cache, value_cache)
    window, sinks = _check_window(window, sinks)
    if window is not None and not causal:
        raise ValueError("a window needs causal attention")
    if query.ndim != 3:
        raise ValueError("query must have shape [tokens, num_heads, head_size]")
    if query.shape[1] % key_cache.shape[2]:
        raise ValueError("num_heads must be divisible by num_kv_heads")
    if (query_lens is None) == (query_start_loc is None):
        raise ValueError("pass exactly one of query_lens and query_start_loc")
    tokens = query.shape[0]
    if query_lens is not None:
        q_lengths = [int(v) for v in query_lens]
        if any(v < 0 for v in q_lengths) or sum(q_lengths) != tokens:
            raise ValueError("query_lens must describe every query row")
        batch = len(q_lengths)
        if not isinstance(seq_lens, torch.Tensor):
            lengths = [int(v) for v in seq_lens]
            if len(lengths) != batch:
                raise ValueError("one sequence length is required per request")
            for q_len, kv_len in zip(q_lengths, lengths):
                if q_len and kv_len < q_len:
                    raise ValueError(
                        "HIF8 post-update KV length cannot be shorter than its query "
                        f"length, got q={q_len}, kv={kv_len}")
        if batch == tokens and all(v == 1 for v in q_lengths):
            # The decode case: each row is its request's last position.
            return paged_decode_attention(query, key_cache, value_cache, block_table, seq_lens, scale=scale,
                                          max_seq_len=max_seq_len, window=window, sinks=sinks, validate=validate)
        starts = [0]
        for v in q_lengths:
            starts.append(starts[-1] + v)
        loc = torch.tensor(starts, dtype=torch.int32).to(query.device)
        if max_query_len is None:
            max_query_len = max(q_lengths, default=0)
    else:
        if query_start_loc.ndim != 1 or query_start_loc.numel() < 1:
            raise ValueError("query_start_loc must have shape [batch + 1]")
        batch = query_start_loc.numel() - 1
        loc = query_start_loc.to(device=query.device, dtype=torch.int32).contiguous()
        if max_query_len is None:
            max_query_len = int((loc[1:] - loc[:-1]).max().item()) if batch else 0
    if block_table.ndim != 2 or block_table.shape[0] < batch:
        raise ValueError("block_table must have shape [batch, max_blocks]")
    block_size = key_cache.shape[1]
    if isinstance(seq_lens, torch.Tensor):
        lens_dev = seq_lens.to(device=query.device, dtype=torch.int32).contiguous()
        if lens_dev.numel() < batch:
            raise ValueError("one sequence length is required per request")
        if max_seq_len is None:
            max_seq_len = int(lens_dev[:batch].max().item()) if batch else 0
    else:
        lengths = [int(v) for v in seq_lens]
        if len(lengths) != batch:
            raise ValueError("one sequence length is required per request")
        if any(v < 0 for v in lengths):
            raise ValueError("sequence lengths must be non-negative")
        lens_dev = torch.tensor(lengths, dtype=torch.int32).to(query.device)
        if max_seq_len is None:
            max_seq_len = max(lengths, default=0)
    if max_seq_len > block_table.shape[1] * block_size:
        raise ValueError("block_table has too few entries for a sequence length")
    table = block_table[:batch]
    if table.dtype not in (torch.int32, torch.int64):
        table = table.to(torch.int64)
    table = table.to(query.device).contiguous()
    if validate and batch:
        # A max_query_len below the longest request would leave that request's
        # later rows unwritten (the grid is sized by it).
        longest = int((loc[1:batch + 1] - loc[:batch]).max().item())
        if longest > max_query_len:
            raise ValueError(f"max_query_len ({max_query_len}) is smaller than a request's query length ({longest})")
    if validate and batch and max_seq_len > 0:
        if bool((lens_dev[:batch] > max_seq_len).any()):
            raise ValueError("max_seq_len is smaller than a sequence length")
        needed = (max_seq_len + block_size - 1) // block_size
        used = (torch.arange(needed, device=query.device)[None, :] * block_size
                < lens_dev[:batch, None].to(torch.int64))
        if window is not None:
            used &= _pages_in_window(lens_dev[:batch], loc[1:] - loc[:-1], needed, block_size, window, sinks)
        ids = table[:, :needed].to(torch.int64)
        if bool(((ids < 0) | (ids >= key_cache.shape[0]))[used].any()):
            raise IndexError("block_table references a block outside the cache")
    extension = native.load_extension()
    if window is not None:
        return native._operator("hif8_window_attention", extension)(
            query.contiguous(), key_cache, value_cache, table, loc, lens_dev, float(scale), window, sinks,
            int(max_query_len), int(max_seq_len))
    return native._operator("hif8_paged_prefill_attention", extension)(
        query.contiguous(), key_cache, value_cache, table, loc, lens_dev, float(scale), int(max_query_len),
        int(max_seq_len), bool(causal))


def _as_int32(t: torch.Tensor, device) -> torch.Tensor:
    """``t`` as a contiguous int32 tensor on ``device``; itself where it is one (the usual call: no copy, few checks)."""
    if t.dtype is torch.int32 and t.device == device and t.is_contiguous():
        return t
    if t.dtype is torch.int64:   # a count past int32 ("all of them") must not wrap
        t = t.clamp(-(1 << 31), (1 << 31) - 1)
    return t.to(device=device, dtype=torch.int32).contiguous()


def _device_lengths(lens, name: str, device) -> tuple[torch.Tensor, list[int] | None]:
    """Request lengths as an int32 device tensor, and as host integers where they came so."""
    if isinstance(lens, torch.Tensor):
        return _as_int32(lens, device), None
    host = [int(v) for v in lens]
    if any(v < 0 for v in host):
        raise ValueError(f"{name} must be non-negative")
    return torch.tensor(host, dtype=torch.int32).to(device), host


def _device_table(block_table: torch.Tensor, batch: int, device) -> torch.Tensor:
    if block_table.ndim != 2 or block_table.shape[0] < batch:
        raise ValueError("block_table must have shape [batch, max_blocks]")
    if block_table.shape[0] == batch and block_table.device == device and block_table.is_contiguous() and \
            block_table.dtype in (torch.int32, torch.int64):
        return block_table
    table = block_table[:batch]
    if table.dtype not in (torch.int32, torch.int64):
        table = table.to(torch.int64)
    return table.to(device).contiguous()


def _request_rows(query, query_lens, query_start_loc, max_query_len, validate: bool):
    """(query_start_loc on the device, batch, max_query_len, host query lengths or None)."""
    if (query_lens is None) == (query_start_loc is None):
        raise ValueError("pass exactly one of query_lens and query_start_loc")
    if query_lens is not None:
        host = [int(v) for v in query_lens]
        if any(v < 0 for v in host) or sum(host) != query.shape[0]:
            raise ValueError("query_lens must describe every query row")
        loc = torch.tensor([0] + host, dtype=torch.int32).cumsum(0, dtype=torch.int32).to(query.device)
        longest = max(host, default=0)
        if max_query_len is None:
            max_query_len = longest
        elif max_query_len < longest:
            raise ValueError(f"max_query_len ({max_query_len}) is smaller than a request's query length ({longest})")
        return loc, len(host), int(max_query_len), host
    if query_start_loc.ndim != 1 or query_start_loc.numel() < 1:
        raise ValueError("query_start_loc must have shape [batch + 1]")
    loc = _as_int32(query_start_loc, query.device)
    batch = loc.shape[0] - 1
    if max_query_len is None or (validate and batch):
        longest = int((loc[1:] - loc[:-1]).max().item()) if batch else 0
        if max_query_len is None:
            max_query_len = longest
        elif longest > max_query_len:
            raise ValueError(f"max_query_len ({max_query_len}) is smaller than a request's query length ({longest})")
    return loc, batch, int(max_query_len), None


def _check_pages(lens: torch.Tensor, table: torch.Tensor, max_seq_len: int, block_size: int, blocks: int) -> None:
    """Host check of what the kernels only skip: lengths past max_seq_len, block ids outside the cache."""
    if not lens.numel() or max_seq_len <= 0:
        if lens.numel() and bool((lens > max_seq_len).any()):
            raise ValueError("max_seq_len is smaller than a sequence length")
        return
    if bool((lens > max_seq_len).any()):
        raise ValueError("max_seq_len is smaller than a sequence length")
    needed = (max_seq_len + block_size - 1) // block_size
    used = torch.arange(needed, device=table.device)[None, :] * block_size < lens[:, None].to(torch.int64)
    ids = table[:, :needed].to(torch.int64)
    if bool(((ids < 0) | (ids >= blocks))[used].any()):
        raise IndexError("block_table references a block outside the cache")


def tree_attention(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    context_lens: Sequence[int] | torch.Tensor,
    tree_mask: torch.Tensor,
    *,
    scale: float,
    query_lens: Sequence[int] | None = None,
    query_start_loc: torch.Tensor | None = None,
    max_query_len: int | None = None,
    max_seq_len: int | None = None,
    validate: bool = True,
) -> torch.Tensor:
    """Attention of a tree of drafted tokens per request: ``query`` ``[T, Hq, D]`` -> ``[T, Hq, Dv]``.

    No counterpart in the reference: the verification step of speculative
    decoding.  Request b has ``context_lens[b]`` cached tokens and
    ``query_lens[b]`` drafts, whose K and V :func:`write_kv_cache` has put
    behind them, at cache rows ``context_lens[b] + j``.  Draft i sees every
    context row and the drafts j of its request where ``tree_mask[row, j]``
    (bool or uint8, ``[T, at least max_query_len]``) is set: its ancestors and,
    usually, itself.  A draft that sees nothing gets zeros, and so do rows that
    ``query_start_loc`` gives to no request (a padded batch); what is not seen
    has no influence, NaN and infinities included.
    Weights are float32 numbers and have 16 bits beside V: a weight below 2^-31
    of its row's largest may count as zero, and an infinite V under it then gives
    NaN instead of an infinity.

    Head sizes 64, 128 and 256 (K and V alike) over pages of a multiple of 16
    rows, with a query that starts at a multiple of 16 bytes, run on the matrix
    cores.  Every other call takes a kernel for any shape (float32 throughout),
    which is many times slower: 8 requests of 16 drafts over 4096 rows take
    50 us with heads of 256 and 1.8 ms with heads of 96.

    The request split is given as for :func:`paged_attention`.  ``max_seq_len``
    bounds ``context_lens[b] + query_lens[b]``; with device tensors pass it and
    ``max_query_len`` and ``validate=False`` to avoid host synchronisations.
    """
    _check_caches(key_cache, value_cache)
    if query.ndim != 3:
        raise ValueError("query must have shape [tokens, num_heads, head_size]")
    if query.shape[1] % key_cache.shape[2]:
        raise ValueError("num_heads must be divisible by num_kv_heads")
    if tree_mask.dtype not in (torch.bool, torch.uint8):
        raise TypeError(f"tree_mask must be bool or uint8, got {tree_mask.dtype}")
    loc, batch, max_query_len, _ = _request_rows(query, query_lens, query_start_loc, max_query_len, validate)
    if tree_mask.ndim != 2 or tree_mask.shape[0] != query.shape[0] or tree_mask.shape[1] < max_query_len:
        raise ValueError("tree_mask must have shape [tokens, at least max_query_len]")
    lens, host = _device_lengths(context_lens, "context_lens", query.device)
    if lens.ndim != 1 or (lens.numel() < batch if host is None else lens.numel() != batch):
        raise ValueError("one context length is required per request")
    total = lens[:batch] + (loc[1:] - loc[:-1]) if max_seq_len is None or validate else None
    if max_seq_len is None:
        max_seq_len = int(total.max().item()) if batch else 0
    if max_seq_len > block_table.shape[1] * key_cache.shape[1]:
        raise ValueError("block_table has too few entries for a sequence length")
    table = _device_table(block_table, batch, query.device)
    if validate and batch:
        _check_pages(total, table, max_seq_len, key_cache.shape[1], key_cache.shape[0])
    extension = native.load_extension()
    return native._operator("hif8_tree_attention", extension)(
        query.contiguous(), key_cache, value_cache, table, loc, lens,
        tree_mask if tree_mask.device == query.device and tree_mask.is_contiguous() else
        tree_mask.to(query.device).contiguous(),
        float(scale), max_query_len, int(max_seq_len))


def accept_drafts(
    key_caches: torch.Tensor | Sequence[torch.Tensor],
    value_caches: torch.Tensor | Sequence[torch.Tensor],
    block_table: torch.Tensor,
    context_lens: Sequence[int] | torch.Tensor,
    accepted: torch.Tensor,
    accepted_counts: Sequence[int] | torch.Tensor,
    *,
    validate: bool = True,
) -> torch.Tensor:
    """Moves the rows of accepted drafts to the end of each request's context, in place.

    No counterpart in the reference; follows :func:`tree_attention`.  Row
    ``context_lens[b] + accepted[b, i]`` of every cache moves to row
    ``context_lens[b] + i`` for ``i < accepted_counts[b]``.  ``accepted``
    (int32, ``[B, width]``) lists draft indices in strictly rising order, the
    path from the root (every parent precedes its children).  The caches are
    one layer's pair or the pairs of all layers, which share ``block_table``
    and no memory; all move in one launch.  Returns the new lengths, int32 ``[B]``, on the
    device.  The pages must belong to one request each.

    ``validate`` checks counts, order and pages on the host.
    """
    keys = [key_caches] if isinstance(key_caches, torch.Tensor) else list(key_caches)
    values = [value_caches] if isinstance(value_caches, torch.Tensor) else list(value_caches)
    if not keys or len(keys) != len(values):
        raise ValueError("accept_drafts needs a value cache for every key cache")
    if validate:  # the operator checks each cache in any case
        for k, v in zip(keys, values):
            _check_caches(k, v)
            if k.shape[:2] != keys[0].shape[:2]:
                raise ValueError("all caches must have the same blocks")
    device = keys[0].device
    if accepted.ndim != 2:
        raise ValueError("accepted must have shape [batch, width]")
    if accepted.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"accepted must be int32 or int64, got {accepted.dtype}")
    batch, width = accepted.shape
    lens, host = _device_lengths(context_lens, "context_lens", device)
    counts, _ = _device_lengths(accepted_counts, "accepted_counts", device)
    if lens.ndim != 1 or lens.numel() < batch or (host is not None and len(host) != batch):
        raise ValueError("one context length is required per request")
    if counts.ndim != 1 or counts.numel() < batch:
        raise ValueError("one accepted count is required per request")
    path = _as_int32(accepted, device)
    table = _device_table(block_table, batch, device)
    if validate and batch:
        live = torch.arange(width, device=device) < counts[:batch, None]
        if bool((counts[:batch] > width).any()) or bool((counts[:batch] < 0).any()):
            raise ValueError("accepted_counts must be within the width of accepted")
        before = torch.nn.functional.pad(path, (1, 0), value=-1)[:, :-1]
        if bool(((path <= before) & live).any()):
            raise ValueError("accepted must list draft indices in strictly rising order")
        if width:
            last = (torch.where(live, path, -1).amax(dim=1) + 1 + lens[:batch]).to(torch.int32)
            most = int(last.max().item())
            if most > table.shape[1] * keys[0].shape[1]:
                raise ValueError("block_table has too few entries for an accepted draft")
            _check_pages(last, table, most, keys[0].shape[1], keys[0].shape[0])
    extension = native.load_extension()
    return native._operator("hif8_accept_drafts", extension)(keys + values, table, lens, path, counts)


def paged_decode_attention_weights(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int] | torch.Tensor,
    key_weights: torch.Tensor,
    *,
    scale: float,
    accumulate: bool = True,
    max_seq_len: int | None = None,
    validate: bool = True,
) -> torch.Tensor:
    """:func:`paged_decode_attention` that also keeps the weight every cached row got.

    No counterpart in the reference; feeds :func:`evict_kv_rows`.
    ``key_weights`` (float32 ``[B, Hkv, at least max_seq_len]``, contiguous)
    receives, in place, the sum of the row's softmax weights over the query
    heads of each KV head: added, or stored with ``accumulate=False``.  Entries
    from ``seq_lens[b]`` on are left as they were.  What :func:`tree_attention` says of
    small weights beside an infinite V, and of the shapes that are fast, holds
    here too.
    """
    _check_caches(key_cache, value_cache)
    if query.ndim != 3:
        raise ValueError("query must have shape [tokens, num_heads, head_size]")
    batch = query.shape[0]
    if query.shape[1] % key_cache.shape[2]:
        raise ValueError("num_heads must be divisible by num_kv_heads")
    lens, table, max_seq_len = _weighted_request(key_cache, block_table, seq_lens, key_weights, batch, max_seq_len,
                                                 validate)
    extension = native.load_extension()
    return native._operator("hif8_paged_decode_attention_weights", extension)(
        query.contiguous(), key_cache, value_cache, table, lens, key_weights, float(scale), max_seq_len,
        bool(accumulate))


def _weighted_request(key_cache, block_table, seq_lens, key_weights, batch: int, max_seq_len, validate: bool):
    """The checks that the calls with ``key_weights`` share: (seq_lens, block table, max_seq_len)."""
    if key_weights.dtype != torch.float32:
        raise TypeError(f"key_weights must be float32, got {key_weights.dtype}")
    if not key_weights.is_contiguous():
        raise ValueError("key_weights must be contiguous")
    lens, host = _device_lengths(seq_lens, "sequence lengths", key_cache.device)
    if lens.ndim != 1 or (lens.numel() < batch if host is None else lens.numel() != batch):
        raise ValueError("one sequence length is required per request")
    if lens.shape[0] != batch:
        lens = lens[:batch]
    if max_seq_len is None:
        max_seq_len = (max(host, default=0) if host is not None else int(lens.max().item())) if batch else 0
    if max_seq_len > block_table.shape[1] * key_cache.shape[1]:
        raise ValueError("block_table has too few entries for a sequence length")
    if key_weights.ndim != 3 or key_weights.shape[0] < batch or key_weights.shape[1] != key_cache.shape[2] or \
            key_weights.shape[2] < max_seq_len:
        raise ValueError("key_weights must have shape [batch, num_kv_heads, at least max_seq_len]")
    table = _device_table(block_table, batch, key_cache.device)
    if validate and batch:
        _check_pages(lens, table, int(max_seq_len), key_cache.shape[1], key_cache.shape[0])
    return lens, table, int(max_seq_len)


def accumulate_key_weights(
    query: torch.Tensor,
    key_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int] | torch.Tensor,
    key_weights: torch.Tensor,
    *,
    scale: float,
    query_lens: Sequence[int] | None = None,
    query_start_loc: torch.Tensor | None = None,
    causal: bool = True,
    accumulate: bool = True,
    max_query_len: int | None = None,
    max_seq_len: int | None = None,
    validate: bool = True,
) -> None:
    """Adds up the softmax weight that many query rows give every cached row, in place.

    The multi-row form of :func:`paged_decode_attention_weights`, for a prompt
    (or the last rows of one) before :func:`evict_kv_rows`; it reads the key
    cache alone and returns nothing.  Request b's query rows are the last
    positions of its ``seq_lens[b]`` cached tokens, given and masked as in
    :func:`paged_attention`.  ``key_weights`` as there; with
    ``accumulate=False`` the sums are stored instead of added.  Shapes that are
    fast as in :func:`tree_attention` (of K alone): a prompt of 1024 takes 46 us with
    heads of 256 and 33 ms with heads of 96.
    """
    if key_cache.dtype != torch.uint8 or key_cache.ndim != 4:
        raise TypeError("key_cache must be a 4-D uint8 tensor")
    if not key_cache.is_contiguous():
        raise ValueError("key_cache must be contiguous")
    if query.ndim != 3:
        raise ValueError("query must have shape [tokens, num_heads, head_size]")
    if query.shape[1] % key_cache.shape[2]:
        raise ValueError("num_heads must be divisible by num_kv_heads")
    loc, batch, max_query_len, _ = _request_rows(query, query_lens, query_start_loc, max_query_len, validate)
    lens, table, max_seq_len = _weighted_request(key_cache, block_table, seq_lens, key_weights, batch, max_seq_len,
                                                 validate)
    extension = native.load_extension()
    native._operator("hif8_key_weights", extension)(
        query.contiguous(), key_cache, table, loc, lens, key_weights, float(scale), max_query_len, max_seq_len,
        bool(causal), bool(accumulate))


def evict_kv_rows(
    key_cache: torch.Tensor,
    value_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: Sequence[int] | torch.Tensor,
    key_weights: torch.Tensor,
    keep: int | Sequence[int] | torch.Tensor,
    *,
    positions: torch.Tensor | None = None,
    sinks: int = 0,
    protect_from: Sequence[int] | torch.Tensor | None = None,
    max_seq_len: int | None = None,
    validate: bool = True,
) -> torch.Tensor:
    """Cuts each request's cache to its ``keep`` rows of largest accumulated weight, in place.

    No counterpart in the reference.  Every KV head keeps its own rows:
    protected ones first (position below ``sinks``, or from ``protect_from[b]``
    on), then by falling ``key_weights``, NaN last, ties by the lower row.
    With ``n = min(seq_lens[b], keep)`` the r-th dropped row before row n
    receives the r-th kept row from row n on - codes, scale, weight and
    position - and the other kept rows stay where they are, so attention over
    the first n rows is attention over the kept ones.  Weights from row n to
    the old length become zero.

    ``positions`` (int32, the shape of ``key_weights``) holds each row's
    position in the sequence and moves along; without it a row's index counts
    as its position, as in a cache that was never cut.  Returns the new
    lengths, int32 ``[B]``, on the device.  The pages must belong to one request.
    """
    _check_caches(key_cache, value_cache)
    batch = len(seq_lens) if not isinstance(seq_lens, torch.Tensor) else seq_lens.numel()
    lens, table, max_seq_len = _weighted_request(key_cache, block_table, seq_lens, key_weights, batch, max_seq_len,
                                                 validate)
    if positions is not None:
        if positions.dtype != torch.int32 or positions.shape != key_weights.shape:
            raise TypeError("positions must be int32 with the shape of key_weights")
        if not positions.is_contiguous():
            raise ValueError("positions must be contiguous")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    keep_each, keep_all = None, 0
    if isinstance(keep, int):
        keep_all = keep
    else:
        keep_each, _ = _device_lengths(keep, "keep", key_cache.device)
        if keep_each.ndim != 1 or keep_each.numel() < batch:
            raise ValueError("one keep count is required per request")
    if keep_all < 0 or (validate and keep_each is not None and bool((keep_each < 0).any())):
        raise ValueError("keep must not be negative")
    if protect_from is not None:
        protect_from = _as_int32(torch.as_tensor(protect_from), key_cache.device)
        if protect_from.ndim != 1 or protect_from.numel() < batch:
            raise ValueError("one protect_from position is required per request")
    extension = native.load_extension()
    return native._operator("hif8_kv_evict", extension)(
        key_cache, value_cache, table, lens, key_weights, positions, keep_each, int(keep_all), int(sinks),
        protect_from, max_seq_len)



def verify_drafts(
    target_probs: torch.Tensor,
    draft_tokens: torch.Tensor,
    uniforms: torch.Tensor,
    *,
    draft_probs: torch.Tensor | None = None,
    parents: torch.Tensor | None = None,
    query_lens: Sequence[int] | None = None,
    query_start_loc: torch.Tensor | None = None,
    max_query_len: int | None = None,
    validate: bool = True,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accepts drafted tokens against the target model's probabilities and draws the next token.

    No counterpart in the reference; stands between attention over the drafts and
    :func:`accept_drafts`.  Row i of a request is a node of its drafts:
    ``draft_tokens`` (int32 / int64 ``[T]``) its token, row i of ``target_probs``
    (float32 ``[T, vocab]``) what the target gives for the token behind it,
    ``uniforms`` (float32 ``[T]``, in [0, 1)) its random number.  Row 0 holds the
    token that the step before answered with, which stands.

    * Drafts drawn from a draft model, in a chain: ``draft_probs`` (float32 ``[T,
      vocab]``), row i what token i was drawn from (row 0 is not read).  Row i + 1
      is accepted after row i where ``u * q(x) < p(x)`` with its own u, q and x; the
      next token comes from ``max(p - q, 0)`` at the row that is not followed, or
      from p behind the last.
    * Given drafts (``draft_probs`` None), in a chain or, by ``parents`` (int32
      ``[T]``, index within the request, below the row's own), in a tree: the
      children of the accepted row in rising order, each accepted where
      ``u * rest < p(x)``, rest being 1 less the p of the tokens refused before it;
      the next token comes from p without the refused tokens.

    Either way the answers are distributed as the target's.  The next token is
    the first v at which the running sum passes u of row 0 times its total; all of
    it in float64.  Returns ``accepted`` (int32 ``[B, max_query_len]``: the path's
    rows in rising order, then -1) and ``accepted_counts`` (int32 ``[B]``), which
    :func:`accept_drafts` takes, and the next tokens (int64 ``[B]``).  A request
    without rows gets 0 and -1, one whose probabilities hold no positive finite
    number -1.

    The request split is given as for :func:`paged_attention`, at most 1024 rows
    each.  ``validate`` checks parents and numbers on the host.
    """
    if target_probs.ndim != 2 or target_probs.shape[1] < 1:
        raise ValueError("target_probs must have shape [tokens, vocab]")
    if target_probs.dtype != torch.float32:
        raise TypeError(f"target_probs must be float32, got {target_probs.dtype}")
    tokens, device = target_probs.shape[0], target_probs.device
    if draft_tokens.shape != (tokens,) or draft_tokens.dtype not in (torch.int32, torch.int64):
        raise ValueError("draft_tokens must hold one int32 or int64 id per row of target_probs")
    if uniforms.shape != (tokens,) or uniforms.dtype != torch.float32:
        raise ValueError("uniforms must hold one float32 number per row of target_probs")
    if draft_probs is not None:
        if parents is not None:
            raise ValueError("draft_probs go with a chain of drafts, not with parents")
        if draft_probs.shape != target_probs.shape or draft_probs.dtype != torch.float32:
            raise ValueError("draft_probs must be float32 with the shape of target_probs")
    if parents is not None and (parents.shape != (tokens,) or parents.dtype not in (torch.int32, torch.int64)):
        raise ValueError("parents must hold one int32 or int64 index per row of target_probs")
    loc, batch, max_query_len, _ = _request_rows(target_probs, query_lens, query_start_loc, max_query_len, validate)
    if max_query_len > 1024:
        raise ValueError("verify_drafts takes at most 1024 rows per request")

    def rows(probs):
        probs = probs.to(device)
        return probs if tokens == 0 or (probs.stride(1) == 1 and probs.stride(0) >= probs.shape[1]) else probs.contiguous()

    up = None if parents is None else _as_int32(parents, device)
    drawn = uniforms.to(device).contiguous()
    if validate and tokens:
        if bool(((drawn < 0) | (drawn >= 1) | drawn.isnan()).any()):
            raise ValueError("uniforms must be in [0, 1)")
        if up is not None and batch:
            row = torch.arange(tokens, device=device)
            request = torch.searchsorted(loc.contiguous(), row, right=True, out_int32=True).long() - 1
            inside = (request >= 0) & (request < batch)
            index = row - loc.long()[request.clamp(0, batch - 1)]
            if bool((inside & (index > 0) & ((up < 0) | (up >= index))).any()):
                raise ValueError("parents must be indices below the row's own")
    extension = native.load_extension()
    return native._operator("hif8_verify_drafts", extension)(
        rows(target_probs), draft_tokens.to(device).contiguous(), drawn, loc,
        None if draft_probs is None else rows(draft_probs), up, max_query_len)


def _check_pool(block_table, free_blocks, free_count, lens, lens_name: str, block_size: int, validate: bool):
    """The checks that the calls with a stack of free pages share: the lengths on the device."""
    device = block_table.device
    if block_table.ndim != 2 or block_table.shape[1] < 1:
        raise ValueError("block_table must have shape [batch, max_blocks]")
    if block_table.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"block_table must be int32 or int64, got {block_table.dtype}")
    if free_blocks.ndim != 1 or free_blocks.dtype != torch.int32:
        raise TypeError("free_blocks must be an int32 tensor [pages]")
    if free_count.numel() != 1 or free_count.dtype != torch.int32:
        raise TypeError("free_count must be an int32 tensor of one element")
    for name, t in (("block_table", block_table), ("free_blocks", free_blocks), ("free_count", free_count)):
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous")
        if t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")
    if block_size < 1:
        raise ValueError("block_size must be positive")
    batch = block_table.shape[0]
    sizes, host = _device_lengths(lens, lens_name, device)
    if sizes.ndim != 1 or (sizes.numel() < batch if host is None else sizes.numel() != batch):
        raise ValueError("one length is required per request")
    if validate:
        if not 0 <= int(free_count.item()) <= free_blocks.numel():
            raise ValueError("free_count must be within free_blocks")
        if bool((sizes[:batch] < 0).any()):
            raise ValueError(f"{lens_name} must be non-negative")
    return sizes


def extend_block_tables(
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    free_count: torch.Tensor,
    context_lens: Sequence[int] | torch.Tensor,
    *,
    block_size: int,
    query_lens: Sequence[int] | None = None,
    query_start_loc: torch.Tensor | None = None,
    total_query_tokens: int | None = None,
    validate: bool = True,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """Takes pages for a step's new tokens, in place, and works out the tokens' slots on the device.

    No counterpart in the reference (its scheduler builds both on the host).
    Request b has ``context_lens[b]`` cached tokens and ``query_lens[b]`` new
    ones.  Every column of its row of ``block_table`` (int32 / int64 ``[B,
    max_blocks]``, an entry below zero holds no page) that the new tokens reach
    without finding a page gets one from the end of the stack ``free_blocks[:
    free_count]`` (int32; the count int32 of one element, on the device), in the
    order (request, column).  Table and count change in place.

    Returns ``slot_mapping`` (int64 ``[T]``, for :func:`write_kv_cache`; -1 where
    there is no page) and ``positions`` (int64 ``[T]``), both -1 for rows that
    ``query_start_loc`` gives to no request, the new ``seq_lens`` (int32 ``[B]``)
    and ``missing`` (int32 ``[B]``): columns that got no page, because the stack was
    empty or the table too narrow.

    With ``query_start_loc`` pass ``total_query_tokens`` (the rows T of the step) and
    ``validate=False`` to avoid host synchronisations.
    """
    context = _check_pool(block_table, free_blocks, free_count, context_lens, "context_lens", block_size, validate)
    if (query_lens is None) == (query_start_loc is None):
        raise ValueError("pass exactly one of query_lens and query_start_loc")
    if query_lens is not None:
        host = [int(v) for v in query_lens]
        if any(v < 0 for v in host):
            raise ValueError("query_lens must be non-negative")
        loc = torch.tensor([0] + host, dtype=torch.int64).cumsum(0).to(torch.int32).to(block_table.device)
        if total_query_tokens is None:
            total_query_tokens = sum(host)
    else:
        if query_start_loc.ndim != 1 or query_start_loc.numel() < 1:
            raise ValueError("query_start_loc must have shape [batch + 1]")
        loc = _as_int32(query_start_loc, block_table.device)
        if total_query_tokens is None:
            total_query_tokens = int(loc[-1].item())
    if loc.numel() - 1 != block_table.shape[0]:
        raise ValueError("block_table must have a row for every request")
    if total_query_tokens < 0:
        raise ValueError("total_query_tokens must not be negative")
    extension = native.load_extension()
    return native._operator("hif8_extend_block_tables", extension)(
        block_table, free_blocks, free_count, context, loc, int(block_size), int(total_query_tokens))


def release_blocks(
    block_table: torch.Tensor,
    free_blocks: torch.Tensor,
    free_count: torch.Tensor,
    seq_lens: Sequence[int] | torch.Tensor,
    *,
    block_size: int,
    window: int | None = None,
    sinks: int = 0,
    validate: bool = True,
) -> None:
    """Gives pages that no later token needs back to the stack of free pages, in place.

    No counterpart in the reference; the way back of :func:`extend_block_tables`, after
    :func:`verify_drafts` or :func:`evict_kv_rows` has shortened requests, or a
    window has moved on.  A page stays where request b's ``seq_lens[b]`` tokens
    reach it and, with ``window``, where it holds one of the first ``sinks`` tokens
    or one that the next token sees.  The others leave ``block_table`` (their entries
    become -1) for the end of ``free_blocks``, in the order (request, column);
    length 0 gives back all of a request.  Pages must belong to one request.
    """
    window, sinks = _check_window(window, sinks)
    lens = _check_pool(block_table, free_blocks, free_count, seq_lens, "seq_lens", block_size, validate)
    extension = native.load_extension()
    native._operator("hif8_release_blocks", extension)(
        block_table, free_blocks, free_count, lens, int(block_size), 0 if window is None else window, int(sinks))


__all__ = [
    "HIF8_CACHE_DTYPE",
    "HIF8_SCALE_BYTES",
    "Hif8KVCacheLayout",
    "accept_drafts",
    "accumulate_key_weights",
    "evict_kv_rows",
    "extend_block_tables",
    "pack_kv_rows",
    "paged_attention",
    "paged_decode_attention",
    "paged_decode_attention_weights",
    "release_blocks",
    "tree_attention",
    "unpack_kv_rows",
    "verify_drafts",
    "write_kv_cache",
]
