"""Refusals of the operators on rows of the KV cache, their Meta shapes and their
workspaces (CPU): tree attention, acceptance of drafts, decode attention with
key weights, key weights of many rows, eviction."""

import ctypes

import pytest
import torch

from conftest import PKG_ROOT
from hif8_rocm import kv_cache, native

LIB = PKG_ROOT / "hif8_rocm" / "libhif8_rocm.so"


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(LIB))
    lib.hif8_last_error.restype = ctypes.c_char_p
    for name, n in (("hif8_tree_attention_workspace_size", 9), ("hif8_paged_decode_attention_weights_workspace_size", 7),
                    ("hif8_key_weights_workspace_size", 8), ("hif8_kv_evict_workspace_size", 3)):
        getattr(lib, name).argtypes = [ctypes.c_int64] * n + [ctypes.c_int] * (name == "hif8_key_weights_workspace_size")
        getattr(lib, name).restype = ctypes.c_size_t
    return lib


def _caches(blocks=4, page=4, hkv=2, d=16, dv=16):
    return (torch.zeros(blocks, page, hkv, d + 4, dtype=torch.uint8),
            torch.zeros(blocks, page, hkv, dv + 4, dtype=torch.uint8))


TABLE = torch.tensor([[0, 1], [2, 3]], dtype=torch.int32)


def _tree(**over):
    kc, vc = _caches()
    a = dict(query=torch.zeros(3, 4, 16, dtype=torch.bfloat16), key_cache=kc, value_cache=vc, block_table=TABLE,
             context_lens=[3, 4], tree_mask=torch.ones(3, 2, dtype=torch.bool), scale=0.25, query_lens=[1, 2])
    a.update(over)
    return kv_cache.tree_attention(**a)


@pytest.mark.parametrize("over, error, match", [
    ({"query": torch.zeros(3, 16, dtype=torch.bfloat16)}, ValueError, "tokens, num_heads"),
    ({"query": torch.zeros(3, 3, 16, dtype=torch.bfloat16)}, ValueError, "divisible"),
    ({"tree_mask": torch.ones(3, 2)}, TypeError, "bool or uint8"),
    ({"tree_mask": torch.ones(3, 1, dtype=torch.bool)}, ValueError, "tree_mask must have shape"),
    ({"tree_mask": torch.ones(2, 2, dtype=torch.bool)}, ValueError, "tree_mask must have shape"),
    ({"query_lens": [1, 1]}, ValueError, "every query row"),
    ({"query_lens": [4, -1]}, ValueError, "every query row"),
    ({"query_lens": None}, ValueError, "exactly one"),
    ({"max_query_len": 1}, ValueError, "smaller than a request's query length"),
    ({"context_lens": [3]}, ValueError, "one context length"),
    ({"context_lens": [3, -1]}, ValueError, "non-negative"),
    ({"context_lens": [3, 7]}, ValueError, "too few entries"),
    ({"max_seq_len": 9}, ValueError, "too few entries"),
    ({"max_seq_len": 5}, ValueError, "smaller than a sequence length"),
    ({"block_table": torch.tensor([[0, 1], [2, 4]], dtype=torch.int32)}, IndexError, "outside the cache"),
    ({"block_table": torch.tensor([[0, 1], [-1, 3]], dtype=torch.int32)}, IndexError, "outside the cache"),
    ({"block_table": TABLE[:1]}, ValueError, "block_table must have shape"),
    ({"key_cache": torch.zeros(4, 4, 2, 20)}, TypeError, "uint8"),
    ({"value_cache": _caches(blocks=3)[1]}, ValueError, "same blocks"),
])
def test_tree_attention_refusals(over, error, match):
    with pytest.raises(error, match=match):
        _tree(**over)


def _accept(**over):
    kc, vc = _caches()
    a = dict(key_caches=kc, value_caches=vc, block_table=TABLE, context_lens=[2, 3],
             accepted=torch.tensor([[0, 2], [1, 0]], dtype=torch.int32), accepted_counts=[2, 1])
    a.update(over)
    return kv_cache.accept_drafts(**a)


@pytest.mark.parametrize("over, error, match", [
    ({"accepted": torch.tensor([[2, 0], [1, 0]], dtype=torch.int32)}, ValueError, "strictly rising"),
    ({"accepted": torch.tensor([[1, 1], [1, 0]], dtype=torch.int32)}, ValueError, "strictly rising"),
    ({"accepted": torch.tensor([[-1, 1], [1, 0]], dtype=torch.int32)}, ValueError, "strictly rising"),
    ({"accepted": torch.tensor([0, 2], dtype=torch.int32)}, ValueError, "batch, width"),
    ({"accepted": torch.zeros(2, 2)}, TypeError, "int32 or int64"),
    ({"accepted_counts": [3, 1]}, ValueError, "within the width"),
    ({"accepted_counts": torch.tensor([-1, 1])}, ValueError, "within the width"),
    ({"accepted_counts": [2]}, ValueError, "one accepted count"),
    ({"context_lens": [2]}, ValueError, "one context length"),
    ({"context_lens": [2, 7]}, ValueError, "too few entries"),
    ({"block_table": torch.tensor([[0, 9], [2, 3]], dtype=torch.int32)}, IndexError, "outside the cache"),
    ({"key_caches": []}, ValueError, "a value cache for every key cache"),
    ({"key_caches": list(_caches())}, ValueError, "a value cache for every key cache"),
    ({"key_caches": [_caches()[0], _caches(blocks=5)[0]], "value_caches": [_caches()[1], _caches(blocks=5)[1]]},
     ValueError, "same blocks"),
])
def test_accept_drafts_refusals(over, error, match):
    with pytest.raises(error, match=match):
        _accept(**over)


def _decode(**over):
    kc, vc = _caches()
    a = dict(query=torch.zeros(2, 4, 16, dtype=torch.bfloat16), key_cache=kc, value_cache=vc, block_table=TABLE,
             seq_lens=[3, 8], key_weights=torch.zeros(2, 2, 8), scale=0.25)
    a.update(over)
    return kv_cache.paged_decode_attention_weights(**a)


WEIGHT_REFUSALS = [
    ({"key_weights": torch.zeros(2, 2, 7)}, ValueError, "key_weights must have shape"),
    ({"key_weights": torch.zeros(2, 4, 8)}, ValueError, "key_weights must have shape"),
    ({"key_weights": torch.zeros(1, 2, 8)}, ValueError, "key_weights must have shape"),
    ({"key_weights": torch.zeros(2, 2, 16)[..., ::2]}, ValueError, "contiguous"),
    ({"key_weights": torch.zeros(2, 2, 8, dtype=torch.float64)}, TypeError, "float32"),
    ({"seq_lens": [3]}, ValueError, "one sequence length"),
    ({"seq_lens": [3, -2]}, ValueError, "non-negative"),
    ({"seq_lens": [3, 9]}, ValueError, "too few entries"),
    ({"max_seq_len": 7}, ValueError, "smaller than a sequence length"),
    ({"block_table": torch.tensor([[0, 1], [2, 4]], dtype=torch.int32)}, IndexError, "outside the cache"),
]


@pytest.mark.parametrize("over, error, match", WEIGHT_REFUSALS)
def test_decode_weights_refusals(over, error, match):
    with pytest.raises(error, match=match):
        _decode(**over)


@pytest.mark.parametrize("over, error, match", WEIGHT_REFUSALS + [
    ({"query_lens": [1, 2]}, ValueError, "every query row"),
    ({"query_lens": None}, ValueError, "exactly one"),
    ({"query": torch.zeros(2, 3, 16, dtype=torch.bfloat16)}, ValueError, "divisible"),
])
def test_accumulate_key_weights_refusals(over, error, match):
    a = dict(query=torch.zeros(2, 4, 16, dtype=torch.bfloat16), key_cache=_caches()[0], block_table=TABLE,
             seq_lens=[3, 8], key_weights=torch.zeros(2, 2, 8), scale=0.25, query_lens=[1, 1])
    a.update(over)
    with pytest.raises(error, match=match):
        kv_cache.accumulate_key_weights(**a)


# The batch of an eviction is its seq_lens: one length fewer is no mistake there.
@pytest.mark.parametrize("over, error, match", [r for r in WEIGHT_REFUSALS if r[2] != "one sequence length"] + [
    ({"keep": -1}, ValueError, "keep must not be negative"),
    ({"keep": [2, -1]}, ValueError, "keep must be non-negative"),
    ({"keep": torch.tensor([2, -1])}, ValueError, "keep must not be negative"),
    ({"keep": [2]}, ValueError, "one keep count"),
    ({"sinks": -1}, ValueError, "sinks"),
    ({"protect_from": [3]}, ValueError, "one protect_from"),
    ({"positions": torch.zeros(2, 2, 8)}, TypeError, "positions must be int32"),
    ({"positions": torch.zeros(2, 2, 9, dtype=torch.int32)}, TypeError, "positions must be int32"),
])
def test_evict_refusals(over, error, match):
    kc, vc = _caches()
    a = dict(key_cache=kc, value_cache=vc, block_table=TABLE, seq_lens=[3, 8], key_weights=torch.zeros(2, 2, 8), keep=2)
    a.update(over)
    with pytest.raises(error, match=match):
        kv_cache.evict_kv_rows(**a)


def test_cpu_tensors_are_refused_by_the_operators():
    for call in (_tree, _accept, _decode):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call()


def test_meta_shapes_and_versions():
    native.load_extension()
    ops = torch.ops.vllm_ascend_hif8

    def meta(*shape, dtype=torch.int32):
        return torch.empty(*shape, dtype=dtype, device="meta")

    q, kc, vc = meta(5, 16, 256, dtype=torch.float16), meta(10, 128, 4, 260, dtype=torch.uint8), \
        meta(10, 128, 4, 132, dtype=torch.uint8)
    out = ops.hif8_tree_attention(q, kc, vc, meta(2, 4), meta(3), meta(2), meta(5, 4, dtype=torch.bool), 1.0, 4, 400)
    assert out.shape == (5, 16, 128) and out.dtype == torch.float16
    w = meta(5, 4, 512, dtype=torch.float32)
    out = ops.hif8_paged_decode_attention_weights(q, kc, vc, meta(5, 4), meta(5), w, 1.0, 500)
    assert out.shape == (5, 16, 128) and w._version == 1
    assert ops.hif8_key_weights(q, kc, meta(2, 4), meta(3), meta(2), w, 1.0, 4, 500) is None and w._version == 2
    lens = ops.hif8_accept_drafts([kc, vc], meta(2, 4), meta(2), meta(2, 3), meta(2))
    assert lens.shape == (2,) and lens.dtype == torch.int32 and kc._version == vc._version == 1
    pos = meta(5, 4, 512)
    lens = ops.hif8_kv_evict(kc, vc, meta(5, 4), meta(5), w, pos, None, 10, 0, None, 500)
    assert lens.shape == (5,) and (kc._version, vc._version, w._version, pos._version) == (2, 2, 3, 1)


def test_workspace_sizes(lib):
    # Nothing to do, or sizes that the calls refuse: none.
    assert lib.hif8_tree_attention_workspace_size(0, 16, 4, 256, 256, 128, 0, 0, 0) == 0
    assert lib.hif8_tree_attention_workspace_size(1, 15, 4, 256, 256, 128, 8, 8, 512) == 0
    assert lib.hif8_tree_attention_workspace_size(1, 16, 4, 256, 256, 128, 8, 8, 512) > 0
    # The logits of every head and cached row are kept between the two launches.
    assert lib.hif8_paged_decode_attention_weights_workspace_size(2, 16, 4, 256, 256, 128, 1000) >= 2 * 16 * 1000 * 4
    assert lib.hif8_key_weights_workspace_size(1, 16, 4, 256, 128, 32, 32, 4096, 1) >= 32 * 16 * 8
    # Two lists of at most half the rows, and a count, per KV head.
    assert lib.hif8_kv_evict_workspace_size(2, 4, 1000) == 2 * 4 * (2 * 501 + 1) * 4


def _p(v=256):
    return ctypes.c_void_p(v)


def test_c_entries_refuse_bad_arguments(lib):
    i64, ptr, i32, f32, size = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float, ctypes.c_size_t
    tree = lib.hif8_tree_attention
    tree.argtypes = [ptr, i32, ptr, ptr] + [i64] * 5 + [ptr, i32, i64, ptr, ptr, ptr] + [i64] * 6 + [f32, ptr, ptr, size, ptr]

    def call(q=_p(), dt=1, d=256, hkv=4, width=4, mask=_p(), mask_w=8, batch=1, hq=16, total=8, mq=8, ml=500, ws=None,
             nbytes=0, bt=0):
        return tree(q, dt, _p(), _p(), 8, 128, hkv, d, 256, _p(), bt, width, _p(), _p(), mask, mask_w, batch, hq, total,
                    mq, ml, 0.1, _p(), ws, nbytes, None)

    for kw, code, text in [
            ({"q": None}, 1, b"null pointer"), ({"mask": None}, 1, b"null pointer"), ({"dt": 5}, 1, b"float16 or bfloat16"),
            ({"d": 254}, 1, b"divisible by four"), ({"d": 516}, 2, b"above 512"), ({"hkv": 3}, 1, b"divisible by num_kv"),
            ({"ml": 513}, 1, b"block table capacity"), ({"mask_w": 7}, 1, b"tree_mask rows"), ({"mq": 0}, 1, b"max_query_len"),
            ({"bt": 3}, 1, b"int32 or int64"), ({}, 1, b"workspace of"), ({"total": -1}, 1, b"positive"),
            ({"ws": _p(8), "nbytes": 1 << 40}, 1, b"16-byte aligned"), ({"q": _p(1)}, 1, b"2-byte aligned")]:
        assert call(**kw) == code and text in lib.hif8_last_error(), (kw, lib.hif8_last_error())
    assert call(batch=0) == 0 and call(total=0) == 0

    evict = lib.hif8_kv_evict
    evict.argtypes = [ptr, ptr] + [i64] * 5 + [ptr, i32, i64, ptr, i64, i64, ptr, ptr, i64, ptr, i64, i64, ptr, ptr, ptr, size, ptr]

    def cut(kc=_p(), d=256, batch=1, ml=500, w=_p(), stride=512, keep=None, keep_all=10, sinks=0, ws=None, nbytes=0):
        return evict(kc, _p(), 8, 128, 4, d, 256, _p(), 0, 4, _p(), batch, ml, w, None, stride, keep, keep_all, sinks, None,
                     _p(), ws, nbytes, None)

    for kw, text in [({"kc": None}, b"null pointer"), ({"w": None}, b"null pointer"), ({"kc": _p(2)}, b"4-byte aligned"),
                     ({"d": 30}, b"divisible by four"), ({"keep_all": -1}, b"negative"), ({"sinks": -1}, b"negative"),
                     ({"stride": 499}, b"shorter than max_seq_len"), ({"ml": 513}, b"block table capacity"),
                     ({}, b"workspace of"), ({"batch": 1 << 20}, b"too large")]:
        assert cut(**kw) == 1 and text in lib.hif8_last_error(), (kw, lib.hif8_last_error())
    assert cut(batch=0) == 0

    accept = lib.hif8_accept_drafts
    accept.argtypes = [ptr, ptr, i64, i64, i64, ptr, i32, i64, ptr, ptr, i64, ptr, i64, ptr, ptr]

    def take(ptrs=(256, 256), row=1040, n=None, path=_p(), batch=1):
        arr, rows = (ctypes.c_void_p * 2)(*ptrs), (ctypes.c_int64 * 2)(row, row)
        return accept(arr, rows, 2 if n is None else n, 8, 128, _p(), 0, 4, _p(), path, 4, _p(), batch, _p(), None)

    for kw, text in [({"ptrs": (256, 0)}, b"null pointer"), ({"ptrs": (256, 258)}, b"4-byte aligned"),
                     ({"row": 1042}, b"multiple of four"), ({"path": None}, b"null pointer"), ({"n": -1}, b"positive")]:
        assert take(**kw) == 1 and text in lib.hif8_last_error(), (kw, lib.hif8_last_error())
    for ptrs in ((256, 256), (256 + 1040 * 8 * 128 - 4, 256)):   # the same cache twice, or one that ends inside another
        assert take(ptrs=ptrs) == 1 and b"must not overlap" in lib.hif8_last_error()
    assert take(batch=0) == 0 and take(n=0) == 0

    weights = lib.hif8_key_weights
    weights.argtypes = [ptr, i32, ptr] + [i64] * 4 + [ptr, i32, i64, ptr, ptr] + [i64] * 5 + [f32, i32, ptr, i64, i32, ptr, size, ptr]

    def add(q=_p(), hq=16, mq=8, ml=500, stride=512, w=_p(), ws=None, nbytes=0):
        return weights(q, 1, _p(), 8, 128, 4, 256, _p(), 0, 4, _p(), _p(), 1, hq, 8, mq, ml, 0.1, 1, w, stride, 1, ws, nbytes, None)

    for kw, text in [({"q": None}, b"null pointer"), ({"w": None}, b"null pointer"), ({"w": _p(2)}, b"4-byte aligned"),
                     ({"hq": 15}, b"divisible"), ({"mq": 0}, b"max_query_len"), ({"stride": 400}, b"shorter"), ({}, b"workspace of")]:
        assert add(**kw) == 1 and text in lib.hif8_last_error(), (kw, lib.hif8_last_error())


def test_counts_past_int32_do_not_wrap():
    t = kv_cache._as_int32(torch.tensor([1 << 40, (1 << 32) + 5, -(1 << 40), 7]), torch.device("cpu"))
    assert t.dtype == torch.int32 and t.tolist() == [(1 << 31) - 1, (1 << 31) - 1, -(1 << 31), 7]
