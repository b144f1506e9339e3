"""Refusals and workspaces of the operators on rows of the KV cache at the edges
of their ranges (CPU)."""

import ctypes

import pytest

from conftest import PKG_ROOT


@pytest.fixture(scope="module")
def lib():
    lib = ctypes.CDLL(str(PKG_ROOT / "hif8_rocm" / "libhif8_rocm.so"))
    lib.hif8_last_error.restype = ctypes.c_char_p
    return lib


def _p(v=256):
    return ctypes.c_void_p(v)


def test_the_padded_tree_entry_refuses_what_the_other_does(lib):
    i64, ptr, i32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int
    tree = lib.hif8_tree_attention_padded
    tree.argtypes = [ptr, i32, ptr, ptr] + [i64] * 5 + [ptr, i32, i64, ptr, ptr, ptr] + [i64] * 6 + \
        [ctypes.c_float, ptr, ptr, ctypes.c_size_t, ptr]

    def call(q=_p(), d=256, mask=_p(), mask_w=8, batch=1, total=8, mq=8, ml=500):
        return tree(q, 1, _p(), _p(), 8, 128, 4, d, 256, _p(), 0, 4, _p(), _p(), mask, mask_w, batch, 16, total, mq, ml, 0.1,
                    _p(), None, 0, None)

    for kw, code, text in [({"q": None}, 1, b"null pointer"), ({"mask": None}, 1, b"null pointer"), ({"d": 516}, 2, b"above 512"),
                           ({"ml": 513}, 1, b"block table capacity"), ({"mask_w": 7}, 1, b"tree_mask rows"),
                           ({"mq": 0}, 1, b"max_query_len"), ({"mq": -1}, 1, b"positive"), ({}, 1, b"workspace of")]:
        assert call(**kw) == code and text in lib.hif8_last_error(), (kw, lib.hif8_last_error())
    assert call(batch=0) == 0 and call(total=0) == 0


def test_workspaces_hold_no_output_per_request(lib):
    """Partial outputs are those of the workers, of which there are as many as the GPU runs at a time: more requests
    add their statistics (8 bytes per query row) and, in the decode form, their logits."""
    tree = lib.hif8_tree_attention_workspace_size
    tree.argtypes, tree.restype = [ctypes.c_int64] * 9, ctypes.c_size_t
    few, many = (tree(b, 16, 4, 256, 256, 128, 64 * b, 64, 4096) for b in (16, 256))
    assert many <= 64 << 20
    assert many - few <= 240 * (64 * 16 * 8 + 4) + 1024
    decode = lib.hif8_paged_decode_attention_weights_workspace_size
    decode.argtypes, decode.restype = [ctypes.c_int64] * 7, ctypes.c_size_t
    few, many = (decode(b, 16, 4, 256, 256, 128, 4096) for b in (256, 1024))
    assert many - few <= 768 * (16 * 4096 * 4 + 4 * 16 * 8 + 4) + 1024


def test_acceptance_without_caches_or_requests_writes_nothing(lib):
    i64, ptr, i32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int
    accept = lib.hif8_accept_drafts
    accept.argtypes = [ptr, ptr, i64, i64, i64, ptr, i32, i64, ptr, ptr, i64, ptr, i64, ptr, ptr]
    lens = (ctypes.c_int32 * 2)(7, 9)
    for caches, batch in ((0, 2), (1, 0)):
        arr, rows = (ctypes.c_void_p * 1)(256), (i64 * 1)(1040)
        assert accept(arr, rows, caches, 8, 128, _p(), 0, 4, _p(), _p(), 4, _p(), batch,
                      ctypes.cast(lens, ctypes.c_void_p), None) == 0
        assert list(lens) == [7, 9]
