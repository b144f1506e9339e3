"""New lengths written over the old ones, which other workgroups have yet to read, are refused (CPU)."""

import ctypes

import pytest

from test_abi import LIB

P, I, L, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t
AT, BATCH = 4096, 6


@pytest.fixture(scope="module")
def lib():
    if not LIB.exists():
        pytest.fail(f"{LIB} is not built; run __graft_entry__.build()")
    lib = ctypes.CDLL(str(LIB))
    lib.hif8_last_error.restype = ctypes.c_char_p
    return lib


@pytest.mark.parametrize("at", [AT, AT + 4, AT - 4, AT + 4 * (BATCH - 1), AT - 4 * (BATCH - 1)])
def test_lengths_in_place_are_refused(lib, at):
    p = P(256)
    f = lib.hif8_extend_block_tables
    f.argtypes = [P, I, L, P, L, P, P, P, L, L, L, P, P, P, P, P]
    assert f(p, 0, 8, p, 10, p, P(AT), p, BATCH, 9, 16, p, p, P(at), p, None) == 1
    assert b"seq_lens must not overlap" in lib.hif8_last_error()
    f = lib.hif8_accept_drafts
    f.argtypes = [P, P, L, L, L, P, I, L, P, P, L, P, L, P, P]
    caches, sizes = (P * 1)(1 << 20), (L * 1)(256)
    assert f(caches, sizes, 1, 4, 16, p, 0, 8, P(AT), p, 4, p, BATCH, P(at), None) == 1
    assert b"new_lens must not overlap" in lib.hif8_last_error()
    f = lib.hif8_kv_evict
    f.argtypes = [P, P, L, L, L, L, L, P, I, L, P, L, L, P, P, L, P, L, L, P, P, P, Z, P]
    assert f(p, p, 4, 16, 2, 64, 64, p, 0, 8, P(AT), BATCH, 100, p, None, 100, None, 10, 0, None, P(at), p, 1 << 30, None) == 1
    assert b"new_lens must not overlap" in lib.hif8_last_error()
