"""Workspace of attention within a sliding window: what the call uses, not what another kernel would (CPU)."""

import ctypes

import pytest

from test_abi import LIB

L, MIB = ctypes.c_int64, 2 ** 20


@pytest.fixture(scope="module")
def size():
    if not LIB.exists():
        pytest.fail(f"{LIB} is not built; run __graft_entry__.build()")
    f = ctypes.CDLL(str(LIB)).hif8_window_attention_workspace_size
    f.argtypes, f.restype = [L] * 11, ctypes.c_size_t
    return f


# A prompt of one request: two FP32 parts per workgroup (128 MiB at these heads) and the images of its rows,
# 33 KiB per 32 rows and KV head.
@pytest.mark.parametrize("rows", [2048, 8192, 32768, 131072])
def test_a_prompt_needs_its_images_and_parts(size, rows):
    most = 128 * MIB + rows // 32 * 4 * 33 * 1024 + 2 * MIB
    got = size(1, 16, 4, 256, 256, 128, rows, rows, rows, 4096, 4)
    print(rows, got / MIB)
    assert 0 < got <= most
    assert rows < 131072 or got < 700 * MIB


def test_images_of_many_requests_are_bounded(size):
    """512 MiB of images, the parts (192 MiB at heads of 128), the plan, whatever the longest request may be."""
    for rows in (4096, 65536):
        got = size(64, 32, 8, 128, 128, 16, 64 * rows, rows, rows, 4096, 4)
        print(rows, got / MIB)
        assert got <= (512 + 192 + 16) * MIB
