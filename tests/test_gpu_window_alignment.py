"""Attention within a sliding window over queries and into outputs that start at any element: what aligned ones give."""

import ctypes
import math

import pytest
import torch

from _kv import build_cache, randn
from test_abi import LIB

pytestmark = pytest.mark.gpu
P, I, L, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("starts, total", [([0, 300], 300), ([3, 293], 297), ([0, 150, 152, 300], 300), ([1, 91, 200], 204)])
def test_long_requests_at_any_alignment(native_ops, device, starts, total, d, dtype):
    lib = ctypes.CDLL(str(LIB))
    f, size = lib.hif8_window_attention, lib.hif8_window_attention_workspace_size
    f.argtypes = [P, I, P, P, L, L, L, L, L, P, I, L, P, P, L, L, L, L, L, L, L, ctypes.c_float, P, P, Z, P]
    size.argtypes, size.restype = [L] * 11, Z
    batch, hq, hkv, page = len(starts) - 1, 8, 2, 16
    lens = [310, 160, 200][:batch]
    kc, vc, table = build_cache(device, lens, hkv, d, page, d)
    table, loc = table.to(device), torch.tensor(starts, dtype=torch.int32, device=device)
    sizes = torch.tensor(lens, dtype=torch.int32, device=device)
    q = randn((total, hq, d), 3, 1.0, dtype).to(device)
    n = size(batch, hq, hkv, d, d, page, total, 300, 320, 70, 5)
    ws = torch.empty(n, dtype=torch.uint8, device=device)

    def call(shift_q, shift_out):
        print(f"starts={starts} d={d} {dtype} shifts {shift_q} {shift_out}", flush=True)
        flat = torch.zeros(q.numel() + 8, dtype=dtype, device=device)
        flat[shift_q:shift_q + q.numel()] = q.flatten()
        out = torch.full((q.numel() + 8,), math.nan, dtype=dtype, device=device)
        rc = f(flat.data_ptr() + 2 * shift_q, 1 if dtype == torch.bfloat16 else 0, kc.data_ptr(), vc.data_ptr(), kc.shape[0],
               page, hkv, d, d, table.data_ptr(), 0, table.shape[1], loc.data_ptr(), sizes.data_ptr(), batch, hq, total, 300,
               320, 70, 5, 1 / math.sqrt(d), out.data_ptr() + 2 * shift_out, ws.data_ptr(), n,
               torch.cuda.current_stream().cuda_stream)
        assert rc == 0
        torch.cuda.synchronize()
        mine = out[shift_out:shift_out + q.numel()]
        assert out[:shift_out].isnan().all() and out[shift_out + q.numel():].isnan().all()
        return mine

    # Short requests among long ones take the any-shape kernel where not both are aligned: other sums, one rounding.
    want, several = call(0, 0), batch == 3
    assert want.isfinite().all()
    for shifts in ((1, 0), (0, 3), (5, 7), (4, 4)):
        got = call(*shifts)
        if several:
            torch.testing.assert_close(got.float(), want.float(), rtol=2 ** -7, atol=2 ** -10)
        else:
            assert torch.equal(got, want)
