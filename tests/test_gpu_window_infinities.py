"""Infinite and NaN codes of V that every query row of a request sees, in the middle of a window that is longer than
any tile: an infinity of the formula's sign, NaN where it gives NaN, the other dims as they were."""

import math

import numpy as np
import pytest
import torch

from _decoding import window_reference
from _kv import build_cache, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("qlens", [[1, 1], [6, 2], [20, 7], [140, 90]])
def test_window_infinities_that_all_rows_see(native_ops, device, qlens, d, dtype):
    from hif8_rocm import kv_cache

    lens, window, sinks, page = [1700, 1500], 1200, 20, 16
    kc, vc, table = build_cache(device, lens, 2, d, page, d, mixed=True)
    q = randn((sum(qlens), 8, d), 3, 1.0, dtype)
    args = {"scale": 1 / math.sqrt(d), "query_lens": qlens, "window": window, "sinks": sinks}
    plain = kv_cache.paged_attention(q.to(device), kc, vc, table.to(device), lens, **args)
    # (row, head, dim, code): alone in a dim, twice of one sign, of both signs.
    for b in range(2):
        for t, head, dim, code in ((1000, 0, 5, 0x6F), (1130, 0, 6, 0xEF), (870, 0, 9, 0x80), (900, 1, 7, 0x6F),
                                   (1201, 1, 7, 0x6F), (777, 1, 11, 0x6F), (1333, 1, 11, 0xEF), (3, 1, 20, 0xEF)):
            vc[int(table[b, t // page]), t % page, head, dim] = code
    print(f"infinite V rows={qlens} d={d} {dtype}", flush=True)
    out = kv_cache.paged_attention(q.to(device), kc, vc, table.to(device), lens, **args)
    want, _ = window_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), lens, qlens,
                               window, sinks, 1 / math.sqrt(d), dtype)
    got, plain = out.double().cpu().numpy(), plain.double().cpu().numpy()
    finite = np.isfinite(want)
    assert (~finite).any(axis=-1).all() and finite.sum() > (~finite).sum()
    assert np.array_equal(np.isnan(got), np.isnan(want))
    odd = ~finite & ~np.isnan(want)
    assert np.array_equal(got[odd], want[odd])
    assert np.array_equal(got[finite], plain[finite])
