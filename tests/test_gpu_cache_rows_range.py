"""The operators on rows of the HiF8 KV cache where a row is nobody's, where row
scales or weights lie far apart, and where a call falls to the any-shape
kernels: against float64 (tests/_rows.py)."""

import math

import numpy as np
import pytest
import torch

from _kv import build_cache, randn
from _rows import tree_reference

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _stale(shape, dtype, device):
    """Leaves NaN in the allocator's free memory of an output's size."""
    torch.cuda.synchronize()
    held = [torch.full(shape, math.nan, dtype=dtype, device=device) for _ in range(8)]
    torch.cuda.synchronize()
    del held


@pytest.mark.parametrize("d, dv, bs", [(256, 256, 128), (64, 64, 16), (96, 96, 20), (20, 36, 12)])
@pytest.mark.parametrize("total, loc", [(14, [2, 5, 12]), (150, [3, 60, 141]), (9, [0, 0, 4]), (9, [9, 9, 9])])
def test_query_rows_of_no_request_are_zeros(native_ops, device, d, dv, bs, total, loc):
    """A padded batch: rows before the first request and behind the last one."""
    from hif8_rocm import kv_cache

    ctx, hq, hkv = [200, 31], 16, 4
    qlens = [loc[1] - loc[0], loc[2] - loc[1]]
    kc, vc, table = build_cache(device, [c + n for c, n in zip(ctx, qlens)], hkv, d, bs, 1, dv=dv)
    q = randn((total, hq, d), 2)
    width = max(max(qlens), 1)
    mask = np.random.default_rng(3).random((total, width)) < 0.5
    print(f"rows {loc} of {total}, d={d} dv={dv}", flush=True)
    _stale((total, hq, dv), torch.bfloat16, device)
    out = kv_cache.tree_attention(q.to(device), kc, vc, table.to(device), torch.tensor(ctx, dtype=I32, device=device),
                                  torch.from_numpy(mask).to(device), scale=1 / math.sqrt(d),
                                  query_start_loc=torch.tensor(loc, dtype=I32, device=device), max_query_len=width,
                                  max_seq_len=max(c + n for c, n in zip(ctx, qlens)), validate=False)
    torch.cuda.synchronize()
    got = out.double().cpu().numpy()
    assert not got[:loc[0]].any() and not got[loc[2]:].any()   # NaN counts as any
    want, bound = tree_reference(q[loc[0]:loc[2]].double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), ctx,
                                 qlens, mask[loc[0]:loc[2]], 1 / math.sqrt(d), torch.bfloat16)
    assert (np.abs(got[loc[0]:loc[2]] - want) <= bound).all()
