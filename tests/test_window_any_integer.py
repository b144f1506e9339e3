"""Windows and counts of first tokens that no 64-bit integer holds: every row is seen (CPU: up to the device)."""

import pytest
import torch

from hif8_rocm import kv_cache

I32 = torch.int32


@pytest.mark.parametrize("window, sinks", [(2 ** 64, 0), (2 ** 63 - 1, 2 ** 63), (5, 10 ** 30), (10 ** 30, 4)])
def test_large_windows_pass_the_checks(window, sinks):
    caches = (torch.zeros(4, 16, 2, 68, dtype=torch.uint8),) * 2
    table, q = torch.tensor([[0, 1, 2, 3]], dtype=I32), torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    seen = {"window": window, "sinks": sinks}
    past = pytest.raises(Exception, match="HIP device|could not be loaded|backend")
    with past:
        kv_cache.paged_decode_attention(q[:1], *caches, table, [64], scale=1.0, **seen)
    with past:
        kv_cache.paged_attention(q, *caches, table, [64], scale=1.0, query_lens=[3], **seen)
    with past:
        kv_cache.release_blocks(table, torch.zeros(4, dtype=I32), torch.zeros(1, dtype=I32), [64], block_size=16, **seen)
    # The checks see what the call would: pages inside the window have to be there.
    with pytest.raises(IndexError):
        kv_cache.paged_attention(q, *caches, torch.tensor([[0, -1, 2, 3]], dtype=I32), [64], scale=1.0, query_lens=[3], **seen)
