"""query_start_loc is caller data: entries far below zero and past the rows are clipped before they are subtracted."""

import pytest
import torch

from _kv import build_cache, randn

pytestmark = pytest.mark.gpu
I32, LOW, HIGH = torch.int32, -2 ** 31, 2 ** 31 - 1


# Requests that are empty once clipped, then one that has all rows (or but for the first).
@pytest.mark.parametrize("rows", [9, 150])
@pytest.mark.parametrize("bad, good", [([3, LOW, None], [0, 0, None]), ([HIGH, LOW, HIGH], [0, 0, None]),
                                       ([LOW + 5, -7, None], [0, 0, None]), ([1, LOW + 1, HIGH], [0, 0, None])])
def test_starts_are_clipped(native_ops, device, bad, good, rows):
    from hif8_rocm import kv_cache

    bad, good = ([rows if v is None else v for v in loc] for loc in (bad, good))
    lens, hkv, page = [40, 200], 2, 16
    kc, vc, table = build_cache(device, lens, hkv, 64, page, 1)
    q = randn((rows, 8, 64), 2).to(device)
    sizes, pages = torch.tensor(lens, dtype=I32, device=device), table.to(device)
    mask = (torch.rand(rows, rows, generator=torch.Generator().manual_seed(1)) < 0.5).to(device)
    g = torch.Generator().manual_seed(2)
    probs = torch.softmax(torch.randn(rows, 300, generator=g), -1).to(device)
    tokens, u = torch.randint(0, 300, (rows,), generator=g).to(device), torch.rand(rows, generator=g).to(device)

    def calls(loc):
        loc = torch.tensor(loc, dtype=I32, device=device)
        opts = {"query_start_loc": loc, "max_query_len": rows, "max_seq_len": 200, "validate": False}
        yield "window", kv_cache.paged_attention(q, kc, vc, pages, sizes, scale=0.1, window=30, sinks=2, **opts)
        yield "prompt", kv_cache.paged_attention(q, kc, vc, pages, sizes, scale=0.1, **opts)
        yield "tree", kv_cache.tree_attention(q, kc, vc, pages, sizes - torch.tensor([0, rows], dtype=I32, device=device),
                                              mask, scale=0.1, **opts)
        w = torch.zeros(2, hkv, 200, device=device)
        kv_cache.accumulate_key_weights(q, kc, pages, sizes, w, scale=0.1, **opts)
        yield "weights", w
        yield "verify", kv_cache.verify_drafts(probs, tokens, u, query_start_loc=loc, max_query_len=rows, validate=False)
        held = torch.full((2, 30), -1, dtype=I32, device=device)
        free, count = torch.arange(40, dtype=I32, device=device), torch.tensor([40], dtype=I32, device=device)
        yield "pages", (*kv_cache.extend_block_tables(held, free, count, sizes, block_size=page, query_start_loc=loc,
                                                      total_query_tokens=rows, validate=False), held, count)

    for (name, got), (_, want) in zip(calls(bad), calls(good)):
        print(f"{name} {bad} of {rows}", flush=True)
        torch.cuda.synchronize()
        for a, b in zip(got if isinstance(got, tuple) else (got,), want if isinstance(want, tuple) else (want,)):
            assert torch.equal(a, b), name
