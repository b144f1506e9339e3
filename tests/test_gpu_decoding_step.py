"""Operators around a decoding step on the GPU, against their plain forms
(tests/_decoding.py): attention within a sliding window, verification of drafts,
pages taken and given back, and a run of them together.  Whole numbers are
compared exactly."""

import math

import numpy as np
import pytest
import torch

from _decoding import extend_reference, release_reference, verify_reference, window_reference
from _kv import build_cache, randn
from _rows import ancestors, tree_reference

pytestmark = pytest.mark.gpu
I32, I64 = torch.int32, torch.int64


def _near(got, want, bound):
    got = got.double().cpu().numpy()
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)])
    over = np.abs(got - want)[finite] / np.maximum(bound[finite], 1e-300)
    print(f"  worst error / bound {over.max(initial=0.0):.3f}", flush=True)
    assert (over <= 1.0).all(), float(over.max())


def _unseen_pages(table, lens, qlens, window, sinks, page, fill):
    """The table with `fill` where no query row looks."""
    table = table.clone()
    for b, (size, n) in enumerate(zip(lens, qlens)):
        low = size - n + 1 - window
        for j in range(table.shape[1]):
            if j * page >= size or ((j + 1) * page <= low and j * page >= sinks) or n == 0:
                table[b, j] = fill
    return table


def _window(device, lens, qlens, window, sinks, hq, hkv, d, page, *, seed=0, dv=None, dtype=torch.bfloat16,
            mixed=False, bt_dtype=I32, q_mul=1.0, spoil=None, pages=-1, decode=False, check=True):
    from hif8_rocm import kv_cache

    print(f"window lens={lens[:4]} rows={qlens[:4]} window={window} sinks={sinks} hq={hq} hkv={hkv} d={d} dv={dv} "
          f"page={page} {dtype}", flush=True)
    kc, vc, table = build_cache(device, lens, hkv, d, page, seed, dv=dv, bt_dtype=bt_dtype, mixed=mixed)
    table = _unseen_pages(table, lens, qlens, window, sinks, page, pages)
    q = randn((sum(qlens), hq, d), seed + 1, q_mul, dtype)
    if spoil:
        spoil(kc, vc, table)
    args = (q.to(device), kc, vc, table.to(device), lens)
    opts = {"scale": 1 / math.sqrt(d), "window": window, "sinks": sinks, "validate": spoil is None}
    if decode:
        out = kv_cache.paged_decode_attention(*args, **opts)
    else:
        out = kv_cache.paged_attention(*args, query_lens=qlens, **opts)
    torch.cuda.synchronize()
    if check:
        want, bound = window_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), lens,
                                       qlens, window, sinks, 1 / math.sqrt(d), dtype)
        _near(out, want, bound)
    return out


@pytest.mark.parametrize("lens, window, sinks, hq, hkv, d, page", [
    ([1], 1, 0, 16, 4, 256, 128),
    ([0, 1, 2, 17], 1, 1, 16, 4, 256, 128),
    ([1500], 1024, 4, 16, 4, 256, 128),
    ([300, 128, 129, 64], 64, 16, 8, 2, 128, 16),
    ([700, 33], 100, 33, 24, 8, 128, 32),              # three query heads per KV head
    ([900], 17, 0, 8, 8, 64, 32),
    ([500, 20], 130, 300, 20, 2, 256, 144),            # pages of nine sixteens, sinks past the window
    ([2100], 2000, 4, 32, 1, 128, 64),
    ([600], 5000, 4, 12, 4, 64, 16),                   # the window covers everything
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_in_a_window(native_ops, device, lens, window, sinks, hq, hkv, d, page, dtype):
    _window(device, lens, [1] * len(lens), window, sinks, hq, hkv, d, page, dtype=dtype, seed=hq + d, decode=True)


@pytest.mark.parametrize("lens, qlens, window, sinks, hq, hkv, d, page", [
    ([40], [5], 16, 4, 16, 4, 256, 128),
    ([5], [5], 2, 0, 16, 4, 256, 128),
    ([300, 12, 0, 77], [7, 12, 0, 1], 50, 4, 8, 2, 128, 16),
    ([400, 300], [130, 33], 64, 21, 24, 8, 128, 32),
    ([333], [333], 100, 4, 16, 4, 256, 128),           # a whole prompt
    ([513], [200], 1, 0, 4, 4, 64, 16),
    ([260, 500, 64], [260, 100, 2], 90, 70, 8, 2, 256, 16),
    ([200], [150], 40, 8, 20, 2, 64, 144),
    ([150], [140], 1000, 4, 14, 2, 128, 64),           # seven query heads per KV head
    ([700], [400], 257, 5, 32, 4, 128, 16),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_in_a_window(native_ops, device, lens, qlens, window, sinks, hq, hkv, d, page, dtype):
    _window(device, lens, qlens, window, sinks, hq, hkv, d, page, dtype=dtype, seed=hq + d)


@pytest.mark.parametrize("d, dv, hq, hkv, page", [(20, 36, 6, 2, 12), (96, 96, 5, 5, 128), (512, 256, 4, 2, 7),
                                                  (128, 64, 4, 4, 16), (256, 256, 4, 1, 8), (80, 80, 2, 1, 1)])
def test_window_any_head_and_page_size(native_ops, device, d, dv, hq, hkv, page):
    _window(device, [137, 3], [30, 2], 40, 5, hq, hkv, d, page, dv=dv, seed=d)
    _window(device, [137, 3], [1, 1], 40, 5, hq, hkv, d, page, dv=dv, seed=d, decode=True)


@pytest.mark.parametrize("qlens", [[1, 1], [9, 3], [150, 129]])
@pytest.mark.parametrize("mixed, bt_dtype, q_mul", [(True, I64, 1.0), (False, I64, 8.0), (True, I32, 8.0)])
def test_window_row_scales_tables_and_peaked_rows(native_ops, device, qlens, mixed, bt_dtype, q_mul):
    for dtype in (torch.bfloat16, torch.float16):
        _window(device, [300, 129], qlens, 70, 20, 16, 4, 256, 128, mixed=mixed, bt_dtype=bt_dtype, q_mul=q_mul,
                dtype=dtype, seed=5)


@pytest.mark.parametrize("qlens", [[1, 1], [9, 3], [150, 129]])
def test_window_scales_of_any_size_and_sign(native_ops, device, qlens):
    """Sidecars that grow and shrink by 2^20 along the rows, negative and zero ones among them."""
    def spoil(kc, vc, table):
        g = torch.Generator().manual_seed(1)
        n = vc.shape[0] * vc.shape[1] * vc.shape[2]
        s = (2.0 ** torch.randint(-20, 0, (n,), generator=g).float()) * torch.randint(-1, 2, (n,), generator=g).float()
        vc.view(n, -1)[:, -4:] = s.view(n, 1).view(torch.uint8).to(vc.device)
        k = torch.where(torch.rand(n, generator=g) < 0.3, -0.01, 0.02) * (torch.rand(n, generator=g) > 0.1)
        kc.view(n, -1)[:, -4:] = k.view(n, 1).view(torch.uint8).to(kc.device)

    for dtype in (torch.bfloat16, torch.float16):
        _window(device, [300, 129], qlens, 90, 20, 16, 4, 256, 128, spoil=spoil, dtype=dtype, seed=9)


@pytest.mark.parametrize("qlens, d", [([1, 1], 256), ([5, 9], 256), ([140, 33], 256), ([100, 129], 64), ([40, 70], 96)])
def test_window_hides_what_it_does_not_show(native_ops, device, qlens, d):
    """NaN, infinities and NaN scales in rows that some or all query rows do not see."""
    lens, window, sinks, page = [300, 200], 60, 20, 16

    def spoil(kc, vc, table):
        for b, (size, n) in enumerate(zip(lens, qlens)):
            low = size - n + 1 - window
            for t in list(range(sinks, max(low, sinks))) + list(range(size, -(-size // page) * page)):
                blk = int(table[b, t // page])
                if not 0 <= blk < kc.shape[0]:
                    continue
                for cache, code in ((kc, 0x80), (vc, (0x80, 0x6F, 0xEF)[t % 3])):
                    cache[blk, t % page, :, :-4] = code
                    cache[blk, t % page, :, -4:] = torch.tensor([0, 0, 0xC0, 0x7F], dtype=torch.uint8, device=cache.device)
            if n > 1:   # seen by the last rows alone; one element each
                for t, code in ((size - 1, 0x80), (size - n // 2, 0x6F)):
                    vc[int(table[b, t // page]), t % page, :, 3] = code
                # seen by the first rows alone
                vc[int(table[b, max(low, 0) // page]), max(low, 0) % page, 0, 7] = 0xEF

    # Pages outside: ids that no cache has.
    for fill in (-7, 2 ** 31 - 1):
        _window(device, lens, qlens, window, sinks, 8, 2, d, page, spoil=spoil, pages=fill, seed=3)


@pytest.mark.parametrize("qlens", [[1], [6], [140]])
def test_window_nan_and_infinite_keys_and_queries(native_ops, device, qlens):
    lens, page = [200], 16

    def spoil(kc, vc, table):
        for t, code in ((lens[0] - 1, 0x80), (lens[0] - 2, 0x6F)):
            kc[int(table[0, t // page]), t % page, 1, 5] = code

    out = _window(device, lens, qlens, 50, 4, 8, 2, 128, page, spoil=spoil, seed=4)
    assert out[-1, 4:].isnan().all() and not out[:, :4].isnan().any()


def test_window_pages_outside_the_cache_are_left_out(native_ops, device):
    def spoil(kc, vc, table):
        table[0, 2], table[1, 0] = 10 ** 6, -1

    for qlens in ([1, 1], [10, 5], [150, 129]):
        _window(device, [300, 129], qlens, 280, 4, 16, 4, 256, 64, spoil=spoil, seed=6)


def test_window_of_every_row_is_causal_attention(native_ops, device):
    """A window as long as the request changes nothing but the rounding of K, V and the weights."""
    from hif8_rocm import kv_cache

    lens, qlens = [250, 64], [120, 64]
    kc, vc, table = build_cache(device, lens, 4, 128, 16, 3)
    q = randn((sum(qlens), 16, 128), 4).to(device)
    table = table.to(device)
    plain = kv_cache.paged_attention(q, kc, vc, table, lens, scale=0.1, query_lens=qlens)
    for window in (250, 2 ** 40):
        out = kv_cache.paged_attention(q, kc, vc, table, lens, scale=0.1, query_lens=qlens, window=window)
        torch.testing.assert_close(out.float(), plain.float(), rtol=2e-2, atol=2e-2)


def test_window_rows_of_no_request_are_zeros(native_ops, device):
    from hif8_rocm import kv_cache

    lens = [100, 30]
    kc, vc, table = build_cache(device, lens, 2, 64, 16, 1)
    for n0 in (3, 100):
        rows = n0 + 30 + 7
        q = randn((rows, 4, 64), 2).to(device)
        # Rows before the first request, between none, and behind the last.
        loc = torch.tensor([2, 2 + n0, 2 + n0 + 30], dtype=I32, device=device)
        out = kv_cache.paged_attention(q, kc, vc, table.to(device), torch.tensor(lens, dtype=I32, device=device),
                                       scale=0.1, query_start_loc=loc, max_query_len=max(n0, 30), max_seq_len=100,
                                       window=20, sinks=2, validate=False)
        assert not out[:2].any() and not out[2 + n0 + 30:].any()
        want = kv_cache.paged_attention(q[2:2 + n0 + 30].clone(), kc, vc, table.to(device), lens, scale=0.1,
                                        query_lens=[n0, 30], window=20, sinks=2)
        assert torch.equal(out[2:2 + n0 + 30], want)


def test_window_request_shorter_than_its_rows(native_ops, device):
    """Rows at positions before the request's start see nothing: zeros."""
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, [20, 9], 2, 128, 16, 1)
    q = randn((150, 4, 128), 2).to(device)
    loc = torch.tensor([0, 140, 150], dtype=I32, device=device)
    out = kv_cache.paged_attention(q, kc, vc, table.to(device), torch.tensor([20, 9], dtype=I32, device=device),
                                   scale=0.1, query_start_loc=loc, max_query_len=140, max_seq_len=20, window=5,
                                   validate=False)
    assert not out[:120].any() and out[120:140].any(-1).all() and not out[140].any() and out[141:].any(-1).all()


@pytest.mark.parametrize("lens, qlens, window, sinks, hq, hkv, d, page", [
    ([300, 300, 300], [64, 65, 66], 50, 4, 8, 2, 128, 16),      # 256, 260 and 264 rows per KV head
    ([600], [128], 90, 4, 8, 2, 64, 16),                        # one request of 512 rows, and of 516
    ([600], [129], 90, 4, 8, 2, 64, 16),
    ([700, 650], [600, 300], 33, 0, 4, 4, 64, 32),              # a query head per KV head
    ([80, 70], [60, 9], 20, 3, 32, 1, 256, 48),                 # 32 query heads per KV head
    ([80, 70], [60, 9], 20, 3, 33, 1, 64, 48),                  # more than that
    ([40, 1, 0, 2, 290], [40, 1, 0, 2, 290], 1, 0, 16, 2, 128, 16),
    ([500, 500], [300, 299], 600, 17, 4, 4, 256, 16),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_around_the_long_ones(native_ops, device, lens, qlens, window, sinks, hq, hkv, d, page, dtype):
    _window(device, lens, qlens, window, sinks, hq, hkv, d, page, dtype=dtype, seed=hq + d)


@pytest.mark.parametrize("lens, qlens, hq, hkv, d", [
    ([70, 40], [60, 9], 64, 1, 128), ([50], [50], 200, 2, 256), ([30, 30], [20, 30], 71, 1, 64),
    ([20, 9, 30], [20, 2, 3], 127, 1, 128), ([24, 20], [4, 1], 256, 1, 64), ([24, 20], [9, 2], 255, 1, 256),
    ([12, 9], [5, 2], 257, 1, 128), ([12, 9], [5, 2], 300, 1, 256),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_window_many_query_heads_per_kv_head(native_ops, device, lens, qlens, hq, hkv, d, dtype):
    _window(device, lens, qlens, 17, 2, hq, hkv, d, 16, dtype=dtype, seed=hq)


@pytest.mark.parametrize("long", [range(0, 150, 7), range(60, 70), range(149, 150), ()])
def test_window_long_requests_among_many(native_ops, device, long):
    """More requests than a wavefront has lanes; long ones between short and empty ones."""
    qlens = [70 if b in long else (0, 1, 3, 2)[b % 4] for b in range(150)]
    lens = [n and n + 5 * (b % 9) for b, n in enumerate(qlens)]
    _window(device, lens, qlens, 24, 4, 8, 2, 64, 16, seed=len(long))


@pytest.mark.parametrize("most", [44800, 80000, 160000])
def test_window_long_requests_in_passes(native_ops, device, most):
    """Requests that may be so long that their images are made in passes; and, as ever, are not."""
    from hif8_rocm import kv_cache

    lens, qlens = [290, 100, 41, 300, 170], [90, 100, 20, 70, 66]
    kc, vc, table = build_cache(device, lens, 4, 256, 16, 3)
    table = torch.cat([table, torch.full((5, most // 16 - table.shape[1]), -1, dtype=I32)], 1)
    q = randn((sum(qlens), 16, 256), 4)
    loc = torch.tensor(np.concatenate([[0], np.cumsum(qlens)]), dtype=I32, device=device)
    out = kv_cache.paged_attention(q.to(device), kc, vc, table.to(device), torch.tensor(lens, dtype=I32, device=device),
                                   scale=0.0625, query_start_loc=loc, max_query_len=100, max_seq_len=most,
                                   window=2 ** 30, sinks=2, validate=False)
    want, bound = window_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), lens, qlens,
                                   2 ** 30, 2, 0.0625, torch.bfloat16)
    _near(out, want, bound)


@pytest.mark.parametrize("starts", [[2, 202], [0, 0], [2, 202, 202, 330], [1, 3, 140, 141]])
def test_window_rows_around_long_requests_are_zeros(native_ops, device, starts):
    from hif8_rocm import kv_cache

    lens = [230] * (len(starts) - 1)
    qlens = [b - a for a, b in zip(starts, starts[1:])]
    kc, vc, table = build_cache(device, lens, 2, 128, 16, 1)
    table = table.to(device)
    q = randn((starts[-1] + 9, 12, 128), 2)
    out = kv_cache.paged_attention(q.to(device), kc, vc, table, torch.tensor(lens, dtype=I32, device=device), scale=0.1,
                                   query_start_loc=torch.tensor(starts, dtype=I32, device=device), max_query_len=200,
                                   max_seq_len=240, window=20, sinks=2, validate=False)
    assert not out[:starts[0]].any() and not out[starts[-1]:].any()
    if sum(qlens):
        want, bound = window_reference(q[starts[0]:starts[-1]].double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(),
                                       table.cpu().numpy(), lens, qlens, 20, 2, 0.1, torch.bfloat16)
        _near(out[starts[0]:starts[-1]], want, bound)


@pytest.mark.parametrize("d, qlens", [(256, [1, 1]), (128, [9, 4]), (256, [90, 70]), (64, [300, 2])])
def test_window_of_a_cache_past_32_bits(native_ops, device, d, qlens):
    """Pages behind the first 4 GiB of the cache answer as the same pages in a small one."""
    from hif8_rocm import kv_cache

    lens, hkv, page = [330, 150], 4, 16
    kc, vc, table = build_cache(device, lens, hkv, d, page, 7)
    q = randn((sum(qlens), 16, d), 8).to(device)
    opts = {"scale": 0.1, "query_lens": qlens, "window": 100, "sinks": 20}
    want = kv_cache.paged_attention(q, kc, vc, table.to(device), lens, **opts)
    blocks = (2 ** 32 + 2 ** 20) // (page * hkv * (d + 4)) + kc.shape[0]
    big = [torch.empty(blocks, *c.shape[1:], dtype=torch.uint8, device=device) for c in (kc, vc)]
    for b, c in zip(big, (kc, vc)):
        b[-c.shape[0]:] = c
    moved = torch.where(table < 0, table, table + (blocks - kc.shape[0]))
    got = kv_cache.paged_attention(q, *big, moved.to(device), lens, **opts)
    assert torch.equal(got, want)


@pytest.mark.parametrize("lens, qlens, hq, hkv, d", [
    ([900, 400], [1, 1], 16, 4, 256), ([900, 400], [6, 3], 16, 4, 256), ([900, 400], [20, 30], 16, 4, 256),
    ([900, 400], [7, 8], 16, 4, 128), ([900, 400], [30, 9], 16, 4, 128), ([900, 400], [2, 4], 16, 4, 64),
    ([900, 400], [7, 8], 16, 4, 64), ([900, 400], [30, 9], 16, 4, 64), ([400, 300], [200, 90], 8, 2, 256),
    ([400, 300], [200, 90], 8, 2, 128), ([400, 300], [200, 90], 8, 2, 64),
])
def test_window_fp16_is_off_by_its_rounding(native_ops, device, lens, qlens, hq, hkv, d):
    """Root mean squares: rounding the exact answer to fp16 is off by about 2^-12.3 of it, a weight rounded to
    fp16 would add as much again (1.4 times); with what that leaves multiplied (2^-22) and logits in float32 (off by
    less than 2^-15, so weights by less than 2^-15) the whole stays within sqrt(1 + 2^-5.4) = 1.012 of the first."""
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, lens, hkv, d, 16, d)
    q = randn((sum(qlens), hq, d), 3, 1.0, torch.float16)
    out = kv_cache.paged_attention(q.to(device), kc, vc, table.to(device), lens, scale=1 / math.sqrt(d),
                                   query_lens=qlens, window=333, sinks=4)
    want, _ = window_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), lens, qlens, 333,
                               4, 1 / math.sqrt(d), torch.float16)
    off, own = (np.sqrt(np.square(x - want).mean()) for x in (out.double().cpu().numpy(), want.astype(np.float16).astype(np.float64)))
    print(f"  off {off:.3e}, the rounding {own:.3e}", flush=True)
    assert off <= 1.05 * own


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("n", [1, 6, 20, 140])
def test_window_infinities_in_fp16(native_ops, device, n, d):
    """Infinite and NaN codes and infinite scales of V, seen by some rows, hidden from others, where P has two parts."""
    lens, page, low = [200], 16, max(200 - n + 1 - 60, 20)

    def spoil(kc, vc, table):
        inf = torch.tensor([0, 0, 0x80, 0x7F], dtype=torch.uint8, device=vc.device)
        for t, head, code in ((199, 0, 0x6F), (198, 1, 0x80), (low, 0, 0xEF), (low - 1, 0, 0x80), (low - 2, 1, 0x6F)):
            vc[int(table[0, t // page]), t % page, head, 5] = code
        vc[int(table[0, 190 // page]), 190 % page, 1, -4:] = inf
        vc[int(table[0, (low - 3) // page]), (low - 3) % page, 0, -4:] = inf

    _window(device, lens, [n], 60, 20, 8, 2, d, page, dtype=torch.float16, spoil=spoil, seed=d + n)


def test_window_of_prompts_captured(native_ops, device):
    """Long requests in a captured call: replays follow lengths, tables and queries, and two graphs share nothing."""
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, [500, 500], 2, 128, 16, 1)
    table = table.to(device)
    graphs = []
    for rows in (160, 300):
        q = torch.zeros(rows, 8, 128, dtype=torch.bfloat16, device=device)
        loc, lens = torch.zeros(3, dtype=I32, device=device), torch.zeros(2, dtype=I32, device=device)

        def call(q=q, loc=loc, lens=lens, rows=rows):
            return kv_cache.paged_attention(q, kc, vc, table, lens, scale=0.1, query_start_loc=loc, max_query_len=rows,
                                            max_seq_len=500, window=100, sinks=4, validate=False)

        call()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = call()
        graphs.append((g, q, loc, lens, out, call))
    for i in range(6):
        for g, q, loc, lens, out, call in graphs:
            n = q.shape[0]
            q.copy_(randn(q.shape, 10 + i))
            split = (0, n, n // 2, n - 3, 70, 1)[i]
            loc.copy_(torch.tensor([0, split, n]))
            lens.copy_(torch.tensor([500 - 17 * i, 300 + 20 * i]))
        for g, *_ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, q, loc, lens, out, call in graphs:
            assert torch.equal(out, call())


def test_window_unaligned_and_strided_queries(native_ops, device):
    from hif8_rocm import kv_cache

    lens = [90]
    kc, vc, table = build_cache(device, lens, 2, 64, 16, 1)
    for n in (1, 40):
        base = randn((n * 4 * 64 + 1,), 3).to(device)
        odd = base[1:].view(n, 4, 64)
        wide = randn((n, 4, 128), 5).to(device)[..., ::2]
        for q in (odd, wide):
            out = kv_cache.paged_attention(q, kc, vc, table.to(device), lens, scale=0.1, query_lens=[n], window=30)
            want = kv_cache.paged_attention(q.clone(memory_format=torch.contiguous_format), kc, vc, table.to(device),
                                            lens, scale=0.1, query_lens=[n], window=30)
            torch.testing.assert_close(out.float(), want.float(), rtol=2 ** -7, atol=1e-3)


# ------------------------------------------------------------- verification
def _verify_case(qlens, vocab, seed, tree=False, sampled=False, peaked=3.0):
    g = np.random.default_rng(seed)
    total = sum(qlens)

    def softmax(x):
        e = np.exp(x - x.max(axis=-1, keepdims=True))
        return (e / e.sum(axis=-1, keepdims=True)).astype(np.float32)

    logits = g.standard_normal((total, vocab)) * peaked
    probs = softmax(logits)
    draft = softmax(logits[np.maximum(np.arange(total) - 1, 0)] + g.standard_normal((total, vocab))) if sampled else None
    tokens, parents = np.zeros(total, dtype=np.int64), np.full(total, -1, dtype=np.int32)
    row = 0
    for n in qlens:
        for i in range(n):
            parents[row + i] = (max(0, i - int(g.integers(1, 5))) if tree else i - 1) if i else -1
            p = draft[row + i] if sampled else probs[row + max(parents[row + i], 0)]
            tokens[row + i] = g.choice(vocab, p=p.astype(np.float64) / p.astype(np.float64).sum()) if sampled else \
                int(np.argsort(-p)[g.integers(0, min(3, vocab))])
        row += n
    return probs, draft, tokens, parents if tree else None, g.random(total).astype(np.float32)


def _verify(device, case, qlens, width=None, tokens_dtype=I64, **opts):
    from hif8_rocm import kv_cache

    probs, draft, tokens, parents, uniforms = case
    dev = {k: None if v is None else torch.from_numpy(v).to(device) for k, v in
           {"draft_probs": draft, "parents": parents}.items()}
    got = kv_cache.verify_drafts(torch.from_numpy(probs).to(device), torch.from_numpy(tokens).to(device, tokens_dtype),
                                 torch.from_numpy(uniforms).to(device), query_lens=qlens, max_query_len=width, **dev,
                                 **opts)
    want = verify_reference(*case, qlens, width or max(qlens, default=0))
    for g, w, name in zip(got, want, ("accepted", "counts", "next")):
        assert np.array_equal(g.cpu().numpy(), w), (name, g.cpu().numpy(), w)
    assert [t.dtype for t in got] == [I32, I32, I64]
    return got


@pytest.mark.parametrize("kind", ["chain", "tree", "sampled"])
@pytest.mark.parametrize("qlens, vocab", [([1], 1), ([5], 7), ([3, 0, 8, 1], 1000), ([12] * 9, 1024), ([65, 2], 1025),
                                          ([6, 4], 50257), ([2] * 70, 999), ([130], 4099)])
def test_verify(native_ops, device, kind, qlens, vocab):
    for seed in range(3):
        case = _verify_case(qlens, vocab, seed, kind == "tree", kind == "sampled", peaked=1.0 + seed)
        _verify(device, case, qlens, tokens_dtype=(I32, I64)[seed % 2])
    _verify(device, case, qlens, width=max(qlens) + 3)


def test_verify_takes_the_whole_chain_or_nothing(native_ops, device):
    qlens, vocab = [9, 9], 3000
    for sampled in (False, True):
        probs, draft, tokens, _, u = _verify_case(qlens, vocab, 1, sampled=sampled)
        u[:] = 0.0                                       # every token of positive probability follows
        got = _verify(device, (probs, draft, tokens, None, u), qlens)
        assert got[1].tolist() == [9, 9]
        probs[np.arange(17), tokens[1:]] = 0.0           # and none of probability 0
        got = _verify(device, (probs, draft, tokens, None, u), qlens)
        assert got[1].tolist() == [1, 1]


def test_verify_greedy_rows(native_ops, device):
    """Rows that hold one token alone: followed as far as the drafts match it, which then is the answer."""
    qlens, vocab = [6], 2050
    probs, _, tokens, _, u = _verify_case(qlens, vocab, 3)
    best = np.array([5, 2049, 0, 1023, 1024, 77])
    probs[:] = 0.0
    probs[np.arange(6), best] = 1.0
    tokens[1:] = best[:5]
    for stop in range(1, 7):
        t = tokens.copy()
        if stop < 6:
            t[stop] = 9
        got = _verify(device, (probs, None, t, None, u), qlens)
        assert got[1].tolist() == [stop] and got[2].tolist() == [best[stop - 1]]


def test_verify_borders(native_ops, device):
    """Uniform rows, whose sums are exact: random numbers on the border itself belong to the next token."""
    vocab = 4096
    probs = np.full((1, vocab), 1 / vocab, dtype=np.float32)
    for k in (0, 1, 1023, 1024, 2047, 4095):
        got = _verify(device, (probs, None, np.zeros(1, dtype=np.int64), None, np.array([k / vocab], np.float32)), [1])
        assert got[2].tolist() == [k]
    # u q < p is strict, and exact for numbers whose product float32 rounds.
    p, q = np.float32(0.1), np.float32(0.3)
    u = np.float32(np.float64(p) / np.float64(q))
    for v in (np.nextafter(u, np.float32(0)), u, np.nextafter(u, np.float32(1))):
        row = np.zeros((2, 8), dtype=np.float32)
        row[0, 3], row[0, 4], row[1, 3] = p, 1 - p, q
        got = _verify(device, (row, np.stack([row[1], row[1]]), np.array([0, 3]), None,
                               np.array([0.5, v], dtype=np.float32)), [2])
        assert got[1].tolist() == [1 + int(np.float64(v) * np.float64(q) < np.float64(p))]


def test_verify_siblings_with_one_token_and_bad_parents(native_ops, device):
    probs = np.zeros((6, 16), dtype=np.float32)
    probs[:, 2], probs[:, 3], probs[:, 5] = 0.5, 0.25, 0.25
    tokens = np.array([0, 2, 2, 3, 5, 2])
    parents = np.array([-1, 0, 0, 0, 9, -3], dtype=np.int32)
    for u in ([0.99, 0.9, 0.1, 0.4, 0.0, 0.0], [0.3, 0.9, 0.0, 0.9, 0.0, 0.0], [0.0, 0.49, 0.0, 0.0, 0.0, 0.0]):
        case = (probs, None, tokens, parents, np.array(u, dtype=np.float32))
        _verify(device, case, [6], validate=False)


def test_verify_rows_without_a_number(native_ops, device):
    """NaN, infinite and negative entries weigh nothing; a residual without weight falls back to p; nothing: -1."""
    vocab = 2100
    probs, draft, tokens, _, u = _verify_case([3, 3, 2, 1, 2], vocab, 4, sampled=True)
    probs[0, :1500], probs[1, 7], probs[2, ::2] = np.nan, np.inf, -0.5
    probs[3:6], draft[4] = 0.0, 0.0
    probs[3, 1999], draft[4, tokens[4]], probs[3, tokens[4]] = 0.25, 1.0, 0.0
    probs[6] = draft[7]                    # the residual is zero everywhere: drawn from p
    u[7] = np.float32(0.999)
    tokens[7] = int(np.argmin(draft[7]))
    probs[6, tokens[7]] = 0.0
    draft[7, tokens[7]] = 0.5
    probs[8] = np.nan
    probs[9:] = -1.0
    got = _verify(device, (probs, draft, tokens, None, u), [3, 3, 2, 1, 2])
    assert got[2][3].item() == -1 and got[2][4].item() == -1
    # Given drafts: all weight lies on the refused token, which then is drawn after all.
    one = np.zeros((2, vocab), dtype=np.float32)
    one[0, 9] = 0.25
    got = _verify(device, (one, None, np.array([1, 9]), None, np.array([0.5, 0.5], dtype=np.float32)), [2])
    assert got[1].tolist() == [1] and got[2].tolist() == [9]


def test_verify_tokens_outside_the_vocabulary(native_ops, device):
    probs, draft, tokens, _, u = _verify_case([4, 4], 500, 5, sampled=True)
    u[:] = 0
    for bad in (-1, 500, 2 ** 40):
        t = tokens.copy()
        t[2], t[5] = bad, bad
        got = _verify(device, (probs, draft, t, None, u), [4, 4], validate=False)
        assert got[1].tolist() == [2, 1]
        _verify(device, (probs, None, t, None, u), [4, 4], validate=False)


def test_verify_strided_rows_and_padded_batches(native_ops, device):
    from hif8_rocm import kv_cache

    probs, draft, tokens, _, u = _verify_case([4, 3], 1003, 6, sampled=True)
    want = verify_reference(probs, draft, tokens, None, u, [4, 3], 4)
    wide = [torch.zeros(9, 1100, device=device) for _ in range(2)]
    for w, x in zip(wide, (probs, draft)):
        w[1:8, 5:1008] = torch.from_numpy(x).to(device)
    pad = torch.nn.functional.pad
    loc = torch.tensor([1, 5, 8], dtype=I32, device=device)
    got = kv_cache.verify_drafts(wide[0][:, 5:1008], pad(torch.from_numpy(tokens), (1, 1)).to(device),
                                 pad(torch.from_numpy(u), (1, 1)).to(device), draft_probs=wide[1][:, 5:1008],
                                 query_start_loc=loc, max_query_len=4, validate=False)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)
    got = kv_cache.verify_drafts(wide[0].t().contiguous().t()[:, 5:1008], pad(torch.from_numpy(tokens), (1, 1)).to(device),
                                 pad(torch.from_numpy(u), (1, 1)).to(device), draft_probs=wide[1][:, 5:1008],
                                 query_start_loc=loc, max_query_len=4)
    for g, w in zip(got, want):
        assert np.array_equal(g.cpu().numpy(), w)


def test_verify_follows_the_target(native_ops, device):
    """First tokens of many requests with one drawn draft: as often as the target says, within six sigma."""
    from hif8_rocm import kv_cache

    batch, vocab = 20000, 6
    p = torch.tensor([0.05, 0.4, 0.1, 0.2, 0.0, 0.25], device=device)
    q = torch.tensor([0.3, 0.1, 0.2, 0.05, 0.2, 0.15], device=device)
    g = torch.Generator(device=device).manual_seed(0)
    drafts = torch.multinomial(q, batch, replacement=True, generator=g)
    tokens = torch.stack([torch.zeros_like(drafts), drafts], 1).reshape(-1)
    u = torch.rand(2 * batch, generator=g, device=device)
    loc = torch.arange(0, 2 * batch + 1, 2, dtype=I32, device=device)
    for draft in (q.expand(2 * batch, vocab).contiguous(), None):
        _, counts, drawn = kv_cache.verify_drafts(p.expand(2 * batch, vocab).contiguous(), tokens, u, draft_probs=draft,
                                                  query_start_loc=loc, max_query_len=2)
        first = torch.where(counts == 2, drafts, drawn)
        for v in range(vocab):
            share = (first == v).double().mean().item()
            sigma = math.sqrt(p[v].item() * (1 - p[v].item()) / batch)
            assert abs(share - p[v].item()) <= 6 * sigma + 1e-12, (v, share)


# -------------------------------------------------------------------- pages
def _pool(device, ctx, page, columns, spare, seed, dtype=I32):
    g = np.random.default_rng(seed)
    held = [-(-c // page) for c in ctx]
    ids = g.permutation(sum(held) + spare).astype(np.int64)
    table = np.full((len(ctx), columns), -1, dtype=np.int64)
    used = 0
    for b, n in enumerate(held):
        table[b, :n] = ids[used:used + n]
        used += n
    free = np.full(len(ids) + 1, -1, dtype=np.int32)
    free[:spare] = ids[used:]
    return torch.from_numpy(table).to(device, dtype), torch.from_numpy(free).to(device), \
        torch.tensor([spare], dtype=I32, device=device)


@pytest.mark.parametrize("dtype", [I32, I64])
@pytest.mark.parametrize("ctx, qlens, page, spare", [
    ([0], [1], 16, 3), ([0], [0], 16, 3), ([15, 16, 17], [1, 1, 1], 16, 5),
    ([100, 0, 5, 64], [60, 1, 0, 129], 64, 9), ([3], [5000], 1, 6000), ([7, 900], [700, 3], 3, 4000),
    ([40] * 1500, [3] * 1500, 8, 3000), (list(range(2100)), [1] * 2100, 16, 200),
    ([0, 5], [64, 64], 16, 5),             # too few pages: the first request gets them
    ([10], [20], 16, 0),
])
def test_extend_block_tables(native_ops, device, ctx, qlens, page, spare, dtype):
    from hif8_rocm import kv_cache

    columns = max(-(-(c + n) // page) for c, n in zip(ctx, qlens)) + 1
    table, free, count = _pool(device, ctx, page, columns, spare, len(ctx), dtype)
    want = extend_reference(table.cpu().numpy(), free.cpu().numpy(), spare, ctx, qlens, page, sum(qlens))
    before = free.clone()
    got = kv_cache.extend_block_tables(table, free, count, ctx, block_size=page, query_lens=qlens)
    for g, w in zip((*got, table, count), want):
        assert np.array_equal(g.cpu().numpy().ravel(), np.asarray(w).ravel())
    assert torch.equal(free, before) and [t.dtype for t in got] == [I64, I64, I32, I32]


def test_extend_keeps_pages_and_pads(native_ops, device):
    """Columns that hold a page keep it; a table that is too narrow counts as missing; padding rows get -1."""
    from hif8_rocm import kv_cache

    table, free, count = _pool(device, [20, 40], 16, 4, 8, 1)
    table[0, 2] = 5                               # a page of rejected drafts
    want = extend_reference(table.cpu().numpy(), free.cpu().numpy(), 8, [20, 40], [25, 60], 16, 90)
    loc = torch.tensor([2, 27, 87], dtype=I32, device=device)
    got = kv_cache.extend_block_tables(table, free, count, torch.tensor([20, 40], dtype=I32, device=device),
                                       block_size=16, query_start_loc=loc, total_query_tokens=90, validate=False)
    shifted = [np.concatenate([[-1, -1], np.asarray(w)[:88]]) for w in want[:2]]
    shifted = [np.where(np.arange(90) < 87, w, -1) for w in shifted]
    for g, w in zip((*got, table, count), (*shifted, *want[2:])):
        assert np.array_equal(g.cpu().numpy().ravel(), np.asarray(w).ravel())
    assert got[3].tolist() == [0, 3]


@pytest.mark.parametrize("dtype", [I32, I64])
@pytest.mark.parametrize("held, lens, page, columns, window, sinks", [
    ([0], [0], 16, 3, None, 0), ([40], [17], 16, 5, None, 0), ([100, 64, 7], [100, 0, 8], 16, 9, None, 0),
    ([5000], [4500], 16, 400, 100, 4), ([300, 20, 0], [290, 20, 0], 16, 20, 1, 17), ([3000] * 40, [2990] * 40, 3, 1003, 64, 0),
    ([64], [64], 16, 4, 16, 0), ([64], [64], 16, 4, 17, 0), ([64], [64], 16, 4, 18, 0), ([64], [64], 16, 4, 2 ** 40, 0),
    ([33000], [32000], 1, 33001, 5, 2 ** 40),
])
def test_release_blocks(native_ops, device, held, lens, page, columns, window, sinks, dtype):
    from hif8_rocm import kv_cache

    table, free, count = _pool(device, held, page, columns, 5, len(held), dtype)
    want = release_reference(table.cpu().numpy(), free.cpu().numpy(), 5, lens, page, window, sinks)
    kv_cache.release_blocks(table, free, count, lens, block_size=page, window=window, sinks=sinks)
    for g, w in zip((table, free, count), want):
        assert np.array_equal(g.cpu().numpy().ravel(), np.asarray(w).ravel())
    again = [t.clone() for t in (table, free, count)]
    kv_cache.release_blocks(table, free, count, lens, block_size=page, window=window, sinks=sinks)
    assert all(torch.equal(a, b) for a, b in zip(again, (table, free, count)))


def test_release_onto_a_full_stack(native_ops, device):
    from hif8_rocm import kv_cache

    table, free, count = _pool(device, [400, 300], 4, 120, 5, 1)
    small = free[:20].clone()
    want = release_reference(table.cpu().numpy(), small.cpu().numpy(), 5, [0, 0], 4)
    kv_cache.release_blocks(table, small, count, [0, 0], block_size=4)
    for g, w in zip((table, small, count), want):
        assert np.array_equal(g.cpu().numpy().ravel(), np.asarray(w).ravel())
    assert count.item() == 20


# ----------------------------------------------------------------- together
def _serve(device, seed, graph):
    """Steps of two requests with chains of drafts under a window, all on the device; yields what a step answers."""
    from hif8_rocm import kv_cache

    page, hq, hkv, d, window, sinks, vocab, n = 16, 8, 2, 128, 40, 4, 600, 4
    g = torch.Generator(device=device).manual_seed(seed)
    kc, vc = kv_cache.Hif8KVCacheLayout(num_blocks=40, block_size=page, num_kv_heads=hkv, head_size=d).allocate(device)
    table = torch.full((2, 20), -1, dtype=I32, device=device)
    free, count = torch.randperm(40, generator=g, device=device).to(I32), torch.tensor([40], dtype=I32, device=device)
    ctx = torch.zeros(2, dtype=I32, device=device)
    ks = torch.full((hkv,), 0.01, device=device)
    loc = torch.tensor([0, n, 2 * n], dtype=I32, device=device)
    key, value = (torch.empty(2 * n, hkv, d, dtype=torch.bfloat16, device=device) for _ in range(2))
    query = torch.empty(2 * n, hq, d, dtype=torch.bfloat16, device=device)
    probs, draft = (torch.empty(2 * n, vocab, device=device) for _ in range(2))
    tokens, u = torch.empty(2 * n, dtype=I64, device=device), torch.empty(2 * n, device=device)
    out = {}

    def inputs():
        for t in (key, value, query):
            t.copy_(torch.randn(t.shape, generator=g, device=device))
        logits = 2 * torch.randn(2 * n, vocab, generator=g, device=device)
        probs.copy_(torch.softmax(logits, -1))
        draft.copy_(torch.softmax(logits.roll(1, 0) + 0.3 * torch.randn(logits.shape, generator=g, device=device), -1))
        tokens.copy_(torch.multinomial(draft, 1, generator=g)[:, 0])
        u.copy_(torch.rand(2 * n, generator=g, device=device))

    def step():
        slots, positions, lens, missing = kv_cache.extend_block_tables(
            table, free, count, ctx, block_size=page, query_start_loc=loc, total_query_tokens=2 * n, validate=False)
        kv_cache.write_kv_cache(key, value, kc, vc, slots, ks, ks, validate=False)
        attn = kv_cache.paged_attention(query, kc, vc, table, lens, scale=0.1, query_start_loc=loc, max_query_len=n,
                                        max_seq_len=320, window=window, sinks=sinks, validate=False)
        path, counts, drawn = kv_cache.verify_drafts(probs, tokens, u, draft_probs=draft, query_start_loc=loc,
                                                     max_query_len=n, validate=False)
        before = ctx.clone()
        ctx.copy_(kv_cache.accept_drafts(kc, vc, table, ctx, path, counts, validate=False))
        kv_cache.release_blocks(table, free, count, ctx, block_size=page, window=window, sinks=sinks, validate=False)
        out.update(slots=slots, positions=positions, lens=lens, missing=missing, attn=attn, path=path, counts=counts,
                   drawn=drawn, before=before)

    inputs()
    if graph:
        step()                                    # warms up; the state goes back
        table.fill_(-1)
        free.copy_(torch.randperm(40, generator=torch.Generator(device=device).manual_seed(seed), device=device).to(I32))
        count.fill_(40)
        ctx.zero_()
        kc.zero_()
        vc.zero_()
        g.manual_seed(seed)
        torch.randperm(40, generator=g, device=device)
        inputs()
        cuda_graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(cuda_graph):
            step()
    for i in range(30):
        if i:
            inputs()
        if graph:
            cuda_graph.replay()
        else:
            step()
        torch.cuda.synchronize()
        yield {**{k: v.clone() for k, v in out.items()}, "kc": kc.clone(), "vc": vc.clone(), "table": table.clone(),
               "free": free.clone(), "count": count.clone(), "ctx": ctx.clone(), "query": query.clone(), "probs": probs,
               "draft": draft, "tokens": tokens, "u": u}


def test_steps_together(native_ops, device):
    """extend -> write -> attention -> verify -> accept -> release: pages are neither lost nor shared, attention
    is that of the table as it stands, and a captured step answers as an eager one."""
    n, lens = 4, [0, 0]
    for i, (s, r) in enumerate(zip(_serve(device, 11, False), _serve(device, 11, True))):
        for k in ("attn", "path", "counts", "drawn", "table", "free", "count", "ctx", "kc", "vc", "slots", "positions"):
            assert torch.equal(s[k], r[k]), (i, k)
        assert s["missing"].tolist() == [0, 0] and s["before"].tolist() == lens
        want = verify_reference(*(s[k].cpu().numpy() for k in ("probs", "draft", "tokens")), None, s["u"].cpu().numpy(),
                                [n, n], n)
        for k, w in zip(("path", "counts", "drawn"), want):
            assert np.array_equal(s[k].cpu().numpy(), w)
        lens = [a + int(c) for a, c in zip(lens, want[1])]
        assert s["ctx"].tolist() == lens
        table, count = s["table"].cpu().numpy(), int(s["count"])
        out = np.sort(np.concatenate([table[table >= 0], s["free"].cpu().numpy()[:count]]))
        assert np.array_equal(out, np.arange(40))
        for b, size in enumerate(lens):
            kept = [j for j in range(20) if j * 16 < size and (j * 16 < 4 or (j + 1) * 16 > size + 1 - 40)]
            assert np.array_equal(np.flatnonzero(table[b] >= 0), kept)
        assert not s["attn"].isnan().any()
    assert lens[0] > 45


def test_attention_of_a_step_reads_the_extended_table(native_ops, device):
    from hif8_rocm import kv_cache

    page, hkv, d = 16, 2, 64
    kc, vc = kv_cache.Hif8KVCacheLayout(num_blocks=30, block_size=page, num_kv_heads=hkv, head_size=d).allocate(device)
    table, free, count = _pool(device, [0, 0], page, 14, 30, 2)
    ctx, scale = [0, 0], torch.full((hkv,), 0.01, device=device)
    for step, qlens in enumerate(([200, 3], [1, 1], [5, 90], [1, 0])):
        slots, _, lens, _ = kv_cache.extend_block_tables(table, free, count, ctx, block_size=page, query_lens=qlens)
        total = sum(qlens)
        kv_cache.write_kv_cache(randn((total, hkv, d), step).to(device), randn((total, hkv, d), step + 9).to(device), kc,
                                vc, slots, scale, scale)
        q = randn((total, 4, d), step + 20)
        out = kv_cache.paged_attention(q.to(device), kc, vc, table, lens, scale=0.125, query_lens=qlens, window=60, sinks=4)
        want, bound = window_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.cpu().numpy(),
                                       lens.tolist(), qlens, 60, 4, 0.125, torch.bfloat16)
        _near(out, want, bound)
        ctx = lens.tolist()
        kv_cache.release_blocks(table, free, count, ctx, block_size=page, window=60, sinks=4)


def test_a_verified_tree_is_accepted(native_ops, device):
    """tree_attention -> verify_drafts -> accept_drafts: the path's rows end behind the context."""
    from hif8_rocm import kv_cache

    ctx, qlens, vocab = [33, 70], [9, 6], 800
    case = _verify_case(qlens, vocab, 2, tree=True, peaked=4.0)
    probs, _, tokens, parents, u = case
    u[:] *= 0.3
    kc, vc, table = build_cache(device, [c + n for c, n in zip(ctx, qlens)], 2, 64, 16, 5)
    mask = np.zeros((15, 9), dtype=bool)
    for at, n in ((0, 9), (9, 6)):
        mask[at:at + n, :n] = ancestors(parents[at:at + n].tolist())
    q = randn((15, 4, 64), 6)
    out = kv_cache.tree_attention(q.to(device), kc, vc, table.to(device), ctx, torch.from_numpy(mask).to(device),
                                  scale=0.1, query_lens=qlens)
    want, bound = tree_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), ctx, qlens, mask,
                                 0.1, torch.bfloat16)
    _near(out, want, bound)
    path, counts, _ = _verify(device, case, qlens)
    assert counts.max() > 1
    before = kc.clone()
    lens = kv_cache.accept_drafts(kc, vc, table.to(device), ctx, path, counts)
    assert lens.tolist() == [c + int(k) for c, k in zip(ctx, counts)]
    for b in range(2):
        for i in range(int(counts[b])):
            frm, to = ctx[b] + int(path[b, i]), ctx[b] + i
            assert torch.equal(kc[int(table[b, to // 16]), to % 16], before[int(table[b, frm // 16]), frm % 16])


def test_two_streams_at_once(native_ops, device):
    from hif8_rocm import kv_cache

    lens, qlens = [900, 400], [130, 2]
    kc, vc, table = build_cache(device, lens, 4, 128, 16, 8)
    table = table.to(device)
    q = [randn((132, 16, 128), s).to(device) for s in (1, 2)]
    case = [_verify_case([5, 5], 30000, s, sampled=True) for s in (1, 2)]
    dev = [[torch.from_numpy(x).to(device) for x in c if x is not None] for c in case]

    def call(i):
        o = kv_cache.paged_attention(q[i], kc, vc, table, lens, scale=0.1, query_lens=qlens, window=300, sinks=4)
        p, d, t, u = dev[i]
        return (o, *kv_cache.verify_drafts(p, t, u, draft_probs=d, query_lens=[5, 5]))

    want = [call(i) for i in (0, 1)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(call(i))
    torch.cuda.synchronize()
    for i in (0, 1):
        for g in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(g, want[i]))
