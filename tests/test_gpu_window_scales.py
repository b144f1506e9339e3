"""Attention within a sliding window where V's row scales lie far apart: requests of few query rows and of
many against float64, every query row by what it sees itself (tests/_window_rows.py)."""

import math

import numpy as np
import pytest
import torch

from _kv import build_cache, randn
from _rows import DECODE
from _window_rows import window_by_row

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16
# Query rows per request at four query heads per KV head: a token, drafts, and more than 256 (token, head) rows.
ROWS = ([1, 1], [6, 3], [20, 9], [130, 70], [70, 2])


def _put_scales(cache, scales):
    cache.view(-1, cache.shape[-1])[:, -4:] = scales.float().reshape(-1, 1).view(torch.uint8).to(cache.device)


def _put(cache, table, b, t, scale):
    """Every head's scale of request b's row t."""
    page = cache.shape[1]
    _put_scales(cache[int(table[b, t // page]), t % page], torch.full((cache.shape[2],), scale))


def _check(kc, vc, table, lens, qlens, window, sinks, q, scale):
    from hif8_rocm import kv_cache

    print(f"lens={lens} rows={qlens} window={window} sinks={sinks} q={tuple(q.shape)} page={kc.shape[1]} {q.dtype}", flush=True)
    device = kc.device
    out = kv_cache.paged_attention(q.to(device), kc, vc, table.to(device), lens, scale=scale, query_lens=qlens,
                                   window=window, sinks=sinks)
    want, bound = window_by_row(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), lens, qlens, window,
                                sinks, scale, q.dtype)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - want) / np.maximum(bound, 1e-300)
    print(f"  worst error / bound {over.max(initial=0.0):.3f}", flush=True)
    assert (over <= 1.0).all(), float(over.max())


def _cache(device, lens, hkv, d, page, seed):
    return build_cache(device, lens, hkv, d, page, seed, scales=([0.9] * hkv, [0.4] * hkv))


@pytest.mark.parametrize("power", [18, 24, 30, 60, 116])
@pytest.mark.parametrize("qlens", ROWS)
@pytest.mark.parametrize("d, page", [(64, 32), (128, 16), (256, 128)])
def test_scales_that_are_not_seen(native_ops, device, d, page, qlens, power):
    """Large finite scales just before the first row's window, behind the length and, where the output's type
    holds what they give, in tokens that only the last rows see."""
    lens, window, sinks, hkv = [400, 333], 60, 20, 2
    for dtype in (BF16, FP16):
        kc, vc, table = _cache(device, lens, hkv, d, page, d + power)
        for b, (size, n) in enumerate(zip(lens, qlens)):
            low = size - n + 1 - window
            hidden = [low - 1, low - 7, low - 33, sinks, sinks + 1] + [t for t in (size, size + 3) if t < -(-size // page) * page]
            for t in hidden + ([size - 1, size - 1 - n // 3] if n > 1 and dtype == BF16 else []):
                _put(vc, table, b, t, math.copysign(2.0 ** power, 1 - 2 * (t % 2)))
        _check(kc, vc, table, lens, qlens, window, sinks, randn((sum(qlens), 4 * hkv, d), 3, 1.0, dtype), 1 / math.sqrt(d))


@pytest.mark.parametrize("window, sinks", [(70, 9), (1000, 0)])
@pytest.mark.parametrize("qlens", ROWS)
@pytest.mark.parametrize("d, page", [(64, 16), (128, 32), (256, 128)])
def test_scales_far_apart(native_ops, device, d, page, qlens, window, sinks):
    """Row scales of V from 2^-100 to 2^100, of both signs, zeros among them; then from 2^-12 to 2^12 in fp16."""
    lens, hkv = [333, 150], 2
    kc, vc, table = _cache(device, lens, hkv, d, page, d + 1)
    g = torch.Generator().manual_seed(d)
    n = vc.shape[0] * vc.shape[1] * hkv
    for dtype, power in ((BF16, 100), (FP16, 12)):
        s = (2.0 ** (2 * power * torch.rand(n, generator=g) - power)) * torch.randint(-1, 2, (n,), generator=g).float()
        _put_scales(vc, s)
        _check(kc, vc, table, lens, qlens, window, sinks, randn((sum(qlens), 4 * hkv, d), d + 2, 1.0, dtype), 1 / math.sqrt(d))


@pytest.mark.parametrize("power", [-100, -70, -40, 40, 70, 100])
@pytest.mark.parametrize("qlens", ROWS)
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scales_all_small_or_all_large(native_ops, device, d, qlens, power):
    lens, hkv = [200, 150], 2
    kc, vc, table = _cache(device, lens, hkv, d, 16, d + 1)
    n = vc.shape[0] * vc.shape[1] * hkv
    _put_scales(vc, 2.0 ** (power + 3 * torch.rand(n, generator=torch.Generator().manual_seed(d))))
    for window in (1, 90):
        _check(kc, vc, table, lens, qlens, window, 4, randn((sum(qlens), 4 * hkv, d), 3), 1 / math.sqrt(d))


@pytest.mark.parametrize("small", [0.0, 2.0 ** -120, -2.0 ** -64, 1.0])
@pytest.mark.parametrize("large", [2.0 ** 63, -2.0 ** 100, 2.0 ** 116])
@pytest.mark.parametrize("qlens", [[6], [130]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_two_rows_of_one_weight_and_distant_scales(native_ops, device, d, qlens, small, large):
    """All logits zero, V zero but in two rows, seen together or apart."""
    lens, hkv = [160], 2
    kc, vc, table = _cache(device, lens, hkv, d, 16, d)
    kc.view(-1, d + 4)[:, :d] = 0
    for first, second in ((small, large), (large, small)):
        _put_scales(vc, torch.zeros(vc.numel() // (d + 4)))
        _put(vc, table, 0, 3, first)
        _put(vc, table, 0, 149, second)
        for window in (8, 40, 200):
            _check(kc, vc, table, lens, qlens, window, 5, randn((sum(qlens), 4 * hkv, d), 6), 1 / math.sqrt(d))


@pytest.mark.parametrize("qlens", [[5], [130]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scales_that_grow_along_the_rows(native_ops, device, d, qlens):
    """Scales that rise or fall over 2^180, alone and against weights that do the opposite."""
    lens, hkv, page = [900], 2, 64
    kc, vc, table = _cache(device, lens, hkv, d, page, d)
    at = torch.zeros(vc.shape[0] * page)
    at[(table[0, :15, None].long() * page + torch.arange(page)).flatten()] = torch.arange(960).float()
    for rise in (0.2, -0.2):
        _put_scales(vc, (2.0 ** (rise * (at - 450)))[:, None].expand(-1, hkv).contiguous())
        for window in (100, 1000):
            _check(kc, vc, table, lens, qlens, window, 3, randn((sum(qlens), 4 * hkv, d), 7), 1 / math.sqrt(d))
    kc.view(-1, hkv, d + 4)[:, :, :d] = 0
    kc.view(-1, hkv, d + 4)[:, :, 0] = 8
    assert DECODE[8] == 1.0
    q = torch.zeros(sum(qlens), 4 * hkv, d, dtype=BF16)
    q[..., 0] = 1.0
    for rise in (0.12, -0.12):
        _put_scales(vc, (2.0 ** (rise * (at - 450)))[:, None].expand(-1, hkv).contiguous())
        _put_scales(kc, (-math.log(2) * rise * (at - 450))[:, None].expand(-1, hkv).contiguous())
        _check(kc, vc, table, lens, qlens, 1000, 3, q, 1.0)


@pytest.mark.parametrize("qlens", [[6], [130]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_small_weights_beside_a_large_one_of_an_empty_v(native_ops, device, d, qlens):
    """A first row that draws nearly all attention and whose V is zero: the output is what the others, at 2^-27
    to 2^-25 each, add up to."""
    lens, hkv, page = [300], 2, 16
    kc, vc, table = _cache(device, lens, hkv, d, page, d)
    kc.view(-1, hkv, d + 4)[:, :, :d] = 0
    kc.view(-1, hkv, d + 4)[:, :, 0] = 8
    first = int(table[0, 0])
    _put_scales(kc, -math.log(2) * (25 + 2 * torch.rand(kc.shape[0] * page, hkv, generator=torch.Generator().manual_seed(d))))
    kc[first, 0, :, 0] = 0
    vc[first, 0, :, :d] = 0
    q = torch.zeros(sum(qlens), 4 * hkv, d, dtype=BF16)
    q[..., 0] = 1.0
    _check(kc, vc, table, lens, qlens, 200, 1, q, 1.0)


@pytest.mark.parametrize("small", [0.0, 2.0 ** -126, 1.0])
@pytest.mark.parametrize("qlens", [[6], [130]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_a_scale_of_the_largest_exponent(native_ops, device, d, qlens, small):
    """Scales of -1.75 x 2^127 over codes of +-0.5, every fifth row, among others of the same weight."""
    lens, hkv = [150], 2
    kc, vc, table = _cache(device, lens, hkv, d, 16, d)
    kc.view(-1, d + 4)[:, :d] = 0
    assert DECODE[24] == 0.5 and DECODE[24 + 128] == -0.5
    codes = torch.randint(0, 2, (vc.numel() // (d + 4), d), generator=torch.Generator().manual_seed(d))
    vc.view(-1, d + 4)[:, :d] = (24 + 128 * codes).to(torch.uint8).to(device)
    _put_scales(vc, torch.full((vc.numel() // (d + 4),), small))
    for t in range(2, 150, 5):
        _put(vc, table, 0, t, -1.75 * 2.0 ** 127)
    _check(kc, vc, table, lens, qlens, 12, 0, randn((sum(qlens), 4 * hkv, d), 5), 1 / math.sqrt(d))


@pytest.mark.parametrize("scales", ["rise", "fall", "far", "far and near", "zeros", "ordinary"])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_scales_over_long_runs(native_ops, device, d, scales):
    """Workgroups with dozens of images each: rows whose references move again and again, or not at all."""
    lens, qlens, hkv, page = [2500], [520], 8, 64
    kc, vc, table = _cache(device, lens, hkv, d, page, d)
    n = vc.shape[0] * page
    at = torch.zeros(n)
    where = (table[0, :40, None].long() * page + torch.arange(page)).flatten()[:2500]
    at[where] = torch.arange(2500).float()
    g = torch.Generator().manual_seed(d)
    power = {"rise": 0.06 * (at - 1250), "fall": -0.06 * (at - 1250), "far": 200 * torch.rand(n, generator=g) - 100,
             "far and near": torch.where(at % 97 == 5, 90.0, 3 * torch.rand(n, generator=g)),
             "zeros": torch.where(at % 50 == 5, -math.inf, torch.zeros(n)), "ordinary": 4 * torch.rand(n, generator=g) - 2}[scales]
    _put_scales(vc, (2.0 ** power)[:, None].expand(-1, hkv).contiguous())
    _check(kc, vc, table, lens, qlens, 1400, 4, randn((520, 2 * hkv, d), 3), 3 / math.sqrt(d))


@pytest.mark.parametrize("qlens", [[1, 1], [6, 3], [130, 70]])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_calls_repeat_themselves(native_ops, device, d, qlens):
    from hif8_rocm import kv_cache

    lens = [2000, 1300]
    kc, vc, table = build_cache(device, lens, 4, d, 16, d, mixed=True)
    for dtype in (BF16, FP16):
        q = randn((sum(qlens), 16, d), 3, 1.0, dtype).to(device)
        outs = [kv_cache.paged_attention(q, kc, vc, table.to(device), lens, scale=0.1, query_lens=qlens, window=700, sinks=4)
                for _ in range(20)]
        assert all(torch.equal(o, outs[0]) for o in outs[1:])
