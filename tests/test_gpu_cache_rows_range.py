"""The operators on rows of the HiF8 KV cache where a row is nobody's, where row
scales or weights lie far apart, and where a call falls to the any-shape
kernels: against float64 (tests/_rows.py)."""

import math

import numpy as np
import pytest
import torch

from _kv import build_cache, randn
from _rows import DECODE, Softmax, tree_reference

pytestmark = pytest.mark.gpu
I32 = torch.int32
TOP = 8


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


def _rows(cache, table, b, n):
    """float64 codes [n, Hkv, D] and row scales [n, Hkv] of request b's first n rows (all in the cache)."""
    raw = cache.cpu().numpy()
    bs = raw.shape[1]
    t = np.arange(n)
    raw = raw[table.numpy()[b, t // bs], t % bs]
    return DECODE[raw[..., :-4]], np.ascontiguousarray(raw[..., -4:]).view(np.float32)[..., 0].astype(np.float64)


def _attention(q, kc, vc, table, lens, rows, sees, scale, dtype):
    """(out, bound, weights, weights' bound) of `rows[b]` query rows per request over lens[b] cached rows.

    P = p s 2^k (s: the V row's scale) has 11 significant bits (2^-11 of p |V|), or 2^-25 absolutely where it is
    subnormal; k puts the largest p |s| at 2^TOP / 4 at least, so that is 2^-(23 + TOP) max(p |s|) |code|."""
    hq, hkv, group = q.shape[1], kc.shape[2], q.shape[1] // kc.shape[2]
    half, tiny = torch.finfo(dtype).eps / 2, torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
    out = np.zeros((sum(rows), hq, vc.shape[3] - 4))
    bound, sums = np.zeros_like(out), np.zeros((len(lens), hkv, max(lens)))
    sums_bound = np.zeros_like(sums)
    at = 0
    for b, (n, m) in enumerate(zip(lens, rows)):
        (k, ks), (v, vs) = _rows(kc, table, b, n), _rows(vc, table, b, n)
        for h in range(hq):
            g = h // group
            sm = Softmax(q[at:at + m, h], k[:, g] * ks[:, g, None], sees(b, n, m), scale)
            value = v[:, g] * vs[:, g, None]
            mag = sm.p @ np.abs(value)
            y = sm.p @ value
            most = (sm.p * np.abs(vs[:, g])).max(axis=1, initial=0.0)
            out[at:at + m, h] = y
            bound[at:at + m, h] = half * np.abs(y) + (2.0 ** -11 + sm.rel) * mag + tiny + \
                2.0 ** -(23 + TOP) * most[:, None] * np.abs(v[:, g]).sum(axis=0)
            sums[b, g, :n] += sm.p.sum(axis=0)
            sums_bound[b, g, :n] += (sm.rel + 2.0 ** -24 * group) * sm.p.sum(axis=0) + 2.0 ** -126
        at += m
    return out, bound, sums, sums_bound


def _near(got, want, bound):
    got = got.double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - want) / np.maximum(bound, 1e-300)
    print(f"  worst error / bound {over.max(initial=0.0):.3f}", flush=True)
    assert (over <= 1.0).all(), float(over.max())


def _put_scales(cache, scales):
    cache.view(-1, cache.shape[-1])[:, -4:] = scales.reshape(-1, 1).view(torch.uint8).to(cache.device)


def _tree_and_decode(device, kc, vc, table, lens, drafts, q, scale, dtype):
    """Both operators over the same rows against the formula: drafts that see all of the request, one row that
    keeps its weights."""
    from hif8_rocm import kv_cache

    assert q.dtype == dtype   # the output's type, whose rounding the bound counts
    batch, hkv = len(lens), kc.shape[2]
    everything = lambda b, n, m: np.ones((m, n), dtype=bool)  # noqa: E731
    args = dict(scale=scale)
    mask = torch.ones(batch * drafts, drafts, dtype=torch.bool, device=device)
    out = kv_cache.tree_attention(q.to(device), kc, vc, table.to(device), [n - drafts for n in lens], mask,
                                  query_lens=[drafts] * batch, **args)
    qn = q.double().numpy()
    want, bound, _, _ = _attention(qn, kc, vc, table, lens, [drafts] * batch, everything, scale, dtype)
    _near(out, want, bound)
    w = torch.zeros(batch, hkv, max(lens), device=device)
    q1 = q[::drafts].contiguous()
    out = kv_cache.paged_decode_attention_weights(q1.to(device), kc, vc, table.to(device), lens, w, **args)
    want, bound, sums, sums_bound = _attention(q1.double().numpy(), kc, vc, table, lens, [1] * batch, everything, scale, dtype)
    _near(out, want, bound)
    _near(w, sums, sums_bound)


@pytest.mark.parametrize("d, hq, hkv, bs, drafts", [(256, 16, 4, 128, 3), (256, 16, 4, 128, 9), (128, 24, 8, 16, 31),
                                                    (64, 4, 4, 32, 5), (96, 4, 2, 20, 3)])
def test_v_scales_far_apart(native_ops, device, d, hq, hkv, bs, drafts):
    """Row scales of V from 2^-100 to 2^100, of both signs, zeros among them: every row counts in the softmax sum."""
    g = torch.Generator().manual_seed(d)
    lens = [40, 333]
    kc, vc, table = build_cache(device, lens, hkv, d, bs, d + 1, scales=([0.9] * hkv, [0.4] * hkv))
    n = vc.shape[0] * vc.shape[1] * hkv
    s = (2.0 ** (200 * torch.rand(n, generator=g) - 100)) * torch.randint(-1, 2, (n,), generator=g).float()
    _put_scales(vc, s)
    print(f"scales d={d} hq={hq} drafts={drafts}", flush=True)
    _tree_and_decode(device, kc, vc, table, lens, drafts, randn((len(lens) * drafts, hq, d), d + 2), 1 / math.sqrt(d),
                     torch.bfloat16)


@pytest.mark.parametrize("small", [0.0, 2.0 ** -120, -2.0 ** -64, 1.0])
@pytest.mark.parametrize("large", [2.0 ** 63, -2.0 ** 100, 2.0 ** 116])
@pytest.mark.parametrize("d", [64, 128, 256, 96])
def test_two_rows_of_one_weight_and_distant_scales(native_ops, device, d, small, large):
    """Two rows with the same logit: the output is half of the large one (and of the small one)."""
    kc, vc, table = build_cache(device, [2], 2, d, 16, d, scales=([0.9] * 2, [0.4] * 2))
    kc.view(-1, d + 4)[:, :d] = 0
    for t, s in ((0, small), (1, large)):
        _put_scales(vc[int(table[0, 0]), t], torch.full((2,), s))
    print(f"two rows d={d} scales {small:g} {large:g}", flush=True)
    _tree_and_decode(device, kc, vc, table, [2], 1, randn((1, 4, d), 5), 1 / math.sqrt(d), torch.bfloat16)
    _put_scales(vc[int(table[0, 0]), 0], torch.full((2,), large))
    _put_scales(vc[int(table[0, 0]), 1], torch.full((2,), small))
    _tree_and_decode(device, kc, vc, table, [2], 1, randn((1, 4, d), 6), 1 / math.sqrt(d), torch.bfloat16)


@pytest.mark.parametrize("d", [64, 256])
def test_scales_that_grow_along_the_rows(native_ops, device, d):
    """Weights fall while scales rise, tile by tile: what was summed first keeps its part."""
    lens, hkv = [900], 2
    kc, vc, table = build_cache(device, lens, hkv, d, 64, d, scales=([0.9] * hkv, [0.4] * hkv))
    at = torch.full((vc.shape[0] * vc.shape[1],), 0)
    at[(table[0, :15, None].long() * 64 + torch.arange(64)).flatten()] = torch.arange(960)
    for rise in (0.2, -0.2):
        _put_scales(vc, (2.0 ** (rise * (at - 450).float()))[:, None].expand(-1, hkv).contiguous())
        _tree_and_decode(device, kc, vc, table, lens, 5, randn((5, 4, d), 7), 1 / math.sqrt(d), torch.bfloat16)
    # Weights that fall as the scales rise, over 2^108 (a weight below 2^-126 of the largest is zero in float32).
    kc.view(-1, hkv, d + 4)[:, :, :d] = 0
    kc.view(-1, hkv, d + 4)[:, :, 0] = 8
    assert DECODE[8] == 1.0
    q = torch.zeros(5, 4, d, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    for rise in (0.12, -0.12):
        by = rise * (at - 450).float()
        _put_scales(vc, (2.0 ** by)[:, None].expand(-1, hkv).contiguous())
        _put_scales(kc, (-math.log(2) * by)[:, None].expand(-1, hkv).contiguous())
        _tree_and_decode(device, kc, vc, table, lens, 5, q, 1.0, torch.bfloat16)


@pytest.mark.parametrize("d, hq, hkv, drafts", [(256, 4, 4, 1), (256, 16, 4, 5), (256, 16, 2, 4), (128, 16, 2, 8), (64, 8, 4, 3)])
def test_small_weights_beside_a_large_one_of_an_empty_v(native_ops, device, d, hq, hkv, drafts):
    """A first row that draws nearly all attention and whose V is zero: the output is what the others, at 2^-27
    to 2^-25 each, add up to."""
    lens = [300] * 130                            # more requests than workers: a request's rows lie in one part
    kc, vc, table = build_cache(device, lens, hkv, d, 16, d + hq, scales=([0.9] * hkv, [0.4] * hkv))
    g = torch.Generator().manual_seed(d)
    kc.view(-1, hkv, d + 4)[:, :, :d] = 0
    kc.view(-1, hkv, d + 4)[:, :, 0] = 8
    assert DECODE[8] == 1.0
    first = table[:, 0].long().to(device)
    logit = -math.log(2) * (25 + 2 * torch.rand(kc.shape[0] * 16, hkv, generator=g))
    _put_scales(kc, logit)
    kc[first, 0, :, 0] = 0                        # logit 0
    vc[first, 0, :, :d] = 0
    q = torch.zeros(len(lens) * drafts, hq, d, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    print(f"sink d={d} hq={hq} drafts={drafts}", flush=True)
    _tree_and_decode(device, kc, vc, table, lens, drafts, q, 1.0, torch.bfloat16)


@pytest.mark.parametrize("d, hq, hkv, bs", [(256, 16, 4, 128), (128, 24, 8, 16), (64, 8, 2, 16), (96, 4, 2, 20)])
def test_infinite_v_under_small_weights(native_ops, device, d, hq, hkv, bs):
    """Infinite codes in context rows: an infinity of their sign where the weight is above 2^-31 of the row's
    largest, no finite number where it is below, and the other dims as if the codes were finite."""
    from hif8_rocm import kv_cache

    lens, drafts = [200], 3
    kc, vc, table = build_cache(device, lens, hkv, d, bs, d, scales=([0.9] * hkv, [0.4] * hkv))
    kc.view(-1, hkv, d + 4)[:, :, :d] = 0
    kc.view(-1, hkv, d + 4)[:, :, 0] = 8
    q = torch.zeros(drafts, hq, d, dtype=torch.bfloat16)
    q[..., 0] = 1.0
    at = {0: 0.0, 3: -20.0, 9: -29.0, 150: -60.0}     # base-2 logits; every other row 2^-40
    _put_scales(kc, torch.full((kc.shape[0] * bs, hkv), -40 * math.log(2)))
    plain = vc.clone()
    for t, x in at.items():
        blk, row = int(table[0, t // bs]), t % bs
        _put_scales(kc[blk, row], torch.full((hkv,), x * math.log(2)))
        if t:
            vc[blk, row, :, t // 3] = 0xEF if t == 9 else 0x6F
    mask = torch.ones(drafts, drafts, dtype=torch.bool, device=device)
    w = torch.zeros(1, hkv, 200, device=device)
    print(f"infinite V d={d}", flush=True)
    for call in (lambda v: kv_cache.tree_attention(q.to(device), kc, v, table.to(device), [197], mask, scale=1.0,
                                                   query_lens=[drafts]),
                 lambda v: kv_cache.paged_decode_attention_weights(q[:1].to(device), kc, v, table.to(device), lens, w,
                                                                   scale=1.0)):
        got, want = call(vc), call(plain)
        dims = torch.ones(d, dtype=torch.bool)
        dims[[1, 3, 50]] = False
        assert torch.equal(got[..., dims.to(device)], want[..., dims.to(device)]) and torch.isfinite(want).all()
        assert (got[..., 1] == math.inf).all() and (got[..., 3] == -math.inf).all()
        assert not torch.isfinite(got[..., 50]).any()


@pytest.mark.parametrize("lens", [[512] * 4, [1024, 1024], [640, 1408], [128] * 5 + [1280, 300], [2048], [100] * 40 + [4000]])
def test_runs_that_end_with_or_within_a_request(native_ops, device, lens):
    """16 workers over 16 tiles or more: parts that end where a worker's run ends, and parts that do not."""
    kc, vc, table = build_cache(device, lens, 32, 64, 16, len(lens))
    print(f"runs lens={lens[:8]}", flush=True)
    for dtype in (torch.bfloat16, torch.float16):
        _tree_and_decode(device, kc, vc, table, lens, 3, randn((len(lens) * 3, 32, 64), 5, 1.0, dtype), 0.125, dtype)


@pytest.mark.parametrize("hq, hkv, d, bs", [(16, 4, 256, 128), (24, 8, 128, 16), (8, 8, 64, 32), (6, 2, 20, 12)])
def test_requests_of_a_batch_are_what_they_are_alone(native_ops, device, hq, hkv, d, bs):
    """A batch against float64, and every request of it against a call of its own."""
    from hif8_rocm import kv_cache

    ctx, qlens = [3000, 40, 0, 517], [30, 6, 3, 1]
    lens = [c + n for c, n in zip(ctx, qlens)]
    kc, vc, table = build_cache(device, lens, hkv, d, bs, 11)
    q = randn((sum(qlens), hq, d), 12)
    mask = np.random.default_rng(13).random((sum(qlens), max(qlens))) < 0.4
    starts = np.cumsum([0] + qlens)

    def sees(b, n, m):
        return np.concatenate([np.ones((m, ctx[b]), dtype=bool), mask[starts[b]:starts[b + 1], :m]], axis=1)

    def call(rows, which):
        return kv_cache.tree_attention(q[rows].to(device), kc, vc, table[which].to(device), [ctx[b] for b in which],
                                       torch.from_numpy(mask[rows]).to(device), scale=1 / math.sqrt(d),
                                       query_lens=[qlens[b] for b in which])

    print(f"batch and alone d={d}", flush=True)
    want, bound, _, _ = _attention(q.double().numpy(), kc, vc, table, lens, qlens, sees, 1 / math.sqrt(d), q.dtype)
    out = call(slice(0, sum(qlens)), [0, 1, 2, 3])
    _near(out, want, bound)
    for b in range(4):
        rows = slice(int(starts[b]), int(starts[b + 1]))
        alone = call(rows, [b])
        _near(alone, want[rows], bound[rows])
        assert torch.equal(alone, call(rows, [b]))
        _near(alone, out[rows].double().cpu().numpy(), 2 * bound[rows])


@pytest.mark.parametrize("d", [64, 128, 256])
def test_key_weights_of_an_unaligned_query(native_ops, device, d):
    """A query that does not start at 16 bytes: the any-shape kernels, in the workspace of the others."""
    from hif8_rocm import kv_cache

    hq, hkv, lens = 8, 2, [333, 90]
    kc, vc, table = build_cache(device, lens, hkv, d, 32, d)
    w = torch.zeros(2, hkv, 340, device=device)
    for rows in ([1, 1], [70, 33]):
        n = sum(rows)
        flat = randn((1 + n * hq * d,), 3).to(device)
        q = flat[1:].view(n, hq, d)
        assert q.data_ptr() % 16 and q.is_contiguous()
        print(f"unaligned query d={d} rows={rows}", flush=True)
        sees = lambda b, n, m: np.arange(n) <= n - m + np.arange(m)[:, None]  # noqa: E731
        want, bound, sums, sums_bound = _attention(q.double().cpu().numpy(), kc, vc, table, lens, rows, sees, 0.1, q.dtype)
        kv_cache.accumulate_key_weights(q, kc, table.to(device), lens, w, scale=0.1, query_lens=rows, accumulate=False)
        most = 2.0 ** -24 * max(rows) * (hq // hkv) * sums    # the rows' sum in float32
        _near(w[..., :333], sums, sums_bound + most)
        if n == 2:
            w.zero_()
            out = kv_cache.paged_decode_attention_weights(q, kc, vc, table.to(device), lens, w, scale=0.1)
            _near(out, want, bound)
            _near(w[..., :333], sums, sums_bound)


@pytest.mark.parametrize("small", [0.0, 2.0 ** -126, 1.0])
@pytest.mark.parametrize("d", [64, 128, 256, 96])
def test_a_v_scale_of_the_largest_exponent(native_ops, device, d, small):
    """A row scale of -1.75 x 2^127 over codes of +-0.5, beside one of the same weight."""
    kc, vc, table = build_cache(device, [2], 2, d, 16, d, scales=([0.9] * 2, [0.4] * 2))
    kc.view(-1, d + 4)[:, :d] = 0
    assert DECODE[24] == 0.5 and DECODE[24 + 128] == -0.5
    vc.view(-1, d + 4)[:, :d] = 24 + 128 * torch.randint(0, 2, (vc.numel() // (d + 4), d), device=device).to(torch.uint8)
    for at, s in ((0, small), (1, -1.75 * 2.0 ** 127)):
        _put_scales(vc[int(table[0, 0]), at], torch.full((2,), s))
    print(f"largest scale d={d} beside {small:g}", flush=True)
    _tree_and_decode(device, kc, vc, table, [2], 1, randn((1, 4, d), 5), 1 / math.sqrt(d), torch.bfloat16)
