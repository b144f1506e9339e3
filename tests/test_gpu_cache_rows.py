"""Operators on rows of the HiF8 KV cache on the GPU, against their plain forms in
float64 (tests/_rows.py, which derives the bounds): tree attention, acceptance
of drafts, decode attention with key weights, key weights of many rows,
eviction, and a run of them together.  Moved rows, lengths and positions are
compared byte for byte."""

import ctypes
import math

import numpy as np
import pytest
import torch

from _kv import build_cache, randn
from _rows import ancestors, evict_reference, tree_reference, weights_reference
from conftest import PKG_ROOT

pytestmark = pytest.mark.gpu
I32 = torch.int32


def _dev(x, device, dtype=None):
    return torch.as_tensor(np.ascontiguousarray(x) if isinstance(x, np.ndarray) else x, dtype=dtype).to(device)


def _tree_mask(qlens, seed, kind="tree"):
    g = np.random.default_rng(seed)
    width = max(max(qlens), 1)
    mask = np.zeros((sum(qlens), width), dtype=bool)
    row = 0
    for n in qlens:
        if kind == "tree":
            part = ancestors([int(g.integers(-1, i)) if i else -1 for i in range(n)])
        elif kind == "any":
            part = g.random((n, n)) < 0.4
        else:
            part = np.zeros((n, n), dtype=bool)
        mask[row:row + n, :n] = part
        mask[row:row + n, n:] = g.random((n, width - n)) < 0.5   # columns of no draft: not looked at
        row += n
    return mask


def _near(got, want, bound):
    got = got.double().cpu().numpy()
    finite = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want)) and np.array_equal(got[~finite & ~np.isnan(want)], want[~finite & ~np.isnan(want)])
    over = np.abs(got - want)[finite] / np.maximum(bound[finite], 1e-300)
    print(f"  worst error / bound {over.max(initial=0.0):.3f}", flush=True)
    assert (over <= 1.0).all(), float(over.max())


def _tree(device, ctx, qlens, hq, hkv, d, bs, *, seed=0, dv=None, dtype=torch.bfloat16, mixed=False, mask="tree",
          bt_dtype=I32, q_mul=1.0, spoil=None, check=True):
    from hif8_rocm import kv_cache

    lens = [c + n for c, n in zip(ctx, qlens)]
    print(f"tree ctx={ctx[:4]} drafts={qlens[:4]} hq={hq} hkv={hkv} d={d} dv={dv} bs={bs} {dtype}", flush=True)
    kc, vc, table = build_cache(device, lens, hkv, d, bs, seed, dv=dv, bt_dtype=bt_dtype, mixed=mixed)
    q = randn((sum(qlens), hq, d), seed + 1, q_mul, dtype)
    m = _tree_mask(qlens, seed + 2, mask)
    if spoil:
        spoil(kc, vc, table, m)
    out = kv_cache.tree_attention(q.to(device), kc, vc, table.to(device), ctx, torch.from_numpy(m).to(device),
                                  scale=1 / math.sqrt(d), query_lens=qlens, validate=spoil is None)
    torch.cuda.synchronize()
    if check:
        want, bound = tree_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), ctx, qlens,
                                     m, 1 / math.sqrt(d), dtype)
        _near(out, want, bound)
    return out


@pytest.mark.parametrize("ctx, qlens, hq, hkv, d, bs", [
    ([512], [8], 16, 4, 256, 128),
    ([0], [1], 16, 4, 256, 128),                       # a first token and nothing else
    ([1, 0, 63, 64, 65], [1, 3, 1, 2, 64], 16, 4, 256, 128),
    ([100, 31], [15, 17], 8, 2, 128, 16),
    ([700], [33], 8, 8, 64, 32),                       # a KV head per query head
    ([257, 3], [5, 20], 24, 8, 128, 16),               # three query heads per KV head
    ([130], [7], 20, 2, 256, 144),                     # pages of nine sixteens
    ([90, 200], [61, 9], 32, 1, 128, 64),              # one KV head
    ([40], [130], 4, 2, 64, 16),                       # more drafts than one tile of cache rows
    ([2000], [3], 16, 4, 256, 128),                    # several splits
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tree_shapes(native_ops, device, ctx, qlens, hq, hkv, d, bs, dtype):
    _tree(device, ctx, qlens, hq, hkv, d, bs, dtype=dtype, seed=hq + d)


@pytest.mark.parametrize("d, dv, hq, hkv, bs", [(20, 36, 6, 2, 12), (96, 96, 5, 5, 128), (512, 256, 4, 2, 7),
                                                (128, 64, 4, 4, 16), (256, 256, 4, 1, 8), (80, 80, 2, 1, 1)])
def test_tree_any_head_and_page_size(native_ops, device, d, dv, hq, hkv, bs):
    _tree(device, [37, 0], [9, 2], hq, hkv, d, bs, dv=dv, seed=d)


@pytest.mark.parametrize("mixed, bt_dtype, q_mul", [(True, torch.int64, 1.0), (False, torch.int64, 8.0), (True, I32, 8.0)])
def test_tree_row_scales_tables_and_peaked_rows(native_ops, device, mixed, bt_dtype, q_mul):
    for dtype in (torch.bfloat16, torch.float16):
        _tree(device, [300, 129], [20, 5], 16, 4, 256, 128, mixed=mixed, bt_dtype=bt_dtype, q_mul=q_mul, dtype=dtype, seed=5)


@pytest.mark.parametrize("mask", ["any", "none"])
def test_tree_masks_that_are_no_trees(native_ops, device, mask):
    out = _tree(device, [0, 50, 0], [70, 9, 3], 16, 4, 256, 128, mask=mask, seed=6)
    if mask == "none":
        assert not out[:70].any() and not out[79:].any()   # nothing seen: zeros


def test_tree_scales_of_any_size_and_sign(native_ops, device):
    """Sidecars that grow and shrink by 2^40 along the rows, negative and zero ones among them."""
    def spoil(kc, vc, table, m):
        g = torch.Generator().manual_seed(1)
        n = vc.shape[0] * vc.shape[1] * vc.shape[2]
        s = (2.0 ** torch.randint(-30, 10, (n,), generator=g).float()) * torch.randint(-1, 2, (n,), generator=g).float()
        vc.view(n, -1)[:, -4:] = s.view(n, 1).view(torch.uint8).to(vc.device)
        k = torch.where(torch.rand(n, generator=g) < 0.3, -0.01, 0.02) * (torch.rand(n, generator=g) > 0.1)
        kc.view(n, -1)[:, -4:] = k.view(n, 1).view(torch.uint8).to(kc.device)

    for dtype in (torch.bfloat16, torch.float16):
        _tree(device, [200], [10], 8, 2, 128, 16, spoil=spoil, seed=7, dtype=dtype)


def test_tree_rows_that_are_not_seen_may_hold_anything(native_ops, device):
    """NaN and infinite codes and scales in pages behind the last draft, and in drafts that
    only some rows see: the others are as if they were not there, those get what the formula gives."""
    def spoil(kc, vc, table, m):
        for b, (c, n) in enumerate(zip([70, 30], [12, 40])):
            last = c + n
            page = kc.shape[1]
            for t in range(last, (last + page - 1) // page * page):
                blk = int(table[b, t // page])
                kc[blk, t % page] = 0x80
                vc[blk, t % page] = 0x80
        for b, start, c, j, code in ((0, 0, 70, 3, 0x80), (1, 12, 30, 5, 0x6F), (1, 12, 30, 33, 0xEF)):
            blk, at = int(table[b, (c + j) // page]), (c + j) % page
            vc[blk, at, :, 1:200:7] = code
            if code == 0x80:
                kc[blk, at, :, 10] = code

    _tree(device, [70, 30], [12, 40], 16, 4, 256, 128, spoil=spoil, seed=8, mask="any")


def test_tree_nan_scales_of_unseen_drafts(native_ops, device):
    def spoil(kc, vc, table, m):
        blk = int(table[0, 0])
        for cache, value in ((kc, math.nan), (vc, math.inf)):
            cache[blk, 22, :, -4:] = torch.tensor([value]).view(torch.uint8).to(cache.device)
        m[:, 2] = False

    _tree(device, [20], [12], 8, 2, 128, 128, spoil=spoil, seed=9)


def test_tree_blocks_outside_the_cache_are_left_out(native_ops, device):
    def spoil(kc, vc, table, m):
        table[0, 1], table[1, 0] = -1, 1 << 20

    _tree(device, [400, 100], [9, 30], 16, 4, 256, 128, spoil=spoil, seed=10)


def test_tree_repeats_itself_and_matches_rows_alone(native_ops, device):
    a = _tree(device, [3000, 40], [30, 6], 16, 4, 256, 128, seed=11, check=False)
    assert torch.equal(a, _tree(device, [3000, 40], [30, 6], 16, 4, 256, 128, seed=11, check=False))


def test_tree_rows_outside_every_request_stay(native_ops, device):
    """Through the C entry: query rows before the first and behind the last request are not written."""
    lib = ctypes.CDLL(str(PKG_ROOT / "hif8_rocm" / "libhif8_rocm.so"))
    lib.hif8_last_error.restype = ctypes.c_char_p
    size = lib.hif8_tree_attention_workspace_size
    size.argtypes, size.restype = [ctypes.c_int64] * 9, ctypes.c_size_t
    i64, ptr, i32 = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int
    lib.hif8_tree_attention.argtypes = [ptr, i32, ptr, ptr] + [i64] * 5 + [ptr, i32, i64, ptr, ptr, ptr] + [i64] * 6 + \
        [ctypes.c_float, ptr, ptr, ctypes.c_size_t, ptr]
    for d, bs in ((256, 128), (96, 20)):
        kc, vc, table = build_cache(device, [210], 4, d, bs, 12)
        q = randn((14, 16, d), 13).to(device)
        loc = torch.tensor([2, 12], dtype=I32, device=device)
        ctx = torch.tensor([200], dtype=I32, device=device)
        mask = torch.ones(14, 10, dtype=torch.bool, device=device)
        table = table.to(device)
        out = torch.full((14, 16, d), 7.0, dtype=torch.bfloat16, device=device)
        need = size(1, 16, 4, d, d, bs, 14, 10, 210)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        p = lambda t: ctypes.c_void_p(t.data_ptr())  # noqa: E731
        st = lib.hif8_tree_attention(p(q), 1, p(kc), p(vc), kc.shape[0], bs, 4, d, d, p(table), 0, table.shape[1], p(loc),
                                     p(ctx), p(mask), 10, 1, 16, 14, 10, 210, 0.1, p(out), p(ws), need,
                                     ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
        torch.cuda.synchronize()
        assert st == 0, lib.hif8_last_error()
        assert (out[:2] == 7).all() and (out[12:] == 7).all() and not (out[2:12] == 7).all()


def test_tree_unaligned_query_and_strided_mask(native_ops, device):
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, [90], 2, 128, 16, 14)
    flat = randn((1 + 10 * 4 * 128,), 15).to(device)
    q = flat[1:].view(10, 4, 128)
    assert q.data_ptr() % 16
    m = torch.from_numpy(_tree_mask([10], 16)).to(device)
    wide = torch.zeros(10, 20, dtype=torch.bool, device=device)
    wide[:, ::2] = m
    args = dict(scale=0.1, query_lens=[10])
    a = kv_cache.tree_attention(q, kc, vc, table.to(device), [80], wide[:, ::2], **args)
    b = kv_cache.tree_attention(q.clone(), kc, vc, table.to(device), [80], m, **args)
    want, bound = tree_reference(q.double().cpu().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), [80], [10],
                                 m.cpu().numpy(), 0.1, torch.bfloat16)
    _near(a, want, bound)
    _near(b, want, bound)


def _far_cache(device, blocks, hkv, d, bs):
    """A cache whose last pages lie beyond 4 GiB; only those are written."""
    kc = torch.empty(blocks, bs, hkv, d + 4, dtype=torch.uint8, device=device)
    vc = torch.empty_like(kc)
    small_k, small_v, table = build_cache(device, [300], hkv, d, bs, 17)
    n = small_k.shape[0]
    kc[blocks - n:], vc[blocks - n:] = small_k, small_v
    return kc, vc, torch.where(table >= 0, table + blocks - n, table), small_k, small_v, table


def test_rows_beyond_4_gib(native_ops, device):
    """Every operator on pages at the end of a cache of over 4 GiB."""
    from hif8_rocm import kv_cache

    blocks, hkv, d, bs = 33000, 4, 256, 128
    assert blocks * bs * hkv * (d + 4) > 1 << 32
    kc, vc, far, sk, sv, near = _far_cache(device, blocks, hkv, d, bs)
    q = randn((12, 16, d), 18).to(device)
    m = torch.from_numpy(_tree_mask([12], 19)).to(device)
    n = sk.shape[0]

    def both(f):
        a, b = f(kc, vc, far.to(device)), f(sk, sv, near.to(device))
        assert torch.equal(a, b) and torch.equal(kc[blocks - n:], sk) and torch.equal(vc[blocks - n:], sv)

    both(lambda k, v, t: kv_cache.tree_attention(q, k, v, t, [288], m, scale=0.06, query_lens=[12]))
    w = [torch.zeros(1, hkv, 384, device=device) for _ in range(2)]
    both(lambda k, v, t: kv_cache.paged_decode_attention_weights(q[:1], k, v, t, [300], w[k is sk], scale=0.06))
    both(lambda k, v, t: (kv_cache.accumulate_key_weights(q, k, t, [300], w[k is sk], scale=0.06, query_lens=[12]),
                          w[k is sk])[1])
    path = torch.tensor([[1, 4, 5, 11]], dtype=I32, device=device)
    both(lambda k, v, t: kv_cache.accept_drafts(k, v, t, [288], path, [4]))
    both(lambda k, v, t: kv_cache.evict_kv_rows(k, v, t, [292], w[k is sk], 100))


# ------------------------------------------------------- key weights

def _weighted(device, lens, qlens, hq, hkv, d, bs, *, seed=0, dtype=torch.bfloat16, causal=True, mixed=False,
              bt_dtype=I32, dv=None, accumulate=True, q_mul=1.0, spoil=None):
    """accumulate_key_weights, and for one row per request the decode form too."""
    from hif8_rocm import kv_cache

    print(f"weights lens={lens[:4]} rows={qlens[:4]} hq={hq} hkv={hkv} d={d} bs={bs} {dtype} causal={causal}", flush=True)
    kc, vc, table = build_cache(device, lens, hkv, d, bs, seed, dv=dv, bt_dtype=bt_dtype, mixed=mixed)
    q = randn((sum(qlens), hq, d), seed + 1, q_mul, dtype)
    if spoil:
        spoil(kc, vc, table)
    scale = 1 / math.sqrt(d)
    width = max(lens) + 5
    start = torch.rand(len(lens), hkv, width, generator=torch.Generator().manual_seed(seed)).float()
    want, bound = weights_reference(q.double().numpy(), kc.cpu().numpy(), table.numpy(), lens, qlens, scale, causal)

    def check(w):
        w = w.double().cpu().numpy()
        for b, n in enumerate(lens):
            assert np.array_equal(w[b, :, n:], start[b, :, n:].double().numpy())   # entries of no row stay
            base = start[b, :, :n].double().numpy() if accumulate else 0.0
            full = base + want[b, :, :n]
            _near(torch.from_numpy(w[b, :, :n]), full, bound[b, :, :n] + 2.0 ** -24 * np.abs(full) + 2.0 ** -126)

    w = start.to(device)
    kv_cache.accumulate_key_weights(q.to(device), kc, table.to(device), lens, w, scale=scale, query_lens=qlens,
                                    causal=causal, accumulate=accumulate, validate=spoil is None)
    check(w)
    if all(n == 1 for n in qlens):
        w = start.to(device)
        out = kv_cache.paged_decode_attention_weights(q.to(device), kc, vc, table.to(device), lens, w, scale=scale,
                                                      accumulate=accumulate, validate=spoil is None)
        check(w)
        mask = np.ones((len(lens), 1), dtype=bool)
        o, e = tree_reference(q.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(),
                              [max(n - 1, 0) for n in lens], [1] * len(lens), mask, scale, dtype)
        for b, n in enumerate(lens):
            if n == 0:
                o[b] = 0.0
        _near(out, o, e)


@pytest.mark.parametrize("lens, hq, hkv, d, bs", [
    ([512], 16, 4, 256, 128), ([1, 2, 64, 65, 500], 16, 4, 256, 128), ([0, 77], 16, 4, 256, 128), ([1500, 3], 8, 8, 64, 32),
    ([300], 24, 8, 128, 16), ([129], 20, 2, 256, 144), ([333], 32, 1, 128, 64), ([70], 6, 2, 20, 12), ([2100], 80, 1, 64, 16),
])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode_weights_shapes(native_ops, device, lens, hq, hkv, d, bs, dtype):
    _weighted(device, lens, [1] * len(lens), hq, hkv, d, bs, dtype=dtype, seed=hq + bs)


@pytest.mark.parametrize("accumulate", [True, False])
def test_decode_weights_modes(native_ops, device, accumulate):
    _weighted(device, [400, 129], [1, 1], 16, 4, 256, 128, mixed=True, bt_dtype=torch.int64, accumulate=accumulate, seed=3)
    _weighted(device, [400, 129], [1, 1], 16, 4, 256, 128, q_mul=8.0, accumulate=accumulate, seed=4)
    _weighted(device, [200], [1], 4, 2, 128, 16, dv=64, accumulate=accumulate, seed=5)


@pytest.mark.parametrize("lens, qlens, hq, hkv, d, bs", [
    ([512], [32], 16, 4, 256, 128), ([200], [200], 16, 4, 256, 128), ([1, 64, 65, 300], [1, 64, 3, 129], 16, 4, 256, 128),
    ([90, 0, 33], [17, 0, 33], 8, 8, 64, 32), ([260], [40], 24, 8, 128, 16), ([140], [70], 20, 2, 256, 144),
    ([5], [9], 16, 4, 256, 128),               # more query rows than cached ones: some see nothing
    ([70, 50], [30, 0], 12, 4, 64, 16), ([100], [37], 6, 2, 20, 12), ([150], [150], 40, 1, 128, 64),
])
@pytest.mark.parametrize("causal", [True, False])
def test_key_weights_shapes(native_ops, device, lens, qlens, hq, hkv, d, bs, causal):
    dtype = torch.float16 if causal and d != 256 else torch.bfloat16
    _weighted(device, lens, qlens, hq, hkv, d, bs, causal=causal, dtype=dtype, seed=hq + d + bs)


@pytest.mark.parametrize("accumulate", [True, False])
def test_key_weights_modes(native_ops, device, accumulate):
    _weighted(device, [300, 129], [100, 20], 16, 4, 256, 128, mixed=True, bt_dtype=torch.int64, accumulate=accumulate, seed=6)
    _weighted(device, [300, 40], [100, 0], 16, 4, 256, 128, q_mul=8.0, accumulate=accumulate, seed=7)


def test_weights_of_blocks_outside_the_cache(native_ops, device):
    def spoil(kc, vc, table):
        table[0, 1], table[1, 0] = -1, 1 << 20

    _weighted(device, [400, 100], [9, 30], 16, 4, 256, 128, seed=8, spoil=spoil)
    _weighted(device, [400, 100], [1, 1], 16, 4, 256, 128, seed=9, spoil=spoil)


def test_weights_of_pages_with_rubbish_behind_the_last_row(native_ops, device):
    def spoil(kc, vc, table):
        blk = int(table[0, 0])
        kc[blk, 70:] = 0x80
        vc[blk, 70:] = 0x80

    _weighted(device, [70], [33], 16, 4, 256, 128, seed=10, spoil=spoil)
    _weighted(device, [70], [1], 16, 4, 256, 128, seed=11, spoil=spoil)


def test_weights_rows_behind_the_last_request_do_not_count(native_ops, device):
    """A padded batch: query rows past query_start_loc[-1] and a block table with more rows."""
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, [300, 90, 10], 4, 256, 128, 20)
    q = randn((40, 16, 256), 21).to(device)
    loc = torch.tensor([0, 20, 30], dtype=I32, device=device)
    lens = torch.tensor([300, 90], dtype=I32, device=device)
    w = torch.zeros(3, 4, 384, device=device)
    kv_cache.accumulate_key_weights(q, kc, table.to(device), lens, w, scale=0.06, query_start_loc=loc, max_query_len=20,
                                    max_seq_len=300, validate=False)
    v = torch.zeros(3, 4, 384, device=device)
    kv_cache.accumulate_key_weights(q[:30].clone(), kc, table[:2].to(device), [300, 90], v, scale=0.06, query_lens=[20, 10])
    assert torch.equal(w, v) and not w[2].any()


# ---------------------------------------------------------- eviction

def _evict(device, lens, keep, hkv, d, bs, *, seed=0, dv=None, positions=False, sinks=0, recent=None, bt_dtype=I32,
           make=None, keep_tensor=True, spoil=None):
    from hif8_rocm import kv_cache

    print(f"evict lens={lens[:4]} keep={keep if isinstance(keep, int) else keep[:4]} d={d} bs={bs}", flush=True)
    kc, vc, table = build_cache(device, lens, hkv, d, bs, seed, dv=dv, bt_dtype=bt_dtype)
    if spoil:
        spoil(table)
    g = torch.Generator().manual_seed(seed)
    width = max(max(lens), 1) + 3
    w = torch.exp(2 * torch.randn(len(lens), hkv, width, generator=g))
    if make:
        make(w)
    pos = None
    if positions:
        pos = torch.stack([torch.stack([torch.randperm(width, generator=g) for _ in range(hkv)]) for _ in lens]).to(I32)
    each = [keep] * len(lens) if isinstance(keep, int) else keep
    want = evict_reference(kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), lens, w.numpy(), each,
                           None if pos is None else pos.numpy(), sinks, recent)
    wd, pd = w.to(device), None if pos is None else pos.to(device)
    k = keep if isinstance(keep, int) or not keep_tensor else torch.tensor(keep, device=device)
    new = kv_cache.evict_kv_rows(kc, vc, table.to(device), lens, wd, k, positions=pd, sinks=sinks, protect_from=recent,
                                 validate=spoil is None)
    assert new.dtype == I32 and new.tolist() == want[4]
    assert np.array_equal(wd.cpu().numpy().view(np.uint32), want[2].view(np.uint32))
    assert np.array_equal(kc.cpu().numpy(), want[0]) and np.array_equal(vc.cpu().numpy(), want[1])
    assert pd is None or np.array_equal(pd.cpu().numpy(), want[3])


@pytest.mark.parametrize("lens, keep, hkv, d, bs", [
    ([600], 512, 4, 256, 128), ([1, 2, 3, 0], 1, 4, 256, 128), ([100, 90], 100, 2, 64, 16), ([300], 0, 2, 128, 16),
    ([1023, 1024, 1025, 2050], [700, 1, 1024, 1025], 2, 64, 144), ([50, 5000], [60, 33], 3, 20, 12), ([129], 128, 1, 64, 32),
])
@pytest.mark.parametrize("positions", [False, True])
def test_evict_shapes(native_ops, device, lens, keep, hkv, d, bs, positions):
    _evict(device, lens, keep, hkv, d, bs, positions=positions, seed=d + bs, dv=d + 4 if d == 20 else None)


def test_evict_protected_rows(native_ops, device):
    _evict(device, [500, 40], 100, 2, 64, 16, sinks=4, recent=[468, 8], seed=1)
    _evict(device, [500, 40], [100, 20], 2, 64, 16, sinks=4, recent=[468, 8], positions=True, bt_dtype=torch.int64, seed=2)
    _evict(device, [500], 10, 2, 64, 16, sinks=8, recent=[100], seed=3)          # more protected than kept
    _evict(device, [500], [30], 2, 64, 16, sinks=1 << 40, keep_tensor=False, seed=4)


def test_evict_ties_and_weights_that_are_no_numbers(native_ops, device):
    def ties(w):
        w[:] = (w > 1).float()
        w[:, 0] = 0.0

    def odd(w):
        w[..., 5::7] = math.nan
        w[..., 3::11] = math.inf
        w[..., 4::13] = -math.inf
        w[..., 2::5] = -0.0
        w[..., 1::5] = 0.0
        w[..., 6::17] = -1.5

    for make in (ties, odd):
        _evict(device, [700, 64], [300, 60], 2, 64, 16, make=make, sinks=2, seed=5)
        _evict(device, [700], 650, 2, 64, 16, make=make, seed=6)


def test_evict_long_rows(native_ops, device):
    _evict(device, [70001], 20000, 1, 64, 16, seed=7, sinks=4, recent=[69900])


def test_evict_rows_of_blocks_outside_the_cache(native_ops, device):
    def spoil(table):
        table[0, 1] = -1

    _evict(device, [200], 90, 2, 64, 16, seed=8, spoil=spoil)


def test_attention_over_the_kept_rows(native_ops, device):
    """Attention over the cut cache is attention over the kept rows: the weights of the others are gone."""
    from hif8_rocm import kv_cache

    lens, keep = [500, 300], 128
    kc, vc, table = build_cache(device, lens, 4, 256, 128, 9)
    q = randn((2, 16, 256), 10).to(device)
    w = torch.zeros(2, 4, 512, device=device)
    kv_cache.paged_decode_attention_weights(q, kc, vc, table.to(device), lens, w, scale=1 / 16)
    sharp = 8.0 / 16
    before = kv_cache.paged_decode_attention(q, kc, vc, table.to(device), lens, scale=sharp).double()
    dropped = torch.zeros(2, 4, 512, device=device)
    kv_cache.paged_decode_attention_weights(q, kc, vc, table.to(device), lens, dropped, scale=sharp)
    order = torch.sort(w, dim=-1, descending=True, stable=True)[1][..., keep:]
    lost = dropped.gather(2, order).sum(-1)                        # per KV head, over its four query heads
    new = kv_cache.evict_kv_rows(kc, vc, table.to(device), lens, w, keep)
    after = kv_cache.paged_decode_attention(q, kc, vc, table.to(device), new, scale=sharp, max_seq_len=keep).double()
    top = max(float(vc[..., :256].numel() and 6.0), 6.0)           # |V| of a normal sample is below six
    diff = (after - before).abs().amax(-1).view(2, 4, 4).amax(-1)
    assert (diff <= 2 * top * lost + 2 * 2.0 ** -8 * top).all()
    assert not w[:, :, keep:].any() and new.tolist() == [keep, keep]


# --------------------------------------------------------- acceptance

@pytest.mark.parametrize("layers, hkv, d, dv, bs, bt_dtype", [(1, 4, 256, 256, 128, I32), (3, 2, 64, 64, 16, torch.int64),
                                                             (70, 1, 20, 36, 12, I32)])
def test_accept_moves_the_path(native_ops, device, layers, hkv, d, dv, bs, bt_dtype):
    from hif8_rocm import kv_cache

    ctx = [37, 0, 200, 5]
    paths = [[0, 2, 5, 6, 9, 11, 12, 13, 20, 30], [], [1, 2, 3], [4]]
    lens = [c + 31 for c in ctx]
    pairs = [build_cache(device, lens, hkv, d, bs, s, dv=dv, bt_dtype=bt_dtype) for s in range(2)]
    table = pairs[0][2]
    keys = [pairs[i % 2][0].clone() for i in range(layers)]
    values = [pairs[i % 2][1].clone() for i in range(layers)]
    want = [c.cpu().numpy().copy() for c in keys + values]
    for c in want:
        old = c.copy()
        for b, path in enumerate(paths):
            for i, a in enumerate(path):
                to, frm = ctx[b] + i, ctx[b] + a
                c[int(table[b, to // bs]), to % bs] = old[int(table[b, frm // bs]), frm % bs]
    accepted = torch.full((4, 10), -1, dtype=torch.int64)
    for b, path in enumerate(paths):
        accepted[b, :len(path)] = torch.tensor(path, dtype=torch.int64)
    new = kv_cache.accept_drafts(keys, values, table.to(device), ctx, accepted.to(device), [len(x) for x in paths])
    assert new.tolist() == [c + len(x) for c, x in zip(ctx, paths)]
    for got, ref in zip(keys + values, want):
        assert np.array_equal(got.cpu().numpy(), ref)


def test_accept_skips_what_is_outside(native_ops, device):
    """Without validation: drafts past the table or in no block move nothing, and counts are clipped."""
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, [64], 2, 64, 16, 3)
    table[0, 2] = 1 << 20
    path = torch.tensor([[2, 30, 50000, 2000000000]], dtype=I32, device=device)
    before = kc.clone()
    new = kv_cache.accept_drafts(kc, vc, table.to(device), [4], path, torch.tensor([9]), validate=False)
    before[int(table[0, 0]), 4] = before[int(table[0, 0]), 6].clone()
    assert new.tolist() == [8] and torch.equal(kc, before)


# ------------------------------------------------- streams, graphs, together

def _step_buffers(device, seed=0):
    from hif8_rocm import kv_cache  # noqa: F401

    ctx, n, keep = [700, 333], 9, 300
    kc, vc, table = build_cache(device, [c + n for c in ctx], 4, 256, 128, seed)
    g = torch.Generator().manual_seed(seed)
    return {
        "kc": kc, "vc": vc, "table": table.to(device), "ctx": torch.tensor(ctx, dtype=I32, device=device),
        "q": randn((2 * n, 16, 256), seed + 1).to(device), "q1": randn((2, 16, 256), seed + 2).to(device),
        "loc": torch.tensor([0, n, 2 * n], dtype=I32, device=device),
        "mask": torch.from_numpy(_tree_mask([n, n], seed + 3)).to(device),
        "path": torch.tensor([[1, 3, 8], [0, 5, 0]], dtype=I32, device=device),
        "counts": torch.tensor([3, 2], dtype=I32, device=device),
        "w": torch.rand(2, 4, 768, generator=g).to(device),
        "pos": torch.arange(768, dtype=I32).expand(2, 4, 768).contiguous().to(device), "keep": keep,
    }


def _step(s):
    """One step of a server with drafts and a bounded cache, without a host synchronisation."""
    from hif8_rocm import kv_cache

    fast = dict(validate=False, max_seq_len=709)
    o1 = kv_cache.tree_attention(s["q"], s["kc"], s["vc"], s["table"], s["ctx"], s["mask"], scale=1 / 16,
                                 query_start_loc=s["loc"], max_query_len=9, **fast)
    lens = kv_cache.accept_drafts(s["kc"], s["vc"], s["table"], s["ctx"], s["path"], s["counts"], validate=False)
    o2 = kv_cache.paged_decode_attention_weights(s["q1"], s["kc"], s["vc"], s["table"], lens, s["w"], scale=1 / 16, **fast)
    kv_cache.accumulate_key_weights(s["q"], s["kc"], s["table"], lens, s["w"], scale=1 / 16, query_start_loc=s["loc"],
                                    max_query_len=9, **fast)
    new = kv_cache.evict_kv_rows(s["kc"], s["vc"], s["table"], lens, s["w"], s["keep"], positions=s["pos"], sinks=4, **fast)
    o3 = kv_cache.paged_decode_attention(s["q1"], s["kc"], s["vc"], s["table"], new, scale=1 / 16, **fast)
    return o1, lens, o2, new, o3


def test_a_step_on_another_stream(native_ops, device):
    want_state = _step_buffers(device)
    want = _step(want_state)
    torch.cuda.synchronize()
    state = _step_buffers(device)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = _step(state)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    for k in ("kc", "vc", "w", "pos"):
        assert torch.equal(state[k], want_state[k]), k


def test_two_graphs_of_a_step(native_ops, device):
    """Two captured steps on their own buffers, replayed in turn with eager steps between: every replay
    equals the eager step on the same inputs, bit for bit."""
    states = [_step_buffers(device, 30), _step_buffers(device, 40)]
    start = [{k: v.clone() for k, v in s.items() if torch.is_tensor(v)} for s in states]

    def reset(i):
        for k, v in start[i].items():
            states[i][k].copy_(v)

    want, ends = [], []
    for i in range(2):
        want.append([t.clone() for t in _step(states[i])])
        ends.append({k: states[i][k].clone() for k in ("kc", "vc", "w", "pos")})
        reset(i)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(_step(states[i]))
        graphs.append(g)
    for rep in range(3):
        for i in (0, 1):
            reset(i)
            other = _step_buffers(device, 50 + rep)
            _step(other)
            torch.cuda.synchronize()
            graphs[i].replay()
            torch.cuda.synchronize()
            print(f"replay {rep} of graph {i}", flush=True)
            for a, b in zip(outs[i], want[i]):
                assert torch.equal(a, b)
            for k, v in ends[i].items():
                assert torch.equal(states[i][k], v), k


def test_prompt_evict_draft_accept_decode(native_ops, device):
    """A request's life: its prompt's key weights, the cut, a tree of drafts written behind the cut cache,
    verified and accepted, and a decode step that keeps its weights - each step against the plain form."""
    from hif8_rocm import kv_cache

    hq, hkv, d, bs, prompt, keep = 16, 4, 256, 128, 260, 100
    kc, vc, table = build_cache(device, [prompt + 50], hkv, d, bs, 60)
    dt = table.to(device)
    q = randn((prompt, hq, d), 61)
    w = torch.zeros(1, hkv, 384, device=device)
    pos = torch.arange(384, dtype=I32).expand(1, hkv, 384).contiguous().to(device)
    kv_cache.accumulate_key_weights(q.to(device), kc, dt, [prompt], w, scale=1 / 16, query_lens=[prompt])
    want, bound = weights_reference(q.double().numpy(), kc.cpu().numpy(), table.numpy(), [prompt], [prompt], 1 / 16)
    _near(w[..., :prompt], want, bound + 2.0 ** -24 * np.abs(want))
    ref = evict_reference(kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), [prompt], w.cpu().numpy(), [keep],
                          pos.cpu().numpy(), 4, [prompt - 16])
    new = kv_cache.evict_kv_rows(kc, vc, dt, [prompt], w, keep, positions=pos, sinks=4, protect_from=[prompt - 16])
    assert np.array_equal(kc.cpu().numpy(), ref[0]) and np.array_equal(pos.cpu().numpy(), ref[3])
    n = 12
    key, value = randn((n, hkv, d), 62), randn((n, hkv, d), 63)
    ks, vs = (x.float().abs().amax(dim=(0, 2)).to(device) / 32768.0 for x in (key, value))
    slots = torch.tensor([int(table[0, t // bs]) * bs + t % bs for t in range(keep, keep + n)])
    kv_cache.write_kv_cache(key.to(device), value.to(device), kc, vc, slots.to(device), ks, vs)
    mask = ancestors([-1, -1, 0, 0, 1, 2, 2, 4, 5, 5, 8, 9])
    qt = randn((n, hq, d), 64)
    out = kv_cache.tree_attention(qt.to(device), kc, vc, dt, new, torch.from_numpy(mask).to(device), scale=1 / 16,
                                  query_lens=[n])
    o, e = tree_reference(qt.double().numpy(), kc.cpu().numpy(), vc.cpu().numpy(), table.numpy(), [keep], [n], mask, 1 / 16,
                          torch.bfloat16)
    _near(out, o, e)
    path = [0, 2, 5, 9, 11]
    before = kc.cpu().numpy()
    lens = kv_cache.accept_drafts(kc, vc, dt, new, torch.tensor([path], dtype=I32), [5])
    assert lens.tolist() == [keep + 5]
    for i, a in enumerate(path):
        to, frm = (int(x) for x in (slots[i], slots[a]))
        assert np.array_equal(kc.view(-1, hkv, d + 4)[to].cpu().numpy(), before.reshape(-1, hkv, d + 4)[frm])
    # The accepted path's last node saw the cache as a decode step now sees it.
    last = kv_cache.paged_decode_attention_weights(qt[11:12].to(device), kc, vc, dt, lens, w, scale=1 / 16)
    half = 2.0 ** -8 * out[11:12].double().abs() + 2 * torch.from_numpy(e[11:12]).to(device)
    assert ((last.double() - out[11:12].double()).abs() <= half).all()
    assert (w[:, :, keep:keep + 5] > 0).all() and not w[:, :, keep + 5:].any()


# ---------------------------------------- many requests, loose bounds, misuse

def _many(count, seed, most=40):
    g = np.random.default_rng(seed)
    return [int(x) for x in g.integers(0, most, count)]


@pytest.mark.parametrize("hq, hkv, d, drafts", [(16, 4, 256, 4), (8, 8, 64, 3), (16, 4, 256, 17), (6, 2, 20, 2)])
def test_tree_of_more_requests_than_workers(native_ops, device, hq, hkv, d, drafts):
    """150 short requests, some of them empty: workers go from one request into the next."""
    ctx = _many(150, 70)
    qlens = [min(n, drafts) for n in _many(150, 71, drafts + 2)]
    ctx[3], qlens[3], ctx[149] = 0, 0, 200
    _tree(device, ctx, qlens, hq, hkv, d, 16 if d != 20 else 5, seed=72, mask="any")


@pytest.mark.parametrize("hq, hkv, d", [(16, 4, 256), (8, 8, 64)])
def test_decode_weights_of_more_requests_than_workers(native_ops, device, hq, hkv, d):
    _weighted(device, _many(150, 73), [1] * 150, hq, hkv, d, 16, seed=74)


@pytest.mark.parametrize("hq, hkv, d", [(40, 1, 256), (140, 2, 256), (80, 1, 128)])
def test_decode_weights_of_many_heads_per_kv_head(native_ops, device, hq, hkv, d):
    _weighted(device, [300, 1, 0, 77], [1] * 4, hq, hkv, d, 32, seed=hq)


@pytest.mark.parametrize("causal", [True, False])
def test_key_weights_of_many_requests(native_ops, device, causal):
    lens = _many(90, 75)
    _weighted(device, lens, [min(n, 1 + i % 5) for i, n in enumerate(lens)], 8, 2, 64, 16, causal=causal, seed=76)


@pytest.mark.parametrize("causal", [True, False])
def test_key_weights_under_loose_bounds(native_ops, device, causal):
    """max_seq_len far above every length: the rows' partial sums are held for 64 query tokens at a time."""
    from hif8_rocm import kv_cache

    lens, qlens, hq, d, bs, most = [300, 90], [150, 37], 64, 64, 16, 1 << 19
    kc, _, table = build_cache(device, lens, 1, d, bs, 77)
    wide = torch.full((2, most // bs), -1, dtype=I32)
    wide[:, :table.shape[1]] = table
    q = randn((sum(qlens), hq, d), 78)
    w = torch.full((2, 1, most), 3.0, device=device)
    loc = torch.tensor([0, 150, 187], dtype=I32, device=device)
    for accumulate in (False, True):
        kv_cache.accumulate_key_weights(q.to(device), kc, wide.to(device), torch.tensor(lens, dtype=I32, device=device), w,
                                        scale=0.125, query_start_loc=loc, max_query_len=150, max_seq_len=most, causal=causal,
                                        accumulate=accumulate, validate=False)
    want, bound = weights_reference(q.double().numpy(), kc.cpu().numpy(), table.numpy(), lens, qlens, 0.125, causal)
    for b, n in enumerate(lens):
        _near(w[b, :, :n], 2 * want[b, :, :n], 2 * bound[b, :, :n] + 2.0 ** -23 * want[b, :, :n])
        assert (w[b, :, n:] == 3).all()


@pytest.mark.parametrize("lens, keep", [([16384, 100], 9000), ([20000], 19999), ([32768, 4097, 5], 4096)])
def test_evict_at_the_edges_of_what_registers_hold(native_ops, device, lens, keep):
    _evict(device, lens, keep, 1, 20, 64, positions=True, sinks=4, seed=79)


def test_evict_keeps_all_rows_for_counts_past_int32(native_ops, device):
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, [90, 40], 2, 64, 16, 80)
    w = torch.rand(2, 2, 90, device=device)
    was = [t.clone() for t in (kc, vc, w)]
    for keep in (torch.tensor([1 << 40, (1 << 32) + 5]), 1 << 40):
        new = kv_cache.evict_kv_rows(kc, vc, table.to(device), [90, 40], w, keep)
        assert new.tolist() == [90, 40] and all(torch.equal(a, b) for a, b in zip(was, (kc, vc, w)))


def test_requests_without_rows(native_ops, device):
    """Nothing but empty requests: outputs of rows that no request has are zeros, stored sums become zero."""
    from hif8_rocm import kv_cache

    kc, vc, table = build_cache(device, [50, 20], 2, 64, 16, 81)
    q = randn((3, 4, 64), 82).to(device)
    loc = torch.zeros(3, dtype=I32, device=device)
    mask = torch.ones(3, 4, dtype=torch.bool, device=device)
    out = kv_cache.tree_attention(q, kc, vc, table.to(device), [50, 20], mask, scale=0.1, query_start_loc=loc)
    assert not out.any()
    assert kv_cache.tree_attention(q[:0], kc, vc, table.to(device), [50, 20], mask[:0], scale=0.1,
                                   query_lens=[0, 0]).shape == (0, 4, 64)
    w = torch.ones(2, 2, 64, device=device)
    kv_cache.accumulate_key_weights(q[:0], kc, table.to(device), [50, 20], w, scale=0.1, query_lens=[0, 0])
    assert (w == 1).all()
    kv_cache.accumulate_key_weights(q[:0], kc, table.to(device), [50, 20], w, scale=0.1, query_lens=[0, 0], accumulate=False)
    assert not w[0, :, :50].any() and not w[1, :, :20].any() and (w[0, :, 50:] == 1).all() and (w[1, :, 20:] == 1).all()


def test_a_longest_request_told_too_short_stays_in_bounds(native_ops, device):
    """Without validation: a request longer than max_query_len leaves the other one's results as they are."""
    from hif8_rocm import kv_cache

    for hq, hkv, d, bs in ((16, 4, 256, 128), (6, 2, 20, 12)):
        lens, qlens = [330, 400], [5, 200]
        kc, vc, table = build_cache(device, lens, hkv, d, bs, 83)
        q = randn((205, hq, d), 84).to(device)
        mask = torch.from_numpy(_tree_mask([205], 85)[:, :6].copy()).to(device)
        loc = torch.tensor([0, 5, 205], dtype=I32, device=device)
        dt = table.to(device)
        args = dict(scale=0.1, query_start_loc=loc, max_query_len=5, max_seq_len=400, validate=False)
        ctx = torch.tensor([325, 200], dtype=I32, device=device)
        out = kv_cache.tree_attention(q, kc, vc, dt, ctx, mask, **args)
        alone = kv_cache.tree_attention(q[:5], kc, vc, dt[:1], [325], mask[:5], scale=0.1, query_lens=[5])
        # Each is rounded once (2^-8) and its weights once (2^-11 of sum p |V|, below two here).
        assert torch.allclose(out[:5].float(), alone.float(), rtol=2.0 ** -7, atol=2.0 ** -9)
        w = torch.zeros(2, hkv, 400, device=device)
        kv_cache.accumulate_key_weights(q, kc, dt, torch.tensor(lens, dtype=I32, device=device), w, **args)
        want, bound = weights_reference(q[:5].double().cpu().numpy(), kc.cpu().numpy(), table.numpy()[:1], lens[:1], [5], 0.1)
        _near(w[:1, :, :330], want, bound)
        assert not w[0, :, 330:].any()


def test_two_calls_at_once(native_ops, device):
    """The same operators on two streams at a time, each on its own outputs."""
    states = [_step_buffers(device, 90), _step_buffers(device, 91)]
    want = []
    for i in (0, 1):
        s = _step_buffers(device, 90 + i)
        want.append((_step(s), s))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for i in (0, 1):
        with torch.cuda.stream(streams[i]):
            got[i] = _step(states[i])
    torch.cuda.synchronize()
    for i in (0, 1):
        for a, b in zip(got[i], want[i][0]):
            assert torch.equal(a, b)
        for k in ("kc", "vc", "w", "pos"):
            assert torch.equal(states[i][k], want[i][1][k]), k


@pytest.mark.parametrize("ctx, qlens, hq, hkv, d, bs", [
    ([40, 30], [150, 30], 6, 2, 20, 12),       # any-shape kernel, a wavefront per output row
    ([25], [130], 8, 4, 512, 16),
    ([2000, 5], [40, 3], 16, 4, 64, 16),
    ([1500, 0, 300], [61, 2, 30], 24, 8, 128, 16),
    ([1100], [16], 16, 16, 128, 48),
])
def test_tree_of_many_rows(native_ops, device, ctx, qlens, hq, hkv, d, bs):
    for mask in ("tree", "any"):
        _tree(device, ctx, qlens, hq, hkv, d, bs, seed=95 + d, mask=mask, dtype=torch.float16, mixed=True)


def test_weights_of_many_heads_and_long_rows(native_ops, device):
    """Decode form where outputs take a wavefront each, and rows over several chunks of the join."""
    _weighted(device, [2100, 1025, 1024, 1] + [33] * 12, [1] * 16, 64, 4, 64, 16, seed=96, dtype=torch.float16)
