"""Refusals of the operators around a decoding step (CPU): the Python functions and the C entries, before any
device memory is touched."""

import ctypes

import pytest
import torch

from hif8_rocm import kv_cache
from test_abi import LIB

I32 = torch.int32


def _caches(d=64, page=16):
    return (torch.zeros(4, page, 2, d + 4, dtype=torch.uint8),) * 2


@pytest.mark.parametrize("window, sinks, message", [
    (0, 0, "window must be"), (-1, 0, "window must be"), (2.0, 0, "window must be"), (True, 0, "window must be"),
    (4, -1, "sinks must be"), (4, 1.5, "sinks must be"), (None, 4, "sinks need a window")])
def test_windows_are_checked(window, sinks, message):
    kc, vc = _caches()
    table, q = torch.zeros(1, 2, dtype=I32), torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    opts = {"scale": 1.0, "window": window, "sinks": sinks}
    with pytest.raises(ValueError, match=message):
        kv_cache.paged_decode_attention(q, kc, vc, table, [1], **opts)
    with pytest.raises(ValueError, match=message):
        kv_cache.paged_attention(q, kc, vc, table, [1], query_lens=[1], **opts)
    pool = (table, torch.zeros(4, dtype=I32), torch.zeros(1, dtype=I32))
    with pytest.raises(ValueError, match=message):
        kv_cache.release_blocks(*pool, [1], block_size=16, window=window, sinks=sinks)


def test_a_window_is_causal():
    kc, vc = _caches()
    with pytest.raises(ValueError, match="causal"):
        kv_cache.paged_attention(torch.zeros(2, 4, 64, dtype=torch.bfloat16), kc, vc, torch.zeros(1, 2, dtype=I32), [5],
                                 scale=1.0, query_lens=[2], window=4, causal=False)


def test_windowed_pages_are_checked_where_they_are_seen():
    """A page outside the window may be gone; one inside raises."""
    kc, vc = _caches()
    table = torch.tensor([[0, -1, -1, 3, 9]], dtype=I32)
    q = torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(IndexError):
        kv_cache.paged_decode_attention(q, kc, vc, table, [64], scale=1.0, window=18, sinks=4)
    with pytest.raises(IndexError):
        kv_cache.paged_attention(q.expand(3, 4, 64), kc, vc, table, [64], scale=1.0, window=15, sinks=4, query_lens=[3])
    with pytest.raises(IndexError):
        kv_cache.paged_decode_attention(q, kc, vc, table, [64], scale=1.0, window=16, sinks=17)
    with pytest.raises(Exception, match="HIP device|could not be loaded|backend"):   # past the checks
        kv_cache.paged_decode_attention(q, kc, vc, table, [64], scale=1.0, window=16, sinks=16)


def _verify_args(tokens=3, vocab=10):
    return [torch.full((tokens, vocab), 0.1), torch.zeros(tokens, dtype=torch.int64), torch.full((tokens,), 0.5)]


def test_verify_drafts_is_checked():
    def refuses(error, message, index=None, value=None, **opts):
        args = _verify_args()
        if index is not None:
            args[index] = value
        with pytest.raises(error, match=message):
            kv_cache.verify_drafts(*args, **{"query_lens": [3], **opts})

    refuses(ValueError, "target_probs must have", 0, torch.zeros(3))
    refuses(ValueError, "target_probs must have", 0, torch.zeros(3, 0))
    refuses(TypeError, "must be float32", 0, torch.zeros(3, 10, dtype=torch.bfloat16))
    refuses(ValueError, "draft_tokens", 1, torch.zeros(2, dtype=torch.int64))
    refuses(ValueError, "draft_tokens", 1, torch.zeros(3))
    refuses(ValueError, "uniforms must hold", 2, torch.zeros(3, dtype=torch.float64))
    refuses(ValueError, r"in \[0, 1\)", 2, torch.tensor([0.0, 1.0, 0.5]))
    refuses(ValueError, r"in \[0, 1\)", 2, torch.tensor([0.0, float("nan"), 0.5]))
    refuses(ValueError, r"in \[0, 1\)", 2, torch.tensor([0.0, -0.1, 0.5]))
    refuses(ValueError, "chain", draft_probs=torch.zeros(3, 10), parents=torch.tensor([-1, 0, 0]))
    refuses(ValueError, "draft_probs must be float32", draft_probs=torch.zeros(3, 9))
    refuses(ValueError, "parents must hold", parents=torch.tensor([-1, 0]))
    refuses(ValueError, "below the row's own", parents=torch.tensor([-1, 1, 0]))
    refuses(ValueError, "below the row's own", parents=torch.tensor([-1, -1, 0]))
    refuses(ValueError, "query_lens must describe", query_lens=[2])
    refuses(ValueError, "exactly one", query_start_loc=torch.tensor([0, 3], dtype=I32))
    refuses(ValueError, "smaller than a request", max_query_len=2)
    big = _verify_args(1025, 2)
    with pytest.raises(ValueError, match="1024"):
        kv_cache.verify_drafts(*big, query_lens=[1025])


def test_page_pools_are_checked():
    def pool(**change):
        p = {"block_table": torch.full((2, 3), -1, dtype=I32), "free_blocks": torch.arange(6, dtype=I32),
             "free_count": torch.tensor([6], dtype=I32)}
        return tuple({**p, **change}.values())

    def refuses(error, message, args, lens=(1, 2), page=16, **opts):
        with pytest.raises(error, match=message):
            kv_cache.extend_block_tables(*args, lens, block_size=page, query_lens=[1, 1], **opts)
        with pytest.raises(error, match=message):
            kv_cache.release_blocks(*args, lens, block_size=page, **opts)

    refuses(ValueError, "block_table must have", pool(block_table=torch.zeros(2, dtype=I32)))
    refuses(TypeError, "block_table must be", pool(block_table=torch.zeros(2, 3)))
    refuses(ValueError, "contiguous", pool(block_table=torch.zeros(3, 2, dtype=I32).t()))
    refuses(TypeError, "free_blocks", pool(free_blocks=torch.arange(6)))
    refuses(TypeError, "free_count", pool(free_count=torch.tensor([6])))
    refuses(TypeError, "free_count", pool(free_count=torch.tensor([6, 1], dtype=I32)))
    refuses(ValueError, "within free_blocks", pool(free_count=torch.tensor([7], dtype=I32)))
    refuses(ValueError, "within free_blocks", pool(free_count=torch.tensor([-1], dtype=I32)))
    refuses(ValueError, "one length", pool(), lens=[1])
    refuses(ValueError, "non-negative", pool(), lens=[1, -2])
    refuses(ValueError, "non-negative", pool(), lens=torch.tensor([1, -2], dtype=I32))
    refuses(ValueError, "block_size", pool(), page=0)
    with pytest.raises(ValueError, match="exactly one"):
        kv_cache.extend_block_tables(*pool(), [1, 2], block_size=16)
    with pytest.raises(ValueError, match="a row for every request"):
        kv_cache.extend_block_tables(*pool(), [1, 2], block_size=16, query_lens=[1])
    with pytest.raises(ValueError, match="query_lens must be"):
        kv_cache.extend_block_tables(*pool(), [1, 2], block_size=16, query_lens=[1, -1])
    with pytest.raises(ValueError, match="total_query_tokens"):
        kv_cache.extend_block_tables(*pool(), [1, 2], block_size=16, query_lens=[1, 1], total_query_tokens=-1)


def _p(v=256):
    return ctypes.c_void_p(v)


P, I, L, Z = ctypes.c_void_p, ctypes.c_int, ctypes.c_int64, ctypes.c_size_t


@pytest.fixture(scope="module")
def lib():
    if not LIB.exists():
        pytest.fail(f"{LIB} is not built; run __graft_entry__.build()")
    lib = ctypes.CDLL(str(LIB))
    lib.hif8_last_error.restype = ctypes.c_char_p
    return lib


def test_window_entry_refuses(lib):
    f = lib.hif8_window_attention
    f.argtypes = [P, I, P, P, L, L, L, L, L, P, I, L, P, P, L, L, L, L, L, L, L, ctypes.c_float, P, P, Z, P]
    base = dict(q=_p(), qd=1, k=_p(), v=_p(), nb=8, bs=16, hkv=2, d=64, dv=64, bt=_p(), btd=0, mb=8, loc=_p(), lens=_p(),
                b=2, hq=4, t=6, mq=4, ml=100, w=32, s=4, sc=1.0, out=_p(), ws=_p(), n=1 << 30, st=None)

    def call(**change):
        return f(*{**base, **change}.values()), lib.hif8_last_error()

    for change, code, message in [
            (dict(w=0), 1, b"window must be positive"), (dict(w=-1), 1, b"window must be positive"),
            (dict(s=-1), 1, b"sinks"), (dict(mq=-1), 1, b"positive"), (dict(mq=0), 1, b"max_query_len"),
            (dict(loc=None), 1, b"query_start_loc"), (dict(hq=5), 1, b"divisible"), (dict(d=62), 1, b"divisible by four"),
            (dict(d=516), 2, b"512"), (dict(qd=3), 1, b"float16"), (dict(btd=2), 1, b"int32 or int64"),
            (dict(ml=129), 1, b"capacity"), (dict(q=None), 1, b"null"), (dict(ws=None), 1, b"workspace"),
            (dict(n=8), 1, b"workspace"), (dict(ws=_p(8)), 1, b"16-byte"), (dict(k=_p(2)), 1, b"4-byte")]:
        rc, text = call(**change)
        assert rc == code and message in text, (change, rc, text)
    assert call(b=0)[0] == 0 and call(t=0)[0] == 0
    size = lib.hif8_window_attention_workspace_size
    size.argtypes, size.restype = [L] * 11, Z
    assert size(2, 4, 2, 64, 64, 16, 6, 4, 100, 32, 4) > 0
    assert size(0, 4, 2, 64, 64, 16, 6, 4, 100, 32, 4) == size(2, 4, 2, 64, 64, 16, 6, 4, 100, 0, 4) == 0
    # A window bounds what a long request needs.
    assert size(2, 4, 2, 64, 64, 16, 6, 4, 1 << 20, 32, 4) == size(2, 4, 2, 64, 64, 16, 6, 4, 1 << 12, 32, 4)
    assert size(2, 4, 2, 64, 64, 16, 6, 4, 4096, 1 << 62, 1 << 62) > 0


def test_verify_entry_refuses(lib):
    f = lib.hif8_verify_drafts
    f.argtypes = [P, L, P, L, L, P, I, P, P, P, L, L, L, P, P, P, P, Z, P]
    base = dict(p=_p(), ps=100, q=_p(), qs=100, v=100, t=_p(), td=0, up=None, u=_p(), loc=_p(), b=2, n=6, w=4, a=_p(),
                c=_p(), x=_p(), ws=_p(), wb=1 << 20, st=None)

    def call(**change):
        return f(*{**base, **change}.values()), lib.hif8_last_error()

    for change, code, message in [
            (dict(v=0), 1, b"positive"), (dict(ps=99), 1, b"vocab apart"), (dict(qs=99), 1, b"vocab apart"),
            (dict(td=2), 1, b"int32 or int64"), (dict(up=_p()), 2, b"chain"), (dict(w=1025), 2, b"1024"),
            (dict(b=1 << 16), 1, b"too large"), (dict(p=None), 1, b"null"), (dict(a=None), 1, b"null"),
            (dict(ws=None), 1, b"workspace"), (dict(wb=8), 1, b"workspace"), (dict(ws=_p(4)), 1, b"8-byte")]:
        rc, text = call(**change)
        assert rc == code and message in text, (change, rc, text)
    assert call(b=0)[0] == 0


def test_page_entries_refuse(lib):
    f = lib.hif8_extend_block_tables
    f.argtypes = [P, I, L, P, L, P, P, P, L, L, L, P, P, P, P, P]
    base = dict(bt=_p(), btd=0, mb=8, fb=_p(), cap=10, fc=_p(), ctx=_p(), loc=_p(), b=2, n=6, bs=16, s=_p(), pos=_p(),
                lens=_p(), miss=_p(), st=None)
    for change, message in [(dict(mb=0), b"positive"), (dict(bs=0), b"positive"), (dict(cap=-1), b"positive"),
                            (dict(btd=3), b"int32 or int64"), (dict(mb=1 << 22), b"too large"),
                            (dict(bt=None), b"null"), (dict(fb=None), b"null"), (dict(s=None), b"null"),
                            (dict(loc=None), b"null")]:
        assert f(*{**base, **change}.values()) == 1 and message in lib.hif8_last_error(), change
    assert f(*{**base, "b": 0, "n": 0}.values()) == 0
    f = lib.hif8_release_blocks
    f.argtypes = [P, I, L, P, L, P, P, L, L, L, L, P, Z, P]
    base = dict(bt=_p(), btd=0, mb=8, fb=_p(), cap=10, fc=_p(), lens=_p(), b=2, bs=16, w=0, s=0, ws=_p(), wb=1 << 20,
                st=None)
    for change, message in [(dict(mb=0), b"positive"), (dict(w=-1), b"window"), (dict(s=-1), b"window"),
                            (dict(btd=3), b"int32 or int64"), (dict(b=1 << 20, mb=1 << 20), b"too large"),
                            (dict(lens=None), b"null"), (dict(ws=None), b"workspace"), (dict(wb=4), b"workspace")]:
        assert f(*{**base, **change}.values()) == 1 and message in lib.hif8_last_error(), change
    assert f(*{**base, "b": 0}.values()) == 0
