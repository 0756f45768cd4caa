"""Refusals of the rotary and paged-cache entry points that need no GPU (the
host checks its arguments before anything is launched), and host-side helpers."""
import pytest
import torch

from qtpytorch_amd import _lib as L

SOME = 1 << 12  # an address that is never read
POOL = dict(codes=SOME, scales=SOME, pages=4, page=16, heads=2, D=64)
BATCH = dict(table=SOME, lengths=SOME, offsets=SOME, B=1, width=2, tokens=3)


def _rotary(**kw):
    a = dict(x=SOME, x_type=0, tokens=3, heads=2, D=64, ts=128, hs=64, freqs=SOME, axis=0, pairs=32, inter=0, pos=SOME,
             pos_bytes=8, axes=1, back=0, y=SOME, stream=0)
    assert set(kw) <= set(a)
    return L.lib().mxk_rotary(*{**a, **kw}.values())


def _append(**kw):
    a = dict(k=SOME, kt=128, kh=64, v=SOME, vt=128, vh=64, q=0, qt=0, qh=0, q_heads=0, x_type=0, **POOL, **BATCH, freqs=0,
             axis=0, pairs=0, inter=0, pos=0, pos_bytes=0, axes=0, q_out=0, stream=0)
    assert set(kw) <= set(a)
    return L.lib().mxk_kv_pages_append(*{**a, **kw}.values())


def _read(**kw):
    a = dict(**POOL, **BATCH, y_type=0, k=SOME, v=SOME, stream=0)
    assert set(kw) <= set(a)
    return L.lib().mxk_kv_pages_read(*{**a, **kw}.values())


def _keep(**kw):
    a = dict(**POOL, **BATCH, path=SOME, steps=2, stream=0)
    assert set(kw) <= set(a)
    return L.lib().mxk_kv_pages_keep(*{**a, **kw}.values())


def _attend(**kw):
    a = dict(q=SOME, q_type=0, qt=128, qh=64, q_heads=4, **POOL, **BATCH, mask=0, words=0, scale=0.125, out=SOME, ws=SOME,
             ws_bytes=1 << 30, stream=0)
    assert set(kw) <= set(a)
    return L.lib().mxk_kv_pages_attend(*{**a, **kw}.values())


@pytest.mark.parametrize("call,kw,text", [
    (_rotary, dict(tokens=-1), b"bad sizes"), (_rotary, dict(tokens=1 << 31), b"bad sizes"), (_rotary, dict(D=4097), b"bad sizes"),
    (_rotary, dict(pairs=33), b"more rotated"), (_rotary, dict(pairs=-1), b"more rotated"), (_rotary, dict(x=0), b"null"),
    (_rotary, dict(y=0), b"null"), (_rotary, dict(freqs=0), b"null"), (_rotary, dict(pos=0), b"null"),
    (_rotary, dict(pos_bytes=2), b"4 or 8"), (_rotary, dict(axes=0), b"axes"), (_rotary, dict(x_type=5), b"x_type"),
    (_append, dict(k=0), b"null"), (_append, dict(v=0), b"null"), (_append, dict(q_heads=2), b"null"),
    (_append, dict(x_type=3), b"x_type"), (_append, dict(pairs=33, freqs=SOME), b"more rotated"),
    (_append, dict(pairs=2), b"null"), (_append, dict(pairs=2, freqs=SOME, pos=SOME, pos_bytes=4), b"axes"),
    (_read, dict(k=0), b"null"), (_read, dict(v=0), b"null"), (_read, dict(y_type=9), b"y_type"),
    (_keep, dict(path=0), b"null"), (_keep, dict(steps=65), b"64"), (_keep, dict(steps=-1), b"64"),
    (_attend, dict(q=0), b"null"), (_attend, dict(out=0), b"null"), (_attend, dict(q_heads=3), b"multiple"),
    (_attend, dict(q_heads=0), b"multiple"), (_attend, dict(scale=0.0), b"positive"),
    (_attend, dict(scale=float("nan")), b"positive"), (_attend, dict(scale=float("inf")), b"positive"),
    (_attend, dict(q_type=7), b"q_type"), (_attend, dict(mask=SOME, words=0), b"words"), (_attend, dict(pages=0), b"without pages"),
    (_attend, dict(tokens=(1 << 30) + 1), b"bad sizes"), (_append, dict(tokens=(1 << 30) + 1), b"bad sizes"),
    (_rotary, dict(tokens=(1 << 30) + 1), b"bad sizes"), (_attend, dict(tokens=30000, width=1 << 30), b"2^31 blocks"),
    (_attend, dict(scale=3e38), b"positive"),
    (_attend, dict(width=400, ws=0), b"workspace"), (_attend, dict(width=400, ws_bytes=100), b"workspace"),
    (_attend, dict(width=400, ws=SOME + 4), b"workspace"),
])
def test_refused(call, kw, text):
    assert call(**kw) == L.MXK_EINVAL
    assert text in L.lib().mxk_last_error()


@pytest.mark.parametrize("call", [_append, _read, _keep, _attend])
@pytest.mark.parametrize("kw,rc", [
    (dict(page=8), L.MXK_EINVAL), (dict(page=24), L.MXK_EINVAL), (dict(page=0), L.MXK_EINVAL), (dict(heads=0), L.MXK_EINVAL),
    (dict(pages=-1), L.MXK_EINVAL), (dict(pages=1 << 31), L.MXK_EINVAL), (dict(D=96), L.MXK_EUNSUPPORTED),
    (dict(codes=0), L.MXK_EINVAL), (dict(scales=0), L.MXK_EINVAL), (dict(codes=SOME + 8), L.MXK_EINVAL),
    (dict(B=-1), L.MXK_EINVAL), (dict(width=1 << 31), L.MXK_EINVAL), (dict(tokens=-5), L.MXK_EINVAL),
    (dict(table=0), L.MXK_EINVAL), (dict(lengths=0), L.MXK_EINVAL), (dict(offsets=0), L.MXK_EINVAL)])
def test_bad_pools_and_batches_are_refused(call, kw, rc):
    assert call(**kw) == rc
    assert L.lib().mxk_last_error()


@pytest.mark.parametrize("call,kw", [(_rotary, dict(tokens=0)), (_rotary, dict(heads=0, x=0, y=0)), (_append, dict(tokens=0, k=0)),
                                     (_read, dict(tokens=0, k=0)), (_keep, dict(steps=0, path=0)), (_keep, dict(B=0)),
                                     (_attend, dict(tokens=0, q=0))])
def test_nothing_to_do(call, kw):
    assert call(**kw) == L.MXK_OK


def test_tree_mask():
    from qtpytorch_amd import kv_tree_mask
    mask, depth = kv_tree_mask([-1, 0, 0, 1, 2, 4], device="cpu")
    assert mask.tolist() == [[0b1], [0b11], [0b101], [0b1011], [0b10101], [0b110101]]
    assert depth.tolist() == [0, 1, 1, 2, 2, 3] and depth.dtype == torch.int32
    mask, depth = kv_tree_mask(list(range(-1, 129)), device="cpu")  # a chain over word borders
    assert mask.shape == (130, 3) and mask[63].tolist() == [-1, 0, 0] and mask[129].tolist() == [-1, -1, 3]
    assert mask[127].tolist() == [-1, -1, 0] and depth[129] == 129
    assert kv_tree_mask([], device="cpu")[0].shape == (0, 1)
    with pytest.raises(ValueError, match="before its parent"):
        kv_tree_mask([-1, 1], device="cpu")
