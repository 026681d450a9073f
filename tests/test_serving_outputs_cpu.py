"""Outputs of the server's operators whose heads share memory are refused by
the C entries (nothing is launched here)."""

import ctypes

import numpy as np
import pytest

from mi355x import _lib
from test_serving_ops_cpu import FAKE, _cache, _kv4_attention, _packed, _rotate, i64s

SHARE = b"share memory"


def _last(rc):
    assert rc == _lib.MK_EINVAL
    return _lib.lib().mk_last_error()


# Windows of four tokens, each of whose heads begins in the one before; heads
# closer than their dimensions; a token of every stride but 0.
@pytest.mark.parametrize("tok,head", [(64, 64), (64, 8), (128, 32), (32, 4096), (8, 1024), (72, 64)])
def test_overlapping_outputs_refused(tok, head):
    L, c = _lib.lib(), _cache()
    good = (1024, 64)
    assert SHARE in _last(_rotate(strides=i64s(*good, *good, tok, head, *good)))
    assert SHARE in _last(_rotate(strides=i64s(*good * 3, tok, head), Hkv=2))
    for st in (i64s(tok, head, *good), i64s(*good, tok, head)):
        assert SHARE in _last(L.mk_kv4_read(ctypes.byref(c), _lib.MK_DT_F32, FAKE, FAKE, st, FAKE, 4, None))
    assert SHARE in _last(_packed(strides=i64s(*good * 3, tok, head), Tq=4, Hq=2, Hkv=2))
    assert SHARE in _last(_kv4_attention(strides=i64s(*[1024, 1024, 64], tok, 0, head), B=4, Hq=2))
    assert SHARE in _last(_kv4_attention(strides=i64s(*[1024, 1024, 64], 8192, tok, head), B=2, L=4, Hq=2))


def test_outputs_on_one_place_refused():
    assert SHARE in _last(_rotate(strides=i64s(1024, 64, 1024, 64, 0, 64, 1024, 64)))
    assert SHARE in _last(_packed(strides=i64s(*[256, 64] * 3, 256, 0)))
    assert SHARE in _last(_kv4_attention(strides=i64s(256, 256, 64, 0, 256, 64)))


def _apart(n, stride, run):
    """By listing every element."""
    at = np.zeros(1, np.int64)
    for m, s in zip(n, stride):
        at = (at[:, None] + np.arange(m) * s).ravel()
    at = (at[:, None] + np.arange(run)).ravel()
    return len(np.unique(at)) == len(at)


def test_exactly_the_overlapping_layouts_are_refused():
    """Any strides, interleaved ones among them: refused if and only if two
    elements are one.  A scale that is refused later keeps the rest from a
    launch."""
    rng = np.random.default_rng(3)
    seen = [0, 0]
    for _ in range(3000):
        n = [int(v) for v in rng.integers(1, 6, 3)]
        st = [8 * int(v) for v in rng.integers(0, 60, 3)]
        want = _apart(n[1:], st[1:], 64)
        last = _last(_packed(Tq=n[1], Tk=n[1], Hq=n[2], Hkv=n[2], scale=3e38, strides=i64s(*[1024, 64] * 3, *st[1:])))
        assert (SHARE not in last) == want and (b"scale" in last) == want, (n, st)
        want = _apart(n, st, 64)
        last = _last(_kv4_attention(cache=_cache(heads=n[2]), B=n[0], L=n[1], Hq=n[2], scale=3e38,
                                    strides=i64s(4096, 1024, 64, *st)))
        assert (SHARE not in last) == want and (b"scale" in last) == want, (n, st)
        seen[want] += 1
    assert min(seen) > 300
    # Interleaved but apart: a token's second head lies behind the next one's first.
    assert b"scale" in _last(_packed(Tq=3, Tk=3, Hq=2, Hkv=2, scale=3e38, strides=i64s(*[1024, 64] * 3, 128, 192)))
    # Products of strides and sizes beyond 64 bits.
    far = i64s(*[1 << 40, 1 << 39] * 4)
    assert b"scale" in _last(_packed(Tq=2, Tk=2, Hq=2, Hkv=2, scale=3e38, strides=far))
    assert SHARE in _last(_packed(Tq=1 << 27, Tk=1 << 27, Hq=4, Hkv=4, scale=3e38, strides=far))


def test_kv4_workspace_query_refuses_what_the_call_refuses():
    """-1 for every size that the attention itself refuses, also where a
    product of sizes would pass 64 bits."""
    need = _lib.lib().mk_attention_kv4_workspace_bytes
    assert need(1, 1, 65535, 65535, 64, 4, 1024) > 0
    for bad in ((2, 1, 4, 2, 64, 1 << 24, 1 << 40), (2, 1, 4, 2, 64, 4, 1 << 62), (2, 1, 4, 2, 64, 4, 24),
                (2, 1, 4, 2, 64, 4, 8), (2, 1, 4, 2, 64, 4, 2048), (1, 1, 65536, 65536, 64, 4, 16)):
        assert need(*bad) == -1, bad
    for page, heads in ((24, 2), (2048, 2), (16, 65536)):
        assert _kv4_attention(cache=_cache(page=page, heads=heads), Hq=heads, B=1) != _lib.MK_OK
