"""The inputs that attention over the 4-bit cache is tested with show what they
are meant to: a result with a planted mistake lies outside the tolerance."""

import numpy as np
import pytest
import torch

import _cached as C
from oracle import serving

CASES = [(65, 64, 1), (200, 64, 3), (1000, 128, 2), (2048, 64, 1), (5700, 64, 1), (2047, 128, 5)]


def _case(kind, n, D, L, seed=7):
    Hq, Hkv = 8, 2
    q, k, v = C.make(kind, [n], L, Hq, Hkv, D, seed)
    kq, vq = (serving.kv4_values(*serving.kv4(x)) for x in (k, v))
    vs = serving.kv4(v)[1]
    return [torch.from_numpy(np.asarray(x, np.float64)) for x in (q[0], kq, vq, vs)] + \
        [torch.from_numpy(C.seen_keys(n, L).astype(np.float64))]


def _result(kind, n, q, k, v, vs, weight):
    ref, mag, step, big = C.attend(q, k, v, vs, weight)
    return ref, C.bound(kind, n, ref, mag, step, big)


def _shown(got, ref, bound):
    """Outside by more than a right kernel's own rounding could hide."""
    return bool(((got - ref).abs() > 2 * bound).any())


@pytest.mark.parametrize("n,D,L", CASES)
def test_every_key_shows_among_equal_weights(n, D, L):
    """Lost or taken twice: single keys in all places, runs of 16, tiles, the
    ends of what a query sees."""
    q, k, v, vs, w = _case("uniform", n, D, L)
    ref, bound = _result("uniform", n, q, k, v, vs, w)
    at = sorted({0, 1, 15, 16, 63, 64, n // 2, n - 1 - L, n - L} & set(range(n - L + 1)))
    for j in at:
        for times in (0.0, 2.0):
            m = w.clone()
            m[:, j] *= times
            assert _shown(_result("uniform", n, q, k, v, vs, m)[0], ref, bound), (j, times)
    for lo, size in ((0, 16), (48, 16), (64 * (n // 128), 64)):
        m = w.clone()
        m[:, lo:lo + size] = 0
        assert _shown(_result("uniform", n, q, k, v, vs, m)[0], ref, bound), (lo, size)
    m = torch.ones_like(w)  # no causal limit
    assert L == 1 or _shown(_result("uniform", n, q, k, v, vs, m)[0], ref, bound)


@pytest.mark.parametrize("n,D,L", CASES)
def test_every_row_shows_its_key(n, D, L):
    """Each query's result is a value of its own; keys or values of another
    place, or lost, give another."""
    q, k, v, vs, w = _case("codes", n, D, L)
    ref, bound = _result("codes", n, q, k, v, vs, w)
    assert ((ref - ref.round()).abs() <= 1e-5).all()  # all the weight on one key
    key = (C.SCALE * torch.einsum("lhd,jhd->lhj", q, k.repeat_interleave(4, 1)) +
           torch.where(w > 0, 0.0, -torch.inf)[:, None]).argmax(-1)
    assert torch.equal(ref.round(), torch.stack([v.repeat_interleave(4, 1)[key[:, h], h] for h in range(8)], 1))
    near = torch.roll(torch.arange(n), 16)
    for kk, vv in ((k[near], v), (k, v[near]), (k.roll(1, 0), v), (k.flip(1), v)):
        assert _shown(_result("codes", n, q, kk, vv, vs, w)[0], ref, bound)
    for i, h in ((0, 0), (L - 1, 7)):
        m = w.clone()
        m[:, key[i, h]] = 0
        assert _shown(_result("codes", n, q, k, v, vs, m)[0], ref, bound)


@pytest.mark.parametrize("n,D,L", CASES)
def test_small_errors_of_the_numbers_show(n, D, L):
    """Scores 5 % or values 8 % too large, the next key's scores."""
    q, k, v, vs, w = _case("random", n, D, L)
    ref, bound = _result("random", n, q, k, v, vs, w)
    for kk, vv in ((1.05 * k, v), (k, 1.08 * v), (k.roll(1, 0), v)):
        assert _shown(_result("random", n, q, kk, vv, vs, w)[0], ref, bound)
