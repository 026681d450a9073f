"""The server's operators on the GPU on the paths that depend on sizes, layouts
and lists: strided outputs, batches that fill the card, far slots, values at the
ends of the range.  Oracles are in float64, tolerances are sums of the
documented roundings: half a step of bf16 is 2^-8 of the value, of f32 2^-24."""

import math

import numpy as np
import pytest

from _gpu import torch
from oracle import serving
from oracle.bf16 import round_bf16
from test_serving_ops_gpu import (DEV, _attention_bound, _check, _cu, _down, _ints, _kv4_case, _ops, _rand,
                                  _rotate_bound, _up)

pytestmark = pytest.mark.gpu


def _window(shape, strides):
    """A view with these strides of fresh memory, all 7."""
    need = 1 + sum((n - 1) * s for n, s in zip(shape, strides))
    return torch.full((need,), 7.0, dtype=torch.bfloat16, device=DEV).as_strided(shape, strides)


def test_outputs_whose_heads_share_memory_are_refused():
    """Overlapping windows of any strides; what interleaves without sharing
    is taken."""
    ops = _ops()
    from mi355x._lib import MKError
    rng = np.random.default_rng(2)
    T, H, D = 6, 2, 64
    q = _up(_rand(rng, (T, H, D)))
    cos, sin = ops.rope_tables(T, D, device=DEV)
    pos, cu, slots = _ints(np.arange(T)), _cu([2, 4]), _ints(np.arange(T), torch.int64)
    cache = ops.KV4Cache(1, H, 16, D, device=DEV)
    ops.kv4_append(cache, q, q, slots)
    table, lens = _ints(np.zeros((T, 1))), _ints(np.full(T, 6))

    def calls(out, out2):
        return [lambda: ops.qk_norm_rope(q, q, pos, cos, sin, q_out=out, k_out=out2),
                lambda: ops.kv4_read(cache, slots, k_out=out, v_out=out2),
                lambda: (ops.attention_packed(q, q, q, cu, 0.1, out=out), q),
                lambda: (ops.attention_kv4(q.unsqueeze(1), cache, table, lens, 0.1, out=out.unsqueeze(1)), q)]

    for strides in ((64, 64, 1), (128, 32, 1), (8, 1024, 1)):
        for call in calls(_window((T, H, D), strides), torch.empty_like(q))[:4]:
            with pytest.raises(MKError, match="share memory"):
                call()
    want = [[t.clone() for t in call()] for call in calls(torch.empty_like(q), torch.empty_like(q))]
    # Heads 6 * 128 + 64 apart lie between the tokens 128 apart.
    for call, (w, w2) in zip(calls(_window((T, H, D), (128, 832, 1)), _window((T, H, D), (832, 128, 1))), want):
        out, out2 = call()
        assert torch.equal(out.reshape(w.shape), w) and torch.equal(out2, w2)


@pytest.mark.parametrize("D", [64, 128])
def test_attention_kv4_largest_values(D):
    """Values as large as they may be, most of them with the weight 1: the sum
    of p and the largest |v| of each key's group, p <= 1, stays in the f32 range
    for 400 keys up to 2^119 (400 < 2^8.65; the format keeps at most 16 / 15
    of a value, 2^0.1).  The waves' runs have two or three tiles, and the running
    maximum may lag by 2^8 (the first tile's scores are 0, all others'
    7.9 .. 8 in units of log 2), so p reaches 1 within a tile."""
    ops = _ops()
    n, H, B, page = 400, 8, 96, 16
    rng = np.random.default_rng(2)
    q = np.zeros((1, H, D), np.float32)
    q[:, :, 0] = 1.0
    k = np.zeros((n, H, D), np.float32)
    k[64:, :, 0] = 5.53
    v = round_bf16(rng.choice([-1.0, 1.0], (n, H, D)).astype(np.float32) * 2.0 ** 119)
    k = round_bf16(k)
    kq = serving.kv4_values(*serving.kv4(k))
    assert (kq[64:, :, 0] * math.log2(math.e) < 8).all() and (kq[64:, :, 0] * math.log2(math.e) > 7.9).all()
    vq = serving.kv4_values(*serving.kv4(v)) / 2.0 ** 119
    assert n * np.abs(vq).max() * 2.0 ** 119 < 2.0 ** 128
    cache = ops.KV4Cache(n // page, H, page, D, device=DEV)
    ops.kv4_append(cache, _up(k), _up(v), _ints(np.arange(n), torch.int64))
    table = np.tile(np.arange(n // page), (B, 1))
    y = ops.attention_kv4(_up(np.tile(q, (B, 1, 1, 1))), cache, _ints(table), _ints(np.full(B, n)), 1.0)
    got = _down(y) / 2.0 ** 119
    ref, mag = serving.attention(q, kq, vq, 1.0, np.ones((1, n), bool))
    bound = _attention_bound(ref, mag, q, k, 1.0, n, kv4=True)
    _check(got, np.tile(ref, (B, 1, 1, 1)), np.tile(bound, (B, 1, 1, 1)), f"kv4 largest values {D}")


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("D,tail", [(64, 0), (128, 0), (64, 8200), (128, 8200)])
def test_attention_packed_scores_of_minus_infinity(D, tail, causal):
    """A query that sees keys, but only with the score -infinity, has no softmax:
    NaN, where one that sees no key gives zeros.  One that sees another key
    too has that one's value."""
    ops = _ops()
    rng = np.random.default_rng(4)
    nq, nk = 70, 50 + tail  # causal: the first 20 queries see nothing where tail = 0
    q = np.zeros((nq, 1, D), np.float32)
    q[:, 0, 0] = 1.0
    k = np.zeros((nk, 1, D), np.float32)
    k[:, 0, 0] = -np.inf
    v = _rand(rng, (nk, 1, D))

    def run():
        return _down(ops.attention_packed(_up(q), _up(k), _up(v), _cu([nq]), 1.0, cu_seqlens_k=_cu([nk]),
                                          causal=causal))[:, 0]

    last = np.arange(nq) + nk - nq if causal else np.full(nq, nk - 1)
    got = run()
    assert (got[last < 0] == 0).all() and np.isnan(got[last >= 0]).all()
    one = nk - 30
    k[one] = 0.0
    got = run()
    assert (got[last < 0] == 0).all() and np.isnan(got[(last >= 0) & (last < one)]).all()
    assert np.array_equal(got[last >= one], np.repeat(v[one].astype(np.float64), (last >= one).sum(), 0))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("n,B,H", [(30, 4, 2), (250, 4, 4), (1000, 4, 2), (200, 70, 8)])
def test_attention_kv4_scores_of_minus_infinity(n, B, H, D):
    """The same over the cache, where scores pass the f32 range: q . k is
    -10^30 times up to 10^30.  Keys in pages the cache does not have are not
    seen."""
    ops = _ops()
    page = 16
    rng = np.random.default_rng(5)
    q = np.zeros((B, 2, H, D), np.float32)
    q[..., 0] = 2.0 ** 100
    k = np.zeros((n, H, D), np.float32)
    k[:, :, 0] = -2.0 ** 100
    v = _rand(rng, (n, H, D))
    pages = -(-n // page)
    cache = ops.KV4Cache(pages, H, page, D, device=DEV)
    table = np.tile(np.arange(pages), (B, 1))
    table[1] = -1                     # no page: zeros
    table[2, 1:] = pages + 1          # the first page alone

    def run():
        ops.kv4_append(cache, _up(k), _up(v), _ints(np.arange(n), torch.int64))
        return _down(ops.attention_kv4(_up(q), cache, _ints(table), _ints([1] + [n] * (B - 1)), 1.0))

    got = run()
    assert (got[0, 0] == 0).all() and np.isnan(got[0, 1]).all()  # one key: the last query alone sees it
    assert (got[1] == 0).all() and np.isnan(got[2:]).all()
    k[n - 1] = 0.0
    got = run()
    vn = serving.kv4_values(*serving.kv4(v[n - 1]))
    assert (got[1] == 0).all() and np.isnan(got[2]).all() and np.isnan(got[3:, 0]).all()
    assert np.array_equal(got[3:, 1], np.tile(round_bf16(vn.astype(np.float32)).astype(np.float64), (max(B - 3, 0), 1, 1)))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hkv,D,layout", [(5, 2, 1, 64, "half"), (3, 20, 20, 80, "interleaved"),
                                               (1100, 32, 8, 128, "half")])
def test_qk_norm_rope_padding_of_new_outputs_is_zero(T, Hq, Hkv, D, layout, dt):
    """Rows with a negative position: zeros in an output made here, left as
    they were in one that is given, also where only one of the two is."""
    ops = _ops()
    rng = np.random.default_rng(T)
    q, k = _up(_rand(rng, (T, Hq, D)), dt), _up(_rand(rng, (T, Hkv, D)), dt)
    pos = rng.integers(0, 9, T)
    pos[[1, T - 1]] = [-1, -2 ** 31]
    kept = torch.from_numpy(pos >= 0).to(DEV)
    cos, sin = ops.rope_tables(9, 32, device=DEV)
    given = [torch.full_like(t, 7.0) for t in (q, k)]
    ops.qk_norm_rope(q, k, _ints(pos), cos, sin, layout=layout, q_out=given[0], k_out=given[1])
    for outs in ({}, {"q_out": 0}, {"k_out": 1}):
        dirty = [torch.full_like(t, float("nan")) for t in (q, k)]  # what an allocator may hand out again
        del dirty
        kw = {name: torch.full_like((q, k)[i], 7.0) for name, i in outs.items()}
        y = ops.qk_norm_rope(q, k, _ints(pos), cos, sin, layout=layout, **kw)
        for got, want, name in zip(y, given, ("q_out", "k_out")):
            assert torch.equal(got[kept], want[kept])
            assert (got[~kept] == (7.0 if name in kw else 0.0)).all()
    alone, none = ops.qk_norm_rope(q, None, _ints(pos), cos, sin, layout=layout)
    assert none is None and (alone[~kept] == 0).all() and torch.equal(alone[kept], given[0][kept])


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,norm", [
    (1024, 32, 8, 128, 128, True), (1025, 21, 3, 128, 64, True), (1100, 7, 14, 256, 64, True), (1030, 3, 2, 512, 512, True),
    (1024, 32, 9, 64, 40, False), (1500, 40, 1, 80, 80, True), (1024, 5, 0, 512, 8, True), (1300, 33, 32, 8, 8, True)])
def test_qk_norm_rope_of_many_tokens(T, Hq, Hkv, D, R, norm, layout, dt):
    """From 1024 tokens and more than 4 groups of heads on, a wave takes three
    groups, the last ones of a token in part: against float64, bit for bit the
    calls of fewer tokens, and in place with padding and unknown positions."""
    ops = _ops()
    rng = np.random.default_rng(T + Hq + D)
    lanes = max(8, 1 << (D // 8 - 1).bit_length())
    assert -(-(Hq + Hkv) * lanes // 64) > 4  # groups of heads that a wave holds at once
    qkv = _rand(rng, (T, Hq + 2 * Hkv, D), 1.5)
    gains = [round_bf16(rng.uniform(0.5, 1.5, D).astype(np.float32)) if norm else None for _ in range(2)]
    pos = rng.integers(0, 77, T)
    cos, sin = ops.rope_tables(77, R, device=DEV)
    x = _up(qkv, dt)
    g = [None if a is None else _up(a, dt) for a in gains]
    g[1] = g[1] if Hkv else None

    def run(lo, hi, at, **kw):
        k = x[lo:hi, Hq:Hq + Hkv] if Hkv else None
        return ops.qk_norm_rope(x[lo:hi, :Hq], k, _ints(at[lo:hi]), cos, sin, g_q=g[0], g_k=g[1], layout=layout, **kw)

    whole = run(0, T, pos)
    parts = [run(0, 700, pos), run(700, T, pos)]
    c, s = cos.double().cpu().numpy()[pos], sin.double().cpu().numpy()[pos]
    for i, (heads, gain) in enumerate(((slice(0, Hq), gains[0]), (slice(Hq, Hq + Hkv), gains[1]))):
        if i and not Hkv:
            assert whole[1] is None
            continue
        assert torch.equal(whole[i], torch.cat([p[i] for p in parts]))
        ref = serving.rotate(qkv[:, heads], gain, c, s, layout, 1e-6)
        _check(_down(whole[i]), ref, _rotate_bound(qkv[:, heads], ref, norm, D, dt), f"rotate {T}x{D} R{R} {layout}")
    # In place, with rows that are left and rows of no position.
    at = pos.copy()
    at[::17], at[5::23] = -1, 77
    kept, lost = torch.from_numpy(at < 0).to(DEV), torch.from_numpy(at == 77).to(DEV)
    known = ~(kept | lost)
    before = x.clone()
    run(0, T, at, q_out=x[:, :Hq], **({"k_out": x[:, Hq:Hq + Hkv]} if Hkv else {}))
    turned = x[:, :Hq + Hkv]
    want = torch.cat([w for w in whole if w is not None], 1)
    assert torch.equal(turned[known], want[known]) and torch.equal(turned[kept], before[kept][:, :Hq + Hkv])
    assert torch.isnan(turned[lost]).all() and torch.equal(x[:, Hq + Hkv:], before[:, Hq + Hkv:])


@pytest.mark.parametrize("lens,L,Hq,Hkv,D", [
    ([1, 63, 200], 1, 8, 2, 128), ([300, 700], 5, 16, 2, 64), ([400] * 96, 2, 16, 8, 64), ([130, 5] * 300, 1, 32, 8, 128)])
def test_attention_kv4_over_its_queries(lens, L, Hq, Hkv, D):
    """out = q, also as a view: the bits of a call with an output of its own,
    with items of one wave, of one workgroup and of several."""
    ops = _ops()
    q, _, _, cache, table = _kv4_case(ops, lens, L, Hq, Hkv, D, 64, 3)
    B, t, n = len(lens), _ints(table), _ints(lens)
    want = ops.attention_kv4(_up(q), cache, t, n, 0.1)
    x = torch.full((B, L, Hq + 3, D), 7.0, dtype=torch.bfloat16, device=DEV)
    for rest in (x, x.transpose(0, 1).contiguous().transpose(0, 1)):
        rest[:, :, :Hq] = _up(q)
        view = rest[:, :, :Hq]
        y = ops.attention_kv4(view, cache, t, n, 0.1, out=view)
        assert y is view and torch.equal(rest[:, :, :Hq], want) and (rest[:, :, Hq:] == 7.0).all()


def test_far_slots():
    """Slots from 2^30 on with pages of 1024, where the page is found by a
    division: the numbers of near slots, on both sides of that place."""
    ops = _ops()
    page, edge = 1024, 2 ** 30
    rng = np.random.default_rng(6)
    slots = np.concatenate([[0, 1023, 1024], edge + np.array([-1025, -1024, -1, 0, 1, 1023, 1024, 2047])])
    T = len(slots)
    k, v = _up(_rand(rng, (T, 1, 64))), _up(_rand(rng, (T, 1, 64)))
    near = ops.KV4Cache(1, 1, 16, 64, device=DEV)
    ops.kv4_append(near, k, v, _ints(np.arange(T), torch.int64))
    want = ops.kv4_read(near, _ints(np.arange(T), torch.int64), dtype=torch.float32)
    far = ops.KV4Cache(edge // page + 2, 1, page, 64, device=DEV)  # 75 GB
    at = _ints(slots, torch.int64)
    ops.kv4_append(far, k, v, at)
    for got, w in zip(ops.kv4_read(far, at, dtype=torch.float32), want):
        assert torch.equal(got, w)
    # In the places that the format documents.
    for a, b in zip((far.k_scale, far.v_scale, far.k_zero, far.v_zero),
                    (near.k_scale, near.v_scale, near.k_zero, near.v_zero)):
        assert torch.equal(a[at // page, 0, 0, at % page], b[0, 0, 0, :T])
    empty = torch.cat([at[3:] - 3, at[3:] + 5])
    empty = empty[~torch.isin(empty, at) & (empty < far.pages * page)]
    assert all((t == 0).all() for t in ops.kv4_read(far, empty))
    # Attention over the last page reads the same keys.
    q = _up(_rand(rng, (1, 1, 1, 64)))
    last = _ints([[edge // page + 1]])
    alone = ops.KV4Cache(1, 1, page, 64, device=DEV)
    for name in ("k", "k_scale", "k_zero", "v", "v_scale", "v_zero"):
        getattr(alone, name)[0] = getattr(far, name)[edge // page + 1]
    y = ops.attention_kv4(q, far, last, _ints([page]), 0.1)
    assert torch.equal(y, ops.attention_kv4(q, alone, _ints([[0]]), _ints([page]), 0.1)) and (y != 0).any()
    del far
    torch.cuda.empty_cache()


def test_expanded_inputs():
    """Inputs whose tokens or heads are one (strides of 0), as expand makes
    them: the bits of the copies."""
    ops = _ops()
    rng = np.random.default_rng(10)
    T, Hq, Hkv, D = 37, 4, 2, 64
    cos, sin = ops.rope_tables(T, D, device=DEV)
    pos, cu, slots = _ints(np.arange(T)), _cu([20, 17]), _ints(np.arange(T), torch.int64)
    table, lens = _ints(np.tile(np.arange(3), (2, 1))), _ints([37, 20])
    for one in ((1, Hq, D), (T, 1, D), (1, 1, D)):
        q = _up(_rand(rng, one)).expand(T, Hq, D)
        k = _up(_rand(rng, (one[0], min(one[1], Hkv), D))).expand(T, Hkv, D)
        got = []
        for a, b in ((q, k), (q.contiguous(), k.contiguous())):
            cache = ops.KV4Cache(3, Hkv, 16, D, device=DEV)
            ops.kv4_append(cache, b, b, slots)
            got.append([*ops.qk_norm_rope(a, b, pos, cos, sin), *ops.kv4_read(cache, slots),
                        ops.attention_packed(a, b, b, cu, 0.1),
                        ops.attention_kv4(a[:2].unsqueeze(1), cache, table, lens, 0.1)])
        assert all(torch.equal(x, y) for x, y in zip(*got))
