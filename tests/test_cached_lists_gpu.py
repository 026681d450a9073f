"""Attention over the 4-bit cache with results that show every key (inputs and
bounds: _cached.py): where the list of 64-key tiles is longer than the waves
that share it (2048), so that a wave takes runs of several tiles (parts of one
item, whole items within a run, runs over the ends of items and sequences, page
ids read anew every 16 tiles), and where a wave takes one tile of an item."""

import numpy as np
import pytest

import _cached as C
from _gpu import torch
from test_serving_ops_gpu import DEV, _check, _down, _ints, _ops, _up

pytestmark = pytest.mark.gpu

RAGGED = [1, 2048, 333, 0, 1500, 2000, 17, 1024, 777, 1999, 65, 1300, 512, 900, 1750, 2047]


def _mixed(B, top, seed):
    return [int(n) for n in np.random.default_rng(seed).integers(0, top, B)]


def _tiles(lens, L, Hq, Hkv):
    return sum(max(1, -(-n // 64)) for n in lens) * Hkv * (-(-L * (Hq // Hkv) // 16))


# name: lengths, new tokens, query heads, key heads, dimensions, page, share of
# table entries that name no page of the cache
BATCHES = {
    "ragged own heads": (RAGGED, 1, 16, 16, 128, 16, 0.0),
    "ragged, small heads": (RAGGED, 1, 32, 16, 64, 64, 0.0),
    "more than 64 sequences": (_mixed(70, 600, 1), 1, 16, 16, 64, 48, 0.0),
    "three blocks of rows": (_mixed(12, 1500, 2), 5, 64, 8, 128, 64, 0.0),
    "two blocks, bad pages": (_mixed(20, 1400, 3), 4, 64, 8, 64, 16, 0.05),
    "bad pages, 128 dimensions": (_mixed(40, 700, 4), 2, 32, 8, 128, 32, 0.1),
    "short items in longer runs": (_mixed(200, 130, 5), 1, 32, 32, 64, 16, 0.0),
    "2047 tiles": ([64 * 89] * 23, 1, 4, 1, 64, 1024, 0.0),
    "2048 tiles": ([64 * 89 - 63] * 23 + [1], 1, 4, 1, 64, 128, 0.0),
    "2049 tiles": ([64 * 89 - 1] * 23 + [65], 1, 4, 1, 64, 128, 0.0),
    "4097 tiles": ([64 * 100] * 40 + [64 * 97 - 5], 1, 1, 1, 64, 64, 0.0),
    "one long, 128 dimensions": ([7000, 3, 7000, 64, 6999], 1, 32, 8, 128, 64, 0.0),
}

SHORT = {
    "1 of 4097": ([4097], 1, 4, 1, 128, 64, 0.0),
    "1 of 8000": ([8000], 1, 16, 1, 128, 64, 0.0),
    "3001 and 2002": ([3001, 2002], 1, 2, 2, 64, 64, 0.0),
    "1000, 10, 0": ([1000, 10, 0], 1, 20, 1, 128, 16, 0.0),
    "1 .. 4 tiles": ([1, 64, 65, 128, 129, 192, 193, 256], 1, 8, 4, 64, 48, 0.0),
    "blocks of few tiles": ([300, 40, 7], 6, 16, 2, 128, 32, 0.0),
    "more new tokens than keys": ([3, 0, 130], 9, 4, 2, 64, 16, 0.0),
    "bad pages": ([900, 450, 30], 3, 8, 2, 64, 32, 0.2),
}


def test_the_batches_are_what_they_say():
    for name, (lens, L, Hq, Hkv, *_) in BATCHES.items():
        tiles = _tiles(lens, L, Hq, Hkv)
        assert tiles == int(name.split()[0]) if name.endswith(" tiles") else tiles >= 2048, (name, tiles)
    assert all(_tiles(lens, *rest[:3]) < 2048 for lens, *rest in SHORT.values())


@pytest.mark.parametrize("kind", ["uniform", "codes", "random"])
@pytest.mark.parametrize("name", [*BATCHES, *SHORT])
def test_every_key_and_row(name, kind):
    ops = _ops()
    lens, L, Hq, Hkv, D, page, bad = {**BATCHES, **SHORT}[name]
    rng = np.random.default_rng(len(name))
    table, slots, pages = C.pages_of(rng, lens, page)
    lost = rng.random(table.shape) < bad
    blocked = [np.repeat(lost[b], page) for b in range(len(lens))] if bad else None
    q, k, v = C.make(kind, lens, L, Hq, Hkv, D, 11, blocked)
    cache = ops.KV4Cache(pages, Hkv, page, D, device=DEV)
    for t in (cache.k_scale, cache.v_scale):  # the worst that places without a key can hold
        t.fill_(float("nan"))
    at = _ints(slots, torch.int64)
    ops.kv4_append(cache, _up(k), _up(v), at)
    table[lost] = rng.choice([-1, pages, 2 ** 31 - 1, -2 ** 31], int(lost.sum()))
    args = (_up(q), cache, _ints(table), _ints(lens), C.SCALE)
    y = ops.attention_kv4(*args)
    # The cache's numbers are exact in f32 and tested apart.
    kc, vc = (t.double() for t in ops.kv4_read(cache, at, dtype=torch.float32))
    vs = cache.v_scale[at // page, :, :, at % page].double()
    qd, ref, bound, first = _up(q).double(), [], [], 0
    for b, n in enumerate(lens):
        weight = torch.from_numpy(C.seen_keys(n, L, blocked[b] if bad else None).astype(np.float64)).to(DEV)
        r, mag, step, big = C.attend(qd[b], kc[first:first + n], vc[first:first + n], vs[first:first + n], weight)
        ref.append(r)
        bound.append(C.bound(kind, n, r, mag, step, big))
        first += n
    _check(_down(y), _down(torch.stack(ref)), _down(torch.stack(bound)), f"{name}, {kind}")
    assert torch.equal(ops.attention_kv4(*args), y)
