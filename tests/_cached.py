"""Batches for attention over the 4-bit cache whose results show every key:
inputs, float64 results and bounds, for the tests on the GPU and for the tests
on the CPU that plant mistakes.

Three kinds:
  uniform  q = 0, so every key weighs the same, and every key has the value 15
           in one of the dimensions of its head and 0 in the others (but for
           the first of each group of 64, which is always 15: the scale is 1).
           The result is 15 count / n, and a key lost or taken twice changes
           one dimension by a count-th, counts being below 128.
  codes    keys are codes of as many 15s as 0s (scale 1), each query is the sign
           pattern of one of them, which gets all the weight: the result is
           that key's value, whole numbers of 0 .. 15.
  random   keys and values at random, queries of whole numbers, so that the
           sums of the scores are exact in f32 and the weights nearly.
"""

import numpy as np
import torch

from oracle.bf16 import round_bf16

BF = 2.0 ** -8    # half a step of bf16, relative
F32 = 2.0 ** -24
U = 2.0 ** -23    # one addition of a sum in f32 that may be truncated
GROUP = 64
SCALE = 0.1


def pages_of(rng, lens, page, spare=2):
    """Block table (pages in no order), slot of every key, number of pages."""
    need = [-(-n // page) for n in lens]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), max(max(need), 1)), -1, dtype=np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    slots = np.concatenate([table[b, np.arange(n) // page].astype(np.int64) * page + np.arange(n) % page
                            for b, n in enumerate(lens)] + [np.zeros(0, np.int64)])
    return table, slots, sum(need) + spare


def seen_keys(n, L, blocked=None):
    """[L, n]: query i sees the keys before n - (L - 1 - i) that are not blocked."""
    seen = np.arange(n)[None, :] < n - (L - 1 - np.arange(L))[:, None]
    return seen if blocked is None else seen & ~blocked[None, :n]


def make(kind, lens, L, Hq, Hkv, D, seed, blocked=None):
    """q [B, L, Hq, D], k and v [sum(lens), Hkv, D] (f32, bf16 values)."""
    rng = np.random.default_rng(seed)
    B, N, group = len(lens), sum(lens), Hq // Hkv
    first = np.concatenate([[0], np.cumsum(lens)])
    if kind == "random":
        wide = np.exp(0.3 * rng.standard_normal((Hkv, D), dtype=np.float32))
        k = (rng.standard_normal((N, Hkv, D), dtype=np.float32) + 0.5) * wide
        q = rng.integers(-3, 4, (B, L, Hq, D)).astype(np.float32)
        return q, round_bf16(k), round_bf16(rng.standard_normal((N, Hkv, D), dtype=np.float32))
    if kind == "uniform":
        k = round_bf16(rng.standard_normal((N, Hkv, D), dtype=np.float32))
        v = np.zeros((N, Hkv, D), np.float32)
        free = np.flatnonzero(np.arange(D) % GROUP)
        turn = rng.integers(0, len(free), (B, Hkv))
        for b, n in enumerate(lens):
            for h in range(Hkv):
                order = (rng.permutation(n) + turn[b, h]) % len(free)
                v[first[b] + np.arange(n), h, free[order]] = 15.0
        v[:, :, ::GROUP] = 15.0
        return np.zeros((B, L, Hq, D), np.float32), k, v
    code = rng.random((N, Hkv, D // GROUP, GROUP), dtype=np.float32).argsort(-1) < GROUP // 2
    k = 15.0 * code.reshape(N, Hkv, D).astype(np.float32)
    v = rng.integers(0, 16, (N, Hkv, D)).astype(np.float32)
    v[:, :, 0::GROUP], v[:, :, 1::GROUP] = 0.0, 15.0
    q = np.zeros((B, L, Hq, D), np.float32)
    for b, n in enumerate(lens):
        seen = seen_keys(n, L, None if blocked is None else blocked[b])
        for i in range(L):
            at = np.flatnonzero(seen[i])
            if not len(at):
                continue
            # The first, the last, ends of tiles and of runs of 16, and any.
            ends = at[np.isin(at % 64, (0, 15, 16, 63))]
            pool = np.concatenate([at[:1], at[-1:], ends, rng.choice(at, max(1, len(ends)))])
            for h in range(Hq):
                j = pool[rng.integers(len(pool))] if (h + i) % 4 else at[-1 - (h + i) // 4 % 2 * (len(at) - 1)]
                q[b, i, h] = np.where(k[first[b] + j, h // group] > 0, 1.0, -1.0)
    return q, k, v


def attend(q, k, v, vs, weight, scale=SCALE):
    """float64 tensors: queries [L, Hq, D] over keys and values [n, Hkv, D] with
    the scales vs [n, Hkv, D/64] of v; weight [L, n] counts how often a query
    sees a key.  -> the result, the same sum with |v|, the sum of p and the
    scale, the largest |score|."""
    L, Hq, D = q.shape
    n, Hkv, group = k.shape[0], k.shape[1], Hq // k.shape[1]
    out = [torch.zeros((L, Hq, D), dtype=torch.float64, device=q.device) for _ in range(3)]
    big = torch.zeros((L, Hq, 1), dtype=torch.float64, device=q.device)
    if n == 0:
        return *out, big
    w = weight.repeat_interleave(group, 0)  # row i * group + g
    for h in range(Hkv):
        rows = q[:, h * group:(h + 1) * group].reshape(L * group, D)
        x = rows @ k[:, h].T.contiguous() * scale
        x = torch.where(w > 0, x, -torch.inf)
        top = x.amax(1, keepdim=True)
        p = torch.where(w > 0, w * torch.exp(x - torch.where(top == -torch.inf, 0.0, top)), 0.0)
        p = p / p.sum(1, keepdim=True).clamp(min=1e-300)
        vh = v[:, h].contiguous()
        steps = vs[:, h].repeat_interleave(GROUP, 1).contiguous()
        for o, y in zip(out, (vh, vh.abs(), steps)):
            o[:, h * group:(h + 1) * group] = (p @ y).reshape(L, group, D)
        size = torch.where(w > 0, x.abs(), 0.0).amax(1, keepdim=True)
        big[:, h * group:(h + 1) * group] = size.reshape(L, group, 1)
    return *out, big


def bound(kind, n, ref, mag, step, big):
    """What the kernel may be off by.
    uniform: sums of whole numbers and powers of two are exact; the weights'
      sum, its reciprocal, a product (2^-20 with the hardware's exp2) and half
      a step of bf16.
    codes: all but 10^-6 of the weight is on one key.
    random: half a step of bf16 of the result; of each weight times a scale
      half a step of bf16, 2^-20 for the hardware's exp2 and each of two joins,
      and the error of its score: a product, a sum of two groups, the scale's
      rounding and an argument of exp2, all rounded, twice (once in the sum of
      the weights); f32 sums over n keys, 2 n additions of them in the result;
      the zero points, taken off as 128 + z <= 143 steps by 64 additions a
      tile's half."""
    if kind == "uniform":
        return ref.abs() * (BF + 2.0 ** -19)
    if kind == "codes":
        return torch.full_like(ref, 1e-3)
    ds = 8 * F32 * (big + 16)
    return BF * ref.abs() + (1 + BF) * (mag * (BF * (1 + 2.0 ** -7) + 3 * 2.0 ** -20 + 2 * ds + 2 * (2 * n + 64) * U) +
                                        step * 143 * 64 * U) + 1e-30
