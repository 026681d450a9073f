"""The server's operators on the GPU on the paths that depend on sizes, layouts
and lists: strided outputs, batches that fill the card, far slots, values at the
ends of the range.  Oracles are in float64, tolerances are sums of the
documented roundings: half a step of bf16 is 2^-8 of the value, of f32 2^-24."""

import numpy as np
import pytest

from _gpu import torch
from test_serving_ops_gpu import DEV, _cu, _ints, _ops, _rand, _up

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
