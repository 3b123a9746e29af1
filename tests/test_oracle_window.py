"""The 64-bit window reference (oracle/window.py) against its definition and torch's own attention."""

import itertools

import pytest
import torch

from oracle import window as W


@pytest.mark.parametrize("causal", [True, False])
def test_visible_is_the_definition(causal):
    for kv, qo, left, sinks in itertools.product((0, 1, 7, 20), (0, 1, 3, 20), (-1, 0, 1, 5, 40), (0, 2, 30)):
        if qo > kv:
            continue
        got = W.visible(kv, qo, left, sinks, causal)
        assert got.shape == (qo, kv)
        for j, t in itertools.product(range(qo), range(kv)):
            i = kv - qo + j
            assert bool(got[j, t]) == ((not causal or t <= i) and (left < 0 or t >= i - left or t < sinks))


def test_attend_agrees_with_torch():
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(n, h, 16, generator=g, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    for left, sinks in ((-1, 0), (3, 1), (100, 0)):
        seen = W.visible(9, 5, left, sinks, True)
        out, bound = W.attend(q, k, v, seen, 2.0 ** -8)
        want = torch.nn.functional.scaled_dot_product_attention(
            q.transpose(0, 1), k.repeat_interleave(2, 1).transpose(0, 1), v.repeat_interleave(2, 1).transpose(0, 1),
            attn_mask=seen).transpose(0, 1)
        assert (out - want).abs().max() < 1e-12
        assert (bound > 0).all() and bound.shape == out.shape


def test_rows_without_keys_are_zero():
    q, k = torch.ones(2, 1, 8), torch.ones(3, 1, 8)
    out, _ = W.attend(q, k, k, torch.tensor([[False] * 3, [True] * 3]), 2.0 ** -8)
    assert (out[0] == 0).all() and (out[1] == 1).all()
