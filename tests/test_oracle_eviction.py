"""The oracles of normed rotation, attention weights and eviction against other ways to the same values."""

import math

import numpy as np
import pytest
import torch

from oracle import eviction as E
from oracle import qk_norm as N
from oracle import rope as R


@pytest.mark.parametrize("interleave", [False, True])
@pytest.mark.parametrize("llama31", [None, dict(low_freq_factor=1.0, high_freq_factor=4.0, old_context_len=8192)])
def test_norm_rope_is_a_norm_and_a_rotation(interleave, llama31):
    """At near positions the fp32 rotation oracle agrees; at far ones the rotation is the complex product."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(9, 3, 64, generator=g)
    w = 1 + 0.3 * torch.randn(64, generator=g)
    pos = torch.arange(9)
    kw = dict(rope_scale=8.0 if llama31 else 1.0, rope_theta=5e5)
    out, bound = N.norm_rope(x, w, pos, 1e-5, 32, interleave, llama31=llama31, **kw)
    y = torch.nn.functional.rms_norm(x.double(), (64,), w.double(), 1e-5)
    ref = R.rope(y.float(), pos.numpy(), rotary_dim=32, interleave=interleave, llama31=llama31, **kw)
    assert (out - ref.double()).abs().max() < 2e-5 and (bound >= 0).all()
    far = torch.tensor([10 ** 6 + 7])
    out, _ = N.norm_rope(x[:1], w, far, 1e-5, 32, interleave, llama31=llama31, **kw)
    f = N.frequencies(32, kw["rope_scale"], kw["rope_theta"], llama31).numpy()
    pairs = y[0, 0, :32].numpy().reshape(16, 2) if interleave else y[0, 0, :32].numpy().reshape(2, 16).T
    turned = (pairs[:, 0] + 1j * pairs[:, 1]) * np.exp(1j * np.array([math.fmod(int(far) * v, 2 * math.pi) for v in f]))
    got = out[0, 0, :32].numpy().reshape(16, 2) if interleave else out[0, 0, :32].numpy().reshape(2, 16).T
    assert np.abs(got - np.stack([turned.real, turned.imag], -1)).max() < 1e-8


def test_probabilities_against_loops():
    g = torch.Generator().manual_seed(2)
    q, k = torch.randn(5, 4, 8, generator=g), torch.randn(7, 2, 8, generator=g)
    seen = torch.arange(7)[None] <= torch.arange(2, 7)[:, None]
    seen[0] = False  # a query that sees nothing adds nothing
    out, bound = E.probabilities(q, k, seen)
    want = torch.zeros(7, 2, dtype=torch.float64)
    for i in range(1, 5):
        for j in range(4):
            e = [math.exp(float(q[i, j].double() @ k[t, j // 2].double()) / math.sqrt(8)) if seen[i, t] else 0.0 for t in range(7)]
            for t in range(7):
                want[t, j // 2] += e[t] / sum(e)
    assert (out - want).abs().max() < 1e-12 and abs(out.sum() - 16) < 1e-12 and (bound[:6] > 0).all()


def test_kept_places_by_hand():
    w = np.array([9, 1, 5, 5, np.nan, -1, 5, 0, 0.5], np.float32)
    assert E.kept_places(w, 9, 2, 2).tolist() == list(range(9))
    assert E.kept_places(w, 5, 1, 1).tolist() == [0, 2, 3, 6, 8]     # three fives
    assert E.kept_places(w, 4, 1, 1).tolist() == [0, 2, 3, 8]        # the first two of them
    assert E.kept_places(w, 3, 3, 0).tolist() == [6, 7, 8]
    assert E.kept_places(w, 3, 0, 3).tolist() == [0, 1, 2]
    assert E.kept_places(w, 8, 0, 0).tolist() == [0, 1, 2, 3, 5, 6, 7, 8]  # NaN goes first
    assert E.kept_places(w[:1], 1, 0, 0).tolist() == [0]
