"""The 64-bit window reference with NaN and infinities among its keys: a row is what the keys it sees make it."""

import pytest
import torch

from oracle import window as W


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", ["k", "v"])
def test_hidden_keys_take_no_part(which, value):
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(40, h, 16, generator=g, dtype=torch.float64) for h in (4, 2, 2))
    seen = W.visible(40, 40, 4, 2, True)
    clean, bound = W.attend(q, k, v, seen, 2.0 ** -8)
    bad = k.clone(), v.clone()
    bad["kv".index(which)][11, 1, 5] = value
    out, bad_bound = W.attend(q, *bad, seen, 2.0 ** -8)
    rows = seen[:, 11]
    assert rows.sum() == 5
    assert torch.equal(out[:, :2], clean[:, :2]) and torch.equal(bad_bound[:, :2], bound[:, :2])  # the other head
    # another order of summation (only the seen keys): a few 2^-52 of sums of order 1
    assert (out[~rows] - clean[~rows]).abs().max() < 1e-14 and (bad_bound[~rows] - bound[~rows]).abs().max() < 1e-14
    if which == "v":
        assert (out[rows, 2:, 5] == value).all() if value == value else out[rows, 2:, 5].isnan().all()
        others = [d for d in range(16) if d != 5]
        assert (out[rows][:, 2:, others] - clean[rows][:, 2:, others]).abs().max() < 1e-14
    else:
        s = q[:, 2:, 5] * value  # the sign of an infinite score
        gone = rows[:, None] & (s == float("-inf"))  # drops the key
        assert out[:, 2:][rows[:, None] & ~gone].isnan().all()
        assert torch.isfinite(out[:, 2:][gone]).all()


def test_a_row_that_sees_nothing_is_zero_beside_a_nan():
    q, k, v = torch.ones(2, 1, 8), torch.ones(3, 1, 8), torch.ones(3, 1, 8)
    v[1] = float("nan")
    out, bound = W.attend(q, k, v, torch.tensor([[False] * 3, [True, False, True]]), 2.0 ** -8)
    assert (out[0] == 0).all() and (out[1] == 1).all() and torch.isfinite(bound).all()
