"""GPU: requests of a few queries and rows: what is not finite in one stays with the keys that its query sees."""

import pytest
import torch

import mx_helpers as H
from gpu_helpers import workspace
from mstar_amd.eviction import kv_weights
from mstar_amd.paged_attention import PagedPrefillWrapper
from oracle import eviction as E
from oracle import window as W

pytestmark = pytest.mark.gpu


def _call(p, gpu, q, new, weights, causal=True):
    hkv, d = p.values.shape[3], p.values.shape[4]
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), q.shape[1], hkv, d, p.ps, device=gpu)
    qo = torch.tensor([0, *torch.tensor(new).cumsum(0).tolist()], dtype=torch.int32)
    w.plan(qo, *p.index(), causal=causal, dtype=q.dtype)
    w.accumulate_weights(q.to(gpu), p.layer, weights, *p.scales)


def _of(p, weights, r):
    """[kv_heads, tokens] of request r."""
    pages = torch.as_tensor(p.kv_indices[p.kv_indptr[r]:p.kv_indptr[r + 1]]).long()
    return weights.cpu()[pages].permute(1, 0, 2).flatten(1)[:, :p.lens[r]]


# one launch (up to 512 tokens on average), and scores through memory; rows in and past the eight that are loaded ahead
@pytest.mark.parametrize("lens", [[40, 30], [0 + 5, 3], [700, 300], [9000, 20], [5, 6000]])
@pytest.mark.parametrize("kind,hq,hkv,d,n", [("bf16", 6, 2, 128, 3), ("bf16", 4, 4, 64, 16), ("f16", 3, 1, 256, 5), ("fp8", 8, 2, 128, 4),
                                             ("mx4", 4, 2, 128, 8)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite(gpu, lens, kind, hq, hkv, d, n, bad):
    lens = [max(x, n) for x in lens]
    p = H.make(gpu, kind, lens, 16, hkv, d, seed=5)
    g = torch.Generator().manual_seed(2)
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    for row in {0, n // 2, n - 1}:
        q = torch.randn(2 * n, hq, d, generator=g).to(dtype)
        q[row, hq // hkv - 1, 3] = bad  # request 0, the last q head of kv head 0
        weights = kv_weights(p.layer)
        _call(p, gpu, q, [n, n], weights)
        off = lens[0] - n
        got = _of(p, weights, 0)
        k = p.rows(0, 0)
        if bad != bad or bool((k[:off + row + 1, 0, 3] >= 0).any()):  # scores of -infinity alone are no NaN
            assert bool(got[0, :off + row + 1].isnan().all()), "keys that the query sees"
        # keys behind it: the sums of the other queries, and of its own other heads, which see none of them
        for h in range(hkv):
            heads = slice(h * hq // hkv, (h + 1) * hq // hkv)
            first = row + 1 if h == 0 else 0
            if first < n:
                want, bound = E.probabilities(q[first:n, heads], k[:, h:h + 1], W.visible(lens[0], n, -1, 0, True)[first:])
                t = off + first
                assert ((got[h, t:].double() - want[t:, 0]).abs() <= bound[t:, 0] + want[t:, 0] * 2.0 ** -23).all(), (row, h)
        assert bool(_of(p, weights, 1).isfinite().all())


@pytest.mark.parametrize("lens", [[40], [9000]])
def test_a_nan_key_of_the_steps_own(gpu, lens):
    """A step's own key that is NaN reaches the queries from its own on, and through them all that they see."""
    n, hq = 4, 6
    p = H.make(gpu, "bf16", lens, 16, 2, 128, seed=5)
    q = torch.randn(n, hq, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    at = lens[0] - 2  # seen by the queries 2 and 3
    p.layer[int(p.kv_indices[at // 16]), 0, at % 16, 1, 0] = float("nan")
    weights = kv_weights(p.layer)
    _call(p, gpu, q, [n], weights)
    got = _of(p, weights, 0)
    assert bool(got[0].isfinite().all()) and bool(got[1].isnan().all())
    weights.zero_()
    p.layer[int(p.kv_indices[at // 16]), 0, at % 16, 1, 0] = 1.0
    at = lens[0] - 1  # seen by the last query alone, which sees every key
    p.layer[int(p.kv_indices[at // 16]), 0, at % 16, 0, 5] = float("nan")
    _call(p, gpu, q, [n], weights)
    got = _of(p, weights, 0)
    assert bool(got[0].isnan().all()) and bool(got[1].isfinite().all())


def test_without_causal_every_key_is_seen(gpu):
    for lens in ([40], [9000]):
        p = H.make(gpu, "bf16", lens, 16, 2, 128, seed=5)
        q = torch.randn(4, 6, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        q[0, 0, 0] = float("nan")
        weights = kv_weights(p.layer)
        _call(p, gpu, q, [4], weights, causal=False)
        got = _of(p, weights, 0)
        assert bool(got[0].isnan().all()) and bool(got[1].isfinite().all())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_more_queries_than_keys(gpu, dtype):
    """Queries before the first key see nothing: NaN in one reaches nothing."""
    hq, hkv, d, ps, n = 4, 1, 128, 16, 4
    g = torch.Generator().manual_seed(4)
    layer = torch.randn(4, 2, ps, hkv, d, generator=g).to(dtype).to(gpu)
    q = torch.randn(n, hq, d, generator=g).to(dtype)
    q[0, 1, 7] = float("nan")
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu)
    w.plan(torch.tensor([0, n], dtype=torch.int32), torch.tensor([0, 1], dtype=torch.int32), torch.tensor([2], dtype=torch.int32),
           torch.tensor([2], dtype=torch.int32), dtype=dtype)
    weights = kv_weights(layer)
    w.accumulate_weights(q.to(gpu), layer, weights)
    got = weights.cpu()[2, 0, :2].double()
    want, bound = E.probabilities(q[2:], layer[2, 0, :2].cpu(), W.visible(2, 2, -1, 0, True))
    assert ((got - want[:, 0]).abs() <= bound[:, 0] + want[:, 0] * 2.0 ** -23).all()
