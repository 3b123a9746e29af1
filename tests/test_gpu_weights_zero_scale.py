"""GPU: scores that are all zero because their scale is: every query gives each key that it sees the same weight."""

import ctypes

import numpy as np
import pytest
import torch

import mx_helpers as H
from gpu_helpers import workspace
from mstar_amd import _lib
from mstar_amd.eviction import kv_weights
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper

pytestmark = pytest.mark.gpu


def _uniform(length, n, causal):
    """[length]: of n queries and one head."""
    w = np.zeros(length)
    for i in range(n):
        seen = length - n + i + 1 if causal else length
        w[:seen] += 1 / seen
    return torch.from_numpy(w)


@pytest.mark.parametrize("d,hq,hkv", [(64, 4, 2), (128, 8, 2), (256, 6, 2)])
@pytest.mark.parametrize("lens,new,causal", [([300, 50], [64, 20], True), ([300, 50], [64, 20], False), ([37, 2000], [37, 33], True),
                                             ([40, 700], [3, 1], True), ([40, 700], None, False)])
@pytest.mark.parametrize("value", [0.0, -0.0])
def test_a_head_whose_scale_is_zero(gpu, d, hq, hkv, lens, new, causal, value):
    """An fp8 layer's head with k_scale 0: chunks, a few queries and single ones agree; the other head is as it was."""
    p = H.make(gpu, "fp8", lens, 16, hkv, d, seed=d)
    counts = new or [1] * len(lens)
    q = torch.randn(sum(counts), hq, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
    if new is None:
        w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, 16, device=gpu)
        w.plan(*p.index())
    else:
        w = PagedPrefillWrapper(workspace(gpu, 64 << 20), hq, hkv, d, 16, device=gpu)
        w.plan(torch.tensor([0, *np.cumsum(new)], dtype=torch.int32), *p.index(), causal=causal)
    plain, weights = kv_weights(p.layer), kv_weights(p.layer)
    w.accumulate_weights(q, p.layer, plain, *p.scales)
    ks = p.scales[0].clone()
    ks[1] = value
    w.accumulate_weights(q, p.layer, weights, ks, p.scales[1])
    assert torch.equal(weights[:, 0], plain[:, 0])
    for r, (length, n) in enumerate(zip(lens, counts)):
        pages = torch.as_tensor(p.kv_indices[p.kv_indptr[r]:p.kv_indptr[r + 1]]).long()
        got = weights[:, 1].cpu()[pages].flatten()[:length].double()
        want = _uniform(length, n, causal) * (hq // hkv)
        # a query's share: the log of a sum of ones (its logarithm off by two units of its size) in fp32, and sums of fewer than 2^8 rows
        assert ((got - want).abs() <= want * (2 * 11 * 2.0 ** -23 + (n * hq + length / 16 + 64) * 2.0 ** -24)).all(), r


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_call_whose_scale_is_zero(gpu, dtype):
    """sm_scale 0 in the C call, over a request of many rows and one of few."""
    hq, hkv, d, lens, new = 4, 1, 128, [100, 60], [50, 2]
    g = torch.Generator().manual_seed(3)
    layer = torch.randn(12, 2, 16, hkv, d, generator=g).to(dtype).to(gpu)
    q = torch.randn(sum(new), hq, d, generator=g).to(dtype).to(gpu)
    qo, indptr, indices, last = (torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, 50, 52], [0, 7, 11], list(range(11)), [4, 12]))
    weights = kv_weights(layer)
    L, mi = _lib.lib(), _lib.TORCH_TO_MI[dtype]
    nbytes = L.mi_attention_weights_bytes(2, 52, 11, 16, hq, hkv, 1, 3)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=gpu)
    _lib.check(L.mi_attention_weights(q.data_ptr(), mi, hq * d, d, ctypes.byref(_lib.paged_kv_desc(layer)), qo.data_ptr(), indptr.data_ptr(),
                                      indices.data_ptr(), last.data_ptr(), 2, 52, 11, hq, 1, 0.0, 3, weights.data_ptr(), ws.data_ptr(), nbytes,
                                      _lib.stream_ptr(gpu)), "mi_attention_weights")
    torch.cuda.synchronize()
    for r, (a, b) in enumerate(((0, 7), (7, 11))):
        got, want = weights[a:b, 0].cpu().flatten()[:lens[r]].double(), _uniform(lens[r], new[r], True) * hq
        assert ((got - want).abs() <= want * (2 * 7 * 2.0 ** -23 + (new[r] * hq + 80) * 2.0 ** -24)).all(), r


def test_what_is_not_finite_still_counts(gpu):
    """Zero times a NaN or an infinity is no zero: those keys and queries make NaN what they meet, whatever the scale."""
    lens, new, hq, hkv, d = [300], [64], 4, 2, 128
    p = H.make(gpu, "fp8", lens, 16, hkv, d, seed=2)
    ks = p.scales[0].clone()
    ks[1] = 0.0
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), hq, hkv, d, 16, device=gpu)
    w.plan(torch.tensor([0, 64], dtype=torch.int32), *p.index())
    pages = torch.as_tensor(p.kv_indices).long()
    for bad in (float("nan"), float("inf")):
        q = torch.randn(64, hq, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        q[10, 3, 5] = bad  # of kv head 1; sees the keys up to 246
        weights = kv_weights(p.layer)
        w.accumulate_weights(q.to(gpu), p.layer, weights, ks, p.scales[1])
        got = weights.cpu()[pages].permute(1, 0, 2).flatten(1)[:, :300]
        assert bool(got[1, :247].isnan().all()) and bool(got[1, 247:].isfinite().all()) and bool(got[0].isfinite().all())
