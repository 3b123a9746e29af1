"""GPU: rotation with append into a microscaled layer leaves q and k as they were where the append is refused."""

import pytest
import torch

from gpu_helpers import workspace
from mstar_amd.mx_cache import MXKVCache
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", [PagedDecodeWrapper, PagedPrefillWrapper])
def test_nothing_is_rotated_before_a_refusal(gpu, kind):
    w = kind(workspace(gpu, 64 << 20), 8, 2, 128, 16, device=gpu)
    index = [torch.tensor(x, dtype=torch.int32) for x in ([0, 1, 2], [2, 0], [5, 9])]
    w.plan(*([torch.tensor([0, 1, 2], dtype=torch.int32)] if kind is PagedPrefillWrapper else []), *index)
    layer = MXKVCache(1, 4, 16, 2, 128, device=gpu)[0]
    g = torch.Generator().manual_seed(0)
    q, k, v = (torch.randn(2, h, 128, generator=g).to(torch.bfloat16).to(gpu) for h in (8, 2, 2))
    pos, one = torch.tensor([4, 8], device=gpu), torch.ones(2, device=gpu)
    before = q.clone(), k.clone()
    for layer_, v_, scales in ((layer, v[:, :1], {}), (layer, v[:1], {}), (layer, v.cpu(), {}), (layer, v, {"k_scale": one}),
                               (MXKVCache(1, 4, 16, 2, 64, device=gpu)[0], v, {}), (MXKVCache(1, 4, 16, 2, 128, device="cpu")[0], v, {})):
        with pytest.raises(ValueError):
            w.rope_set_kv_cache(layer_, q, k, v_, pos, **scales)
        assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    with pytest.raises(ValueError):
        w.rope_set_kv_cache(layer, q[:1], k[:1], v[:1], pos)  # fewer tokens than planned
    assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    w.rope_set_kv_cache(layer, q, k, v, pos)
    assert not torch.equal(q, before[0]) and layer.codes.any()
