"""GPU: a run that is refused for what it should accumulate has not appended, and has not rotated or normalised q and k."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager

pytestmark = pytest.mark.gpu

HQ, HKV, D, PS, PAGES = 4, 2, 64, 16, 16


@pytest.mark.parametrize("weights,window", [(False, -1), (False, 3), (True, 3)])
def test_nothing_is_changed(gpu, weights, window):
    cfg = KVCacheConfig(num_layers=1, num_kv_heads=HKV, head_dim=D, max_seq_len=256, max_num_pages=PAGES, page_size=PS, num_qo_heads=HQ)
    kv = torch.zeros(1, PAGES, 2, PS, HKV, D, dtype=torch.bfloat16, device=gpu)
    mgr = PagedAllocationManager(cfg, kv, device=gpu)
    mgr.add_request("r", ["main"])
    cm = BatchedCacheManager(["r"], {"r": "main"}, kv, mgr, WorkspaceBufferManager(64 << 20, gpu), cfg, gpu,
                             kv_weights=kv_weights(kv) if weights else None)
    cm.plan_attention([5])
    cm.plan_rope([5])
    x = torch.ones(5, HQ + 2 * HKV, D, dtype=torch.bfloat16, device=gpu)
    q, k, v = x.split([HQ, HKV, HKV], 1)
    w = torch.full((D,), 2.0, device=gpu)
    for call in (lambda: cm.run_attention(q, k, v, accumulate=True, window_left=window),
                 lambda: cm.apply_rope_and_run_attention(q, k, v, accumulate=True, window_left=window),
                 lambda: cm.apply_rope_and_run_attention(q, k, v, accumulate=True, window_left=window, q_norm_weight=w, k_norm_weight=w)):
        with pytest.raises(ValueError):
            call()
        torch.cuda.synchronize()
        assert not bool(kv.any()) and bool((x == 1).all())
