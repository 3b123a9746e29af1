"""GPU: evictions that would move a plan's pages from under it are refused."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager

pytestmark = pytest.mark.gpu

HQ, HKV, D, PS, PAGES = 4, 2, 64, 16, 32


def test_a_step_that_is_planned_ahead(gpu):
    """The next step's plan holds the pages and lengths of now."""
    cfg = KVCacheConfig(num_layers=1, num_kv_heads=HKV, head_dim=D, max_seq_len=512, max_num_pages=PAGES, page_size=PS, num_qo_heads=HQ)
    kv = torch.zeros(1, PAGES, 2, PS, HKV, D, dtype=torch.bfloat16, device=gpu)
    mgr = PagedAllocationManager(cfg, kv, device=gpu)
    mgr.add_request("r", ["main"])
    cm = BatchedCacheManager(["r"], {"r": "main"}, kv, mgr, WorkspaceBufferManager(64 << 20, gpu), cfg, gpu, kv_weights=kv_weights(kv))

    def run(n):
        q, k, v = torch.ones(n, HQ + 2 * HKV, D, dtype=torch.bfloat16, device=gpu).split([HQ, HKV, HKV], 1)
        cm.run_attention(q, k, v, accumulate=True)
        cm.advance_seq_lens()

    cm.plan_attention([100])
    run(100)
    cm.plan_attention([1])  # ahead, as the graph runner's plan thread does
    cm._pre_planned_labels.add("main")
    st = mgr.get_state("r", "main")
    pages = list(st.page_indices)
    with pytest.raises(ValueError, match="planned"):
        cm.evict(40)
    assert st.page_indices == pages and st.seq_len == 100
    assert cm.evict(100) == 0  # nothing to cut
    cm.plan_attention([1])
    run(1)
    assert cm.evict(40) == 7 - 3
