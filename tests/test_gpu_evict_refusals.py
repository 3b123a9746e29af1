"""GPU: evictions that would move a plan's pages from under it, or write weights over ones still to be read, are refused."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import evict_kv_cache, kv_weights
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


def test_out_weights_over_weights(gpu):
    """The same tensor is in place; a part of it would be written over places still to be read."""
    kv = torch.zeros(2, PAGES, 2, PS, HKV, D, dtype=torch.bfloat16, device=gpu)
    flat = torch.rand(3 * PAGES * HKV * PS, device=gpu)
    w = flat[: 2 * PAGES * HKV * PS].view(2, PAGES, HKV, PS)
    idx = [torch.tensor(x, dtype=torch.int32, device=gpu) for x in ([0, 4], [3, 1, 2, 0], [5])]
    was = flat.clone()
    for at in (4, PAGES * HKV * PS):
        other = flat[at:at + w.numel()].view(w.shape)
        for a, b in ((w, other), (other, w)):
            with pytest.raises(ValueError, match="overlap"):
                evict_kv_cache(kv, a, *idx, keep=20, out_weights=b)
    torch.cuda.synchronize()
    assert torch.equal(flat, was)
    one = w.clone()
    a = evict_kv_cache(kv, one, *idx, keep=20, out_weights=one.view(one.shape))  # in place
    b = evict_kv_cache(kv[0], w[0], *idx, keep=20, out_weights=w[1])  # beside one another
    torch.cuda.synchronize()
    assert torch.equal(a[0], b)
