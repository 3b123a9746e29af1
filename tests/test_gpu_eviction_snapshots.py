"""GPU: a snapshot taken right behind an eviction, over a copy that was made before it and holds more pages."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from mstar_amd.mx_cache import MXKVCache

pytestmark = pytest.mark.gpu

HQ, HKV, D, PS, PAGES, LAYERS = 4, 2, 64, 16, 96, 2


@pytest.mark.parametrize("kind", ["bf16", "mx4"])
def test_right_after_a_cut(gpu, kind):
    cfg = KVCacheConfig(num_layers=LAYERS, num_kv_heads=HKV, head_dim=D, max_seq_len=1024, max_num_pages=PAGES, page_size=PS,
                        num_qo_heads=HQ)
    mx = kind == "mx4"
    kv = MXKVCache(LAYERS, PAGES, PS, HKV, D, bits=4, device=gpu) if mx else torch.zeros(LAYERS, PAGES, 2, PS, HKV, D,
                                                                                        dtype=torch.bfloat16, device=gpu)
    mgr = PagedAllocationManager(cfg, None if mx else kv, device=gpu)
    for r in "abc":
        mgr.add_request(r, ["main", "copy"])
    cm = BatchedCacheManager(list("abc"), {r: "main" for r in "abc"}, kv, mgr, WorkspaceBufferManager(64 << 20, gpu), cfg, gpu,
                             kv_weights=kv_weights(kv))
    g = torch.Generator().manual_seed(3)

    def step(new):
        cm.plan_attention(new)
        for layer in range(LAYERS):
            x = torch.randn(sum(new), HQ + 2 * HKV, D, generator=g).to(torch.bfloat16).to(gpu)
            cm.run_attention(*x.split([HQ, HKV, HKV], 1), layer_idx=layer, accumulate=True)
        cm.advance_seq_lens()

    def same():
        torch.cuda.synchronize()
        for r in "abc":
            a, b = mgr.get_state(r, "main"), mgr.get_state(r, "copy")
            assert (a.seq_len, a.position_id_start, a.evicted, a.dropped) == (b.seq_len, b.position_id_start, b.evicted, b.dropped)
            x, y = a.page_indices, b.page_indices
            assert len(x) == len(y) and not set(x) & set(y)
            for pool in ([kv.codes, kv.scales] if mx else [kv]) + [cm.kv_weights]:
                assert torch.equal(pool[:, x], pool[:, y])
        held = [p for r in "abc" for label in ("main", "copy") for p in mgr.get_state(r, label).page_indices]
        assert sorted(held + list(mgr.page_allocator.free_pages)) == list(range(PAGES))

    step([100, 20, 49])
    cm.snapshot_all("main", "copy")
    same()
    assert cm.evict(40, recent=8, sinks=2) == 4 + 1
    assert [mgr.get_state(r, "main").dropped for r in "abc"] == [60, 0, 9]
    cm.snapshot_all("main", "copy")
    same()
    step([1, 1, 1])
    cm.snapshot_all("main", "copy")
    same()
    cm.set_active_label("copy")
    cm.evict(32)  # now the copy, and it is whole again behind the next snapshot
    cm.snapshot_all("main", "copy")
    same()
