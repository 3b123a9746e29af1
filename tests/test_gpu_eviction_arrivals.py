"""GPU: eviction of requests whose tokens came by a transfer or back from host memory into pages that others have used."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from mstar_amd.kv_transfer import CPUPagePool
from oracle import eviction as E

pytestmark = pytest.mark.gpu

HQ, HKV, D, PS, PAGES, LAYERS = 4, 2, 64, 16, 40, 2


def _pool(gpu):
    cfg = KVCacheConfig(num_layers=LAYERS, num_kv_heads=HKV, head_dim=D, max_seq_len=512, max_num_pages=PAGES, page_size=PS, num_qo_heads=HQ)
    kv = torch.randn(LAYERS, PAGES, 2, PS, HKV, D, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
    mgr = PagedAllocationManager(cfg, kv, device=gpu)
    for r in "ab":
        mgr.add_request(r, ["main"])
    # what other requests left: all of it heavier than anything that follows
    cm = BatchedCacheManager(["a"], {"a": "main"}, kv, mgr, WorkspaceBufferManager(64 << 20, gpu), cfg, gpu,
                             kv_weights=kv_weights(kv).fill_(1e6))
    return cm, mgr, kv, cfg


def _step(cm, n, gpu, seed):
    cm.plan_attention([n])
    for layer in range(LAYERS):
        x = torch.randn(n, HQ + 2 * HKV, D, generator=torch.Generator().manual_seed(seed + layer)).to(torch.bfloat16).to(gpu)
        cm.run_attention(*x.split([HQ, HKV, HKV], 1), layer_idx=layer, accumulate=True)
    cm.advance_seq_lens()


def _evict_by_what_was_seen(cm, mgr, kv, n, given, keep):
    """Weights are those of the steps since the tokens arrived, and eviction goes by them."""
    st = mgr.get_state("a", "main")
    pages = list(st.page_indices)
    w = cm.kv_weights[:, pages].transpose(2, 3).flatten(1, 2)[:, :n].cpu()
    assert abs(float(w.sum()) - given * HQ * LAYERS) < 1e-3 * given * HQ * LAYERS
    rows = kv[:, pages].transpose(1, 2).flatten(2, 3)[:, :, :n].cpu()  # [layers, K and V, tokens, heads, d]
    cm.evict(keep, recent=4, sinks=1)
    torch.cuda.synchronize()
    kept = kv[:, st.page_indices].transpose(1, 2).flatten(2, 3)[:, :, :keep].cpu()
    for layer in range(LAYERS):
        for h in range(HKV):
            places = torch.as_tensor(E.kept_places(w[layer, :, h].numpy(), keep, 4, 1))
            assert torch.equal(kept[layer, :, :, h], rows[layer][:, places, h])


def test_reloaded(gpu):
    cm, mgr, kv, cfg = _pool(gpu)
    host = CPUPagePool(cfg, 32)
    _step(cm, 100, gpu, 1)
    mgr.offload_request("a", host)
    mgr.alloc("b", "main", 50)
    mgr.reload_request("a", host)
    _step(cm, 3, gpu, 5)
    _evict_by_what_was_seen(cm, mgr, kv, 103, 3, 40)


@pytest.mark.parametrize("first", [0, 40, 48])
def test_read(gpu, first):
    """The whole of a producer's state, and the rest of one of which some tokens are here, with their weights."""
    producer, pm, _, _ = _pool(gpu)
    cm, mgr, kv, _ = _pool(gpu)
    _step(producer, first or 90, gpu, 1)
    mgr.sync_retrieve("a", "main", pm.get_per_label_seq_info("a")["main"])
    seen = 0
    if first:  # a look at them, from a step that is taken back (by a manager of its own: this one keeps to chunks)
        chunks = cm
        cm = BatchedCacheManager(["a"], {"a": "main"}, kv, mgr, cm.buffer_manager, cm.kv_cache_config, gpu, kv_weights=cm.kv_weights)
        cm.plan_attention([1])
        for layer in range(LAYERS):
            x = torch.randn(1, HQ + 2 * HKV, D, generator=torch.Generator().manual_seed(7)).to(torch.bfloat16).to(gpu)
            cm.run_attention(*x.split([HQ, HKV, HKV], 1), layer_idx=layer, accumulate=True)
        st = mgr.get_state("a", "main")
        page, slot = st.page_indices[first // PS], first % PS
        torch.cuda.synchronize()
        cm = chunks
        seen = 1 - float(cm.kv_weights[:, page, :, slot].sum()) / (HQ * LAYERS)
        _step(producer, 90 - first, gpu, 3)
        mgr.sync_retrieve("a", "main", pm.get_per_label_seq_info("a")["main"])
    _step(cm, 3, gpu, 5)
    _evict_by_what_was_seen(cm, mgr, kv, 93, 3 + seen, 40)
