"""CPU: the pages and states of snapshots."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager

PS, PAGES = 16, 64


class _Manager(BatchedCacheManager):
    """Copies pages by indexing: on the CPU there is no launch."""

    def _copy_pages(self, pools, src, dst):
        for kv in pools:
            kv[:, dst] = kv[:, src]


@pytest.fixture
def cm():
    cfg = KVCacheConfig(num_layers=2, num_kv_heads=1, head_dim=64, max_seq_len=1 << 10, max_num_pages=PAGES, page_size=PS)
    kv = torch.rand(2, PAGES, 2, PS, 1, 64)
    mgr = PagedAllocationManager(cfg, kv, device="cpu")
    for r in "ab":
        mgr.add_request(r, ["main", "copy"])
    w = kv_weights(kv)
    return _Manager(["a", "b"], {r: "main" for r in "ab"}, kv, mgr, WorkspaceBufferManager(64, "cpu"), cfg, "cpu",
                    kv_weights=w.copy_(torch.rand(w.shape)))


def _grow(cm, r, n, label="main"):
    st = cm._get_state(r, label)
    cm.alloc_manager.alloc(r, label, st.seq_len + n)
    for i, page in enumerate(st.page_indices):  # new rows, and every token's weight
        if i >= st.seq_len // PS:
            cm.kv_cache[:, page] = torch.rand(cm.kv_cache[:, page].shape)
        cm.kv_weights[:, page] = torch.rand(cm.kv_weights[:, page].shape)
    st.seq_len += n
    st.position_id_start += n


def test_weights_of_a_source_shorter_than_its_copy(cm):
    """No request was cut, and one's copy has gone on beyond it: every request's weights still go to its own copy's pages."""
    _grow(cm, "a", 20)
    _grow(cm, "b", 50)
    cm.snapshot_all("main", "copy")
    _grow(cm, "a", 60, "copy")
    _grow(cm, "b", 3)
    others = cm._get_state("a", "copy").page_indices[2:]
    was = cm.kv_weights[:, others].clone()
    cm.snapshot_all("main", "copy")
    for r, n in (("a", 2), ("b", 4)):
        x, y = (cm._get_state(r, label).page_indices[:n] for label in ("main", "copy"))
        assert torch.equal(cm.kv_weights[:, x], cm.kv_weights[:, y])
    assert torch.equal(cm.kv_weights[:, others], was)
