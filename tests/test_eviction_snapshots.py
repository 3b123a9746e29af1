"""CPU: the pages and states of snapshots where the source, the copy or both were cut by eviction."""

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


def _cut(cm, r, keep, label="main"):
    st = cm._get_state(r, label)
    need = -(-keep // PS)
    cm.alloc_manager.page_allocator.free(st.page_indices[need:])
    st.dropped += st.seq_len - keep
    st.page_indices, st.seq_len, st.evicted = st.page_indices[:need], keep, True
    cm.kv_cache[:, st.page_indices] = torch.rand(cm.kv_cache[:, st.page_indices].shape)


def _same(cm, a="main", b="copy"):
    held = []
    for r in cm.request_ids:
        x, y = cm._get_state(r, a), cm._get_state(r, b)
        assert (x.seq_len, x.position_id_start, x.evicted, x.dropped) == (y.seq_len, y.position_id_start, y.evicted, y.dropped)
        assert len(x.page_indices) == len(y.page_indices) == -(-x.seq_len // PS)
        assert torch.equal(cm.kv_cache[:, x.page_indices], cm.kv_cache[:, y.page_indices])
        assert torch.equal(cm.kv_weights[:, x.page_indices], cm.kv_weights[:, y.page_indices])
        held += x.page_indices + y.page_indices
    # every page once: held by a state, or free
    assert sorted(held + list(cm.alloc_manager.page_allocator.free_pages)) == list(range(PAGES))


@pytest.mark.parametrize("keep", [1, 16, 17, 32, 99])
@pytest.mark.parametrize("realloc", [False, True])
def test_right_after_a_cut(cm, keep, realloc):
    """The copy was made before the cut and has more pages than are left."""
    _grow(cm, "a", 100)
    _grow(cm, "b", 20)
    cm.snapshot_all("main", "copy")
    _same(cm)
    _cut(cm, "a", keep)
    _grow(cm, "b", 30)
    cm.snapshot_all("main", "copy", realloc=realloc)
    _same(cm)
    _grow(cm, "a", 9)
    _grow(cm, "b", 1)
    cm.snapshot_all("main", "copy", realloc=realloc)
    _same(cm)


def test_a_cut_copy_gets_the_whole_source_back(cm):
    """The copy was cut, the source was not: the copy is whole again, and goes on as whole copies do."""
    _grow(cm, "a", 100)
    _grow(cm, "b", 20)
    cm.snapshot_all("main", "copy")
    _cut(cm, "a", 40, "copy")
    cm.snapshot_all("main", "copy")
    _same(cm)
    assert not cm._get_state("a", "copy").evicted
    before = cm.kv_cache.clone()
    st = cm._get_state("a")
    cm.alloc_manager.alloc("a", "main", 130)
    st.seq_len = st.position_id_start = 130
    cm.kv_cache[:, st.page_indices[6:]] = 7.0
    cm.snapshot_all("main", "copy")
    _same(cm)
    leading = cm._get_state("a", "copy").page_indices[:6]
    assert torch.equal(cm.kv_cache[:, leading], before[:, leading])


def test_restoring_a_source_from_its_copy(cm):
    _grow(cm, "a", 100)
    _grow(cm, "b", 20)
    cm.snapshot_all("main", "copy")
    _cut(cm, "a", 33)
    cm.snapshot_all("copy", "main")
    _same(cm)
    assert cm._get_state("a").seq_len == 100 and not cm._get_state("a").evicted


def test_a_refused_snapshot_changes_nothing(cm):
    """The second request's lists disagree (its copy holds pages ahead, none was cut): no state and no page has changed."""
    _grow(cm, "a", 40)
    _grow(cm, "b", 20)
    cm.snapshot_all("main", "copy")
    _grow(cm, "a", 4)
    cm.alloc_manager.alloc("b", "copy", 60)
    states = [cm._get_state(r, label) for r in "ab" for label in ("main", "copy")]
    was = [(st.seq_len, st.position_id_start, st.evicted, st.dropped, list(st.page_indices)) for st in states]
    kv, w = cm.kv_cache.clone(), cm.kv_weights.clone()
    with pytest.raises(ValueError, match="destination pages"):
        cm.snapshot_all("main", "copy")
    assert was == [(st.seq_len, st.position_id_start, st.evicted, st.dropped, list(st.page_indices)) for st in states]
    assert torch.equal(kv, cm.kv_cache) and torch.equal(w, cm.kv_weights)


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
