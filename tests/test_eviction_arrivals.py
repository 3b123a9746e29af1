"""CPU: weights of tokens that arrive in a pool by a transfer or from host memory: none, whatever their pages' last owners left."""

import pytest
import torch

from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.eviction import kv_weights
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from mstar_amd.kv_transfer import OffloadedState, SequenceInfo

PS, PAGES, LAYERS, HEADS = 16, 32, 2, 3


class _Reader:
    def get_kv_transfer_info(self):
        return "here"

    def read_pages_async(self, info, local, remote, first, last):
        return None


class _HostPool:
    """A CPU pool that keeps no rows."""

    def __init__(self):
        self.offloaded = {}

    def offload_pages(self, rid, label, kv, pages, seq_len, pos, **more):
        self.offloaded.setdefault(rid, {})[label] = OffloadedState(list(range(len(pages))), seq_len, pos, **more)

    def reload_pages(self, rid, label, kv, pages):
        st = self.offloaded[rid].pop(label)
        return st.seq_len, st.position_id_start

    def sync(self):
        pass


def _pool(weights=True):
    cfg = KVCacheConfig(num_layers=LAYERS, num_kv_heads=HEADS, head_dim=64, max_seq_len=1 << 10, max_num_pages=PAGES, page_size=PS)
    kv = torch.zeros(LAYERS, PAGES, 2, PS, HEADS, 64)
    mgr = PagedAllocationManager(cfg, kv, device="cpu", transfer_engine=_Reader())
    for r in "ab":
        mgr.add_request(r, ["main"])
    w = kv_weights(kv).fill_(5.0)
    cm = BatchedCacheManager(["a"], {"a": "main"}, kv, mgr, WorkspaceBufferManager(64, "cpu"), cfg, "cpu", kv_weights=w if weights else None)
    return mgr, cm, w


def _rest(w, pages):
    return w[:, [p for p in range(PAGES) if p not in pages]]


@pytest.mark.parametrize("here,there", [(0, 1), (0, 16), (0, 50), (20, 21), (20, 32), (20, 33), (32, 60), (37, 48)])
def test_read_tokens_bring_no_weights(here, there):
    mgr, _, w = _pool()
    st = mgr.get_state("a", "main")
    mgr.alloc("a", "main", here)
    st.seq_len = st.position_id_start = here
    mgr.start_async_retrieve("a", "main", SequenceInfo(there, there, "there", list(range(8))))
    mine = w[:, st.page_indices].transpose(1, 2).flatten(2)  # [layers, heads, slots]
    assert bool((mine[..., :here] == 5).all()) and not bool(mine[..., here:there].any())
    assert bool((_rest(w, st.page_indices) == 5).all())


def test_reloaded_tokens_bring_no_weights():
    mgr, _, w = _pool()
    host = _HostPool()
    st = mgr.get_state("a", "main")
    mgr.alloc("a", "main", 40)
    st.seq_len = 40
    mgr.offload_request("a", host)
    mgr.alloc("b", "main", 100)  # another request uses pages meanwhile
    assert bool((w == 5).all())
    mgr.reload_request("a", host)
    st = mgr.get_state("a", "main")
    assert len(st.page_indices) == 3 and not bool(w[:, st.page_indices].any()) and bool((_rest(w, st.page_indices) == 5).all())
    w[:, st.page_indices] = 2.0  # a caller that sets its own goes on from them
    cm = _pool()[1]
    assert cm.alloc_manager.kv_weights is cm.kv_weights and bool((w[:, st.page_indices] == 2).all())


def test_a_pool_without_weights():
    mgr, _, w = _pool(weights=False)
    host = _HostPool()
    mgr.start_async_retrieve("a", "main", SequenceInfo(50, 50, "there", list(range(8))))
    mgr.offload_request("a", host)
    mgr.reload_request("a", host)
    assert mgr.kv_weights is None and bool((w == 5).all())


def test_weights_given_later_are_the_pools():
    mgr, cm, w = _pool(weights=False)
    cm.kv_weights = w
    mgr.start_async_retrieve("a", "main", SequenceInfo(16, 16, "there", [0]))
    assert not bool(w[:, mgr.get_state("a", "main").page_indices].any())


def _cut(mgr, keep):
    st = mgr.get_state("a", "main")
    mgr.page_allocator.free(st.page_indices[-(-keep // PS):])
    st.dropped += st.seq_len - keep
    st.page_indices, st.seq_len, st.evicted = st.page_indices[: -(-keep // PS)], keep, True


@pytest.mark.parametrize("removed", [False, True])
def test_a_cut_state_is_cut_when_it_comes_back(removed):
    """Also to a request that was removed and added again meanwhile, and its state on the GPU is empty and whole until then."""
    mgr, _, _ = _pool()
    host = _HostPool()
    mgr.alloc("a", "main", 100)
    st = mgr.get_state("a", "main")
    st.seq_len = st.position_id_start = 100
    _cut(mgr, 40)
    mgr.offload_request("a", host)
    assert (st.seq_len, st.evicted, st.dropped) == (0, False, 0)
    if removed:
        mgr.remove_request("a")
        mgr.add_request("a", ["main"])
    mgr.reload_request("a", host)
    st = mgr.get_state("a", "main")
    assert (st.seq_len, st.position_id_start, st.evicted, st.dropped) == (40, 100, True, 60)
    with pytest.raises(ValueError, match="evicted"):
        mgr.start_async_retrieve("a", "main", SequenceInfo(110, 110, "there", list(range(8))))


def test_a_state_filled_anew_behind_an_offload_is_whole():
    mgr, _, _ = _pool()
    mgr.alloc("a", "main", 100)
    st = mgr.get_state("a", "main")
    st.seq_len = st.position_id_start = 100
    _cut(mgr, 40)
    mgr.offload_request("a", _HostPool())
    mgr.alloc("a", "main", 20)  # a prompt once more
    st.seq_len = st.position_id_start = 20
    mgr.start_async_retrieve("a", "main", SequenceInfo(50, 50, "there", list(range(8))))
    assert (st.seq_len, st.evicted) == (50, False)


def test_host_pools_of_plain_states():
    """A pool that knows nothing of cuts holds whole states as before."""

    class Plain(_HostPool):
        def offload_pages(self, rid, label, kv, pages, seq_len, pos):
            self.offloaded.setdefault(rid, {})[label] = type("State", (), dict(cpu_page_indices=list(range(len(pages))), seq_len=seq_len,
                                                                               position_id_start=pos))

    mgr, _, _ = _pool()
    host = Plain()
    mgr.alloc("a", "main", 40)
    st = mgr.get_state("a", "main")
    st.seq_len = st.position_id_start = 40
    mgr.offload_request("a", host)
    mgr.reload_request("a", host)
    assert (st.seq_len, st.evicted, st.dropped) == (40, False, 0)
