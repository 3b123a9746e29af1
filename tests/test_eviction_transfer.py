"""CPU: what a reader takes of states that eviction has cut."""

import pytest

from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from mstar_amd.kv_transfer import SequenceInfo


class _Reader:
    """Notes what is read."""

    def __init__(self):
        self.reads = []

    def get_kv_transfer_info(self):
        return "here"

    def read_pages_async(self, info, local, remote, first, last):
        self.reads.append((list(local), list(remote), int(first[0]), int(last[-1])))


def _manager():
    cfg = KVCacheConfig(num_layers=1, num_kv_heads=1, head_dim=64, max_seq_len=1 << 12, max_num_pages=64, page_size=16)
    mgr = PagedAllocationManager(cfg, transfer_engine=_Reader())
    mgr.add_request("r", ["main"])
    return mgr


def _cut(mgr, keep):
    st = mgr.get_state("r", "main")
    mgr.alloc("r", "main", keep)
    st.seq_len, st.position_id_start, st.evicted = keep, 100, True
    return st


def test_a_cut_state_is_read_whole():
    producer, reader = _manager(), _manager()
    _cut(producer, 40)
    info = producer.get_per_label_seq_info("r")["main"]
    assert info.evicted and info.seq_len == 40
    reader.start_async_retrieve("r", "main", info)
    st = reader.get_state("r", "main")
    assert (st.seq_len, st.position_id_start, st.evicted) == (40, 100, True)
    assert reader.kv_transfer_engine.reads == [([0, 1, 2], info.page_indices, 0, 8)]


def test_the_rest_of_a_cut_state_is_refused():
    reader = _manager()
    reader.start_async_retrieve("r", "main", SequenceInfo(20, 20, "there", [5, 6]))
    with pytest.raises(ValueError, match="evicted"):  # cut at the producer since
        reader.start_async_retrieve("r", "main", SequenceInfo(40, 100, "there", [5, 6, 7], evicted=True))
    st = reader.get_state("r", "main")
    assert (st.seq_len, len(st.page_indices), st.evicted) == (20, 2, False)
    reader.reset_label("r", "main")
    reader.start_async_retrieve("r", "main", SequenceInfo(40, 100, "there", [5, 6, 7], evicted=True))
    assert reader.get_state("r", "main").evicted
    with pytest.raises(ValueError, match="evicted"):  # cut here
        reader.start_async_retrieve("r", "main", SequenceInfo(60, 120, "there", [5, 6, 7, 8]))
    reader.start_async_retrieve("r", "main", SequenceInfo(30, 30, "there", [5, 6]))  # nothing to read
    assert len(reader.kv_transfer_engine.reads) == 2


def test_whole_states_go_on():
    reader = _manager()
    for n, pages in ((20, [5, 6]), (40, [5, 6, 7])):
        reader.start_async_retrieve("r", "main", SequenceInfo(n, n, "there", pages))
    assert reader.kv_transfer_engine.reads[1] == ([1, 2], [6, 7], 4, 8)
