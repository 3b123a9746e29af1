"""CPU: a reader that holds tokens and is told of a state that eviction has cut, longer or shorter than its own."""

import pytest

from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from mstar_amd.kv_transfer import SequenceInfo


class _Reader:
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


def _given(mgr, tokens, keep=None):
    """A state that was given so many tokens and cut to ``keep`` afterwards, as an eviction leaves it."""
    st = mgr.get_state("r", "main")
    mgr.alloc("r", "main", tokens)
    st.seq_len = st.position_id_start = tokens
    if keep is not None:
        _cut(st, keep)
    return st


def _cut(st, keep):
    st.dropped += st.seq_len - keep
    st.page_indices, st.seq_len, st.evicted = st.page_indices[: -(-keep // 16)], keep, True


@pytest.mark.parametrize("given", [49, 60, 61, 62, 100])
def test_a_cut_state_shorter_than_the_readers_is_refused(given):
    """60 tokens here, 48 left of ``given`` there: what is here is not a part of it, however their lengths compare."""
    producer, reader = _manager(), _manager()
    _given(producer, given, 48)
    st = _given(reader, 60)
    pages = list(st.page_indices)
    with pytest.raises(ValueError, match="evicted"):
        reader.start_async_retrieve("r", "main", producer.get_per_label_seq_info("r")["main"])
    assert (st.seq_len, st.position_id_start, st.evicted, st.page_indices) == (60, 60, False, pages)
    assert not reader.kv_transfer_engine.reads and not st.read_in_progress


def test_only_the_flag_and_lengths_are_needed():
    """A description that says no more than that its state is cut."""
    reader = _manager()
    _given(reader, 60)
    with pytest.raises(ValueError, match="evicted"):
        reader.start_async_retrieve("r", "main", SequenceInfo(48, 62, "there", [5, 6, 7], evicted=True))
    with pytest.raises(ValueError, match="evicted"):
        reader.start_async_retrieve("r", "main", SequenceInfo(60, 60, "there", [5, 6, 7, 8], evicted=True))


def test_the_same_cut_state_again_is_nothing_to_read():
    producer, reader = _manager(), _manager()
    st = _given(producer, 100, 40)
    for _ in range(3):
        reader.start_async_retrieve("r", "main", producer.get_per_label_seq_info("r")["main"])
    assert len(reader.kv_transfer_engine.reads) == 1
    st.seq_len += 8  # it goes on, and is cut to the same length again: other tokens
    st.position_id_start += 8
    mgr_pages = list(st.page_indices)
    _cut(st, 40)
    assert st.page_indices == mgr_pages[:3]
    with pytest.raises(ValueError, match="evicted"):
        reader.start_async_retrieve("r", "main", producer.get_per_label_seq_info("r")["main"])
    reader.reset_label("r", "main")
    reader.start_async_retrieve("r", "main", producer.get_per_label_seq_info("r")["main"])
    got = reader.get_state("r", "main")
    assert (got.seq_len, got.position_id_start, got.evicted, got.dropped) == (40, 108, True, 68)
    assert len(reader.kv_transfer_engine.reads) == 2


def test_positions_that_stand_still():
    """Tokens that share a position (an image's): a cut at one length and position is told from another by what was dropped."""
    producer, reader = _manager(), _manager()
    st = _given(producer, 100, 40)
    reader.start_async_retrieve("r", "main", producer.get_per_label_seq_info("r")["main"])
    st.seq_len += 8
    _cut(st, 40)
    with pytest.raises(ValueError, match="evicted"):
        reader.start_async_retrieve("r", "main", producer.get_per_label_seq_info("r")["main"])


def test_a_reader_that_has_gone_on():
    """From a cut state that it has read, and been cut again itself: nothing to read there."""
    producer, reader = _manager(), _manager()
    _given(producer, 100, 40)
    info = producer.get_per_label_seq_info("r")["main"]
    reader.start_async_retrieve("r", "main", info)
    st = reader.get_state("r", "main")
    reader.alloc("r", "main", 50)
    st.seq_len, st.position_id_start = 50, 110
    reader.start_async_retrieve("r", "main", info)
    _cut(st, 32)
    reader.start_async_retrieve("r", "main", info)
    assert (st.seq_len, st.position_id_start, st.dropped) == (32, 110, 78) and len(reader.kv_transfer_engine.reads) == 1


def test_a_reader_cut_by_itself():
    """48 of 60 tokens here: nothing to read of a whole state up to 60, a refusal behind that."""
    reader = _manager()
    _given(reader, 60, 48)
    for there in (30, 48, 59, 60):
        reader.start_async_retrieve("r", "main", SequenceInfo(there, there, "there", [5, 6, 7, 8]))
    for info in (SequenceInfo(61, 61, "there", [5, 6, 7, 8]), SequenceInfo(40, 62, "there", [5, 6, 7]),
                 SequenceInfo(40, 60, "there", [5, 6, 7], evicted=True, dropped=20)):
        with pytest.raises(ValueError, match="evicted"):
            reader.start_async_retrieve("r", "main", info)
    assert not reader.kv_transfer_engine.reads


def test_an_empty_state_has_nothing_to_be_behind():
    reader = _manager()
    reader.start_async_retrieve("r", "main", SequenceInfo(0, 0, "there", []))
    reader.start_async_retrieve("r", "main", SequenceInfo(0, 0, "there", [], evicted=True))
    assert reader.get_state("r", "main").seq_len == 0 and not reader.kv_transfer_engine.reads
