"""CPU: what stands for a KV layer, and what does not."""

import pytest
import torch

from mstar_amd import _lib
from mstar_amd.mx_cache import MXKVCache, read_kv_cache


def test_a_pool_is_no_layer():
    pool = MXKVCache(2, 4, 16, 2, 128, device="cpu")
    assert _lib.paged_kv_desc(pool[1]) is pool[1].desc
    for bad in (pool, [pool[0]], None, 3, pool[0].desc):
        with pytest.raises(ValueError, match="layer"):
            _lib.paged_kv_desc(bad)
        with pytest.raises(ValueError):
            read_kv_cache(bad, *[torch.zeros(1, dtype=torch.int32)] * 3, 0)
    one = torch.ones(2)
    with pytest.raises(ValueError, match="scales"):
        _lib.paged_kv_desc(pool[0], one, one)
