"""CPU: which passes of the attention weights a ragged plan asks for, whatever the attention takes for a short request."""

import numpy as np
import pytest
import torch

from mstar_amd import _lib, paged_attention
from mstar_amd.paged_attention import PagedPrefillWrapper


class _Lib:
    """Plans without a GPU, with a given limit of short requests."""

    def __init__(self, short):
        self.short = short

    def mi_prefill_short_rows(self, *sizes):
        return self.short

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.mark.parametrize("short", [1, 4, 8, 16])
@pytest.mark.parametrize("new,want", [([1], 1), ([2], 1), ([4], 1), ([5], 2), ([0], 0), ([0, 0], 0), ([4, 4, 1], 1), ([5, 4], 3), ([0, 600], 2),
                                      ([2] * 130, 1), ([5] * 130, 2), ([3] * 130 + [9], 3), ([2, 2, 300], 3), ([3, 0], 1)])
def test_parts(monkeypatch, short, new, want):
    """4 q heads a kv head: requests of up to 4 tokens have at most 16 rows."""
    monkeypatch.setattr(_lib, "lib", lambda: _Lib(short))
    monkeypatch.setattr(_lib, "stream_ptr", lambda device=None: 0)
    monkeypatch.setattr(torch.cuda, "Stream", lambda **kw: None)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    monkeypatch.setattr(paged_attention, "_pinned_args", lambda parts, n: False)
    monkeypatch.setattr(paged_attention, "_host_args", lambda parts: [t.to(torch.int32) for t in parts])
    w = PagedPrefillWrapper(torch.empty(64, dtype=torch.uint8), 8, 2, 128, 16, device=torch.device("cpu"))
    b = len(new)
    w.plan(torch.tensor([0, *np.cumsum(new)], dtype=torch.int32), torch.arange(b + 1, dtype=torch.int32), torch.arange(b, dtype=torch.int32),
           torch.ones(b, dtype=torch.int32))
    assert w._weights_batch()[3] == want
