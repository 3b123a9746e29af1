"""CPU: what a run refuses before it launches anything, for every kind of layer, with and without a window.

The wrappers' state is set by hand, as a plan leaves it: nothing here reaches a kernel.
"""

import pytest
import torch

from mstar_amd.mx_cache import MXKVCache
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper

CPU = torch.device("cpu")
BF = torch.bfloat16


def _wrapper(kind, tokens=3, counted=True):
    w = kind.__new__(kind)
    w.device, w.dtype, w.use_cuda_graph = CPU, BF, False
    w.num_qo_heads, w.num_kv_heads, w.head_dim, w.page_size = 8, 2, 128, 16
    w._n_req = w._plan_batch = tokens
    if kind is PagedPrefillWrapper:
        w._total_tokens, w._counted_tokens, w.causal = tokens, tokens if counted else 0, True
        w._plan_max_tokens, w._serial, w._run_short, w._run_tiles = tokens, True, True, True
    w._sm_scale = 1.0
    return w


LAYERS = {"mx8": lambda: MXKVCache(1, 4, 16, 2, 128, bits=8, device="cpu")[0],
          "mx4": lambda: MXKVCache(1, 4, 16, 2, 128, bits=4, device="cpu")[0],
          "bf16": lambda: torch.zeros(4, 2, 16, 2, 128, dtype=BF)}
WINDOWS = [{}, {"window_left": 3}]


@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("layer", LAYERS)
@pytest.mark.parametrize("kind", [PagedDecodeWrapper, PagedPrefillWrapper])
def test_out_that_does_not_take_the_rows(kind, layer, window):
    w, q = _wrapper(kind), torch.zeros(3, 8, 128, dtype=BF)
    for bad in (torch.zeros(2, 8, 128, dtype=BF), torch.zeros(3, 7, 128, dtype=BF), torch.zeros(3, 8, 64, dtype=BF),
                torch.zeros(3, 8, 128, dtype=torch.float16), torch.zeros(3, 8, 128), torch.zeros(3, 8, 128, dtype=BF, device="meta"),
                torch.zeros(3, 1024, dtype=BF), torch.zeros(3, 8, 256, dtype=BF)[..., ::2], torch.zeros(0, 8, 128, dtype=BF)):
        with pytest.raises(ValueError, match="out"):
            w.run(q, LAYERS[layer](), out=bad, **window)


@pytest.mark.parametrize("window", WINDOWS)
@pytest.mark.parametrize("layer", LAYERS)
@pytest.mark.parametrize("kind", [PagedDecodeWrapper, PagedPrefillWrapper])
def test_q_shorter_than_the_plan(kind, layer, window):
    w = _wrapper(kind)
    for rows in (0, 2):
        with pytest.raises(ValueError):
            w.run(torch.zeros(rows, 8, 128, dtype=BF), LAYERS[layer](), **window)


@pytest.mark.parametrize("layer,window", [("mx8", {}), ("mx4", {}), ("bf16", {"window_left": 3})])
def test_q_shorter_than_the_stated_count(layer, window):
    """A caller's own count binds windowed and microscaled runs too."""
    w = _wrapper(PagedPrefillWrapper, counted=False)
    with pytest.raises(ValueError, match="planned"):
        w.run(torch.zeros(2, 8, 128, dtype=BF), LAYERS[layer](), **window)


@pytest.mark.parametrize("kind", [PagedDecodeWrapper, PagedPrefillWrapper])
def test_wider_out(kind):
    """More heads or elements than q's: refused beside a window or a microscaled layer."""
    w, q = _wrapper(kind), torch.zeros(3, 8, 128, dtype=BF)
    for layer, window in (("mx8", {}), ("bf16", {"window_left": 3})):
        for bad in (torch.zeros(3, 9, 128, dtype=BF), torch.zeros(3, 8, 256, dtype=BF)):
            with pytest.raises(ValueError, match="out"):
                w.run(q, LAYERS[layer](), out=bad, **window)
