"""Cached tokens by the attention they get, and eviction of those that get least.

A request's cache is held to a budget: every step ``accumulate_weights`` of the wrappers
(:mod:`mstar_amd.paged_attention`) adds the step's attention probabilities to a number for
each (token, kv head), and now and then :func:`evict_kv_cache` keeps the first tokens, the
last ones and the heaviest of the others, head by head, and moves them together.

* :func:`kv_weights` -- the weights of a cache's slots, beside its pages;
* :func:`evict_kv_cache` -- one layer or a whole pool, any cache format;
* ``BatchedCacheManager(kv_weights=...)`` with ``accumulate_weights`` and ``evict``, which also
  gives the pages back.

Keys stay rotated to the positions they were written at, and new tokens go on from the
request's last position: only the places in the cache change.

Weights live beside one pool and stay there: tokens that arrive in it by a transfer or from host memory bring
none.  Where a ``BatchedCacheManager`` has the pool's weights, the allocation manager zeroes those tokens' slots as it
queues the copies; a caller that has kept weights writes them behind that, and one that moves pages itself zeroes them.

No counterpart in the reference, whose caches only grow.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .mx_cache import MXKVCache, MXKVLayer, _index

__all__ = ["kv_weights", "evict_kv_cache"]


def _pool_shape(kv_cache) -> tuple[int, ...]:
    """``(layers, max_pages, kv_heads, page_size)``, without ``layers`` for one layer."""
    if isinstance(kv_cache, MXKVCache):
        return (len(kv_cache), *_pool_shape(kv_cache[0]))
    if not isinstance(kv_cache, (torch.Tensor, MXKVLayer)):
        raise ValueError(f"a KV cache is a tensor, an MXKVLayer or an MXKVCache, not {type(kv_cache).__name__}")
    shape = kv_cache.shape
    if len(shape) == 5 and shape[1] == 2:
        return (shape[0], shape[3], shape[2])
    shape = tuple(shape)
    if len(shape) not in (5, 6) or shape[-4] != 2:
        raise ValueError(f"kv_cache must be [(num_layers,) max_pages, 2, page_size, num_kv_heads, head_dim], got {shape}")
    return (*shape[:-5], shape[-5], shape[-2], shape[-3])


def kv_weights(kv_cache: torch.Tensor | MXKVLayer | MXKVCache) -> torch.Tensor:
    """Zero weights for a KV layer or pool: fp32 ``[(num_layers,) max_pages, num_kv_heads, page_size]`` on its device."""
    return torch.zeros(_pool_shape(kv_cache), dtype=torch.float32, device=kv_cache.device)


def _layers(kv_cache, layers: int):
    """(descriptor of the first layer, stride of a layer in its units, stride of a layer's scales in bytes)."""
    if isinstance(kv_cache, MXKVCache):
        return kv_cache[0].desc, kv_cache.codes.stride(0), kv_cache.scales.stride(0)
    if isinstance(kv_cache, MXKVLayer):
        return kv_cache.desc, 0, 0
    layer = kv_cache[0] if kv_cache.dim() == 6 else kv_cache
    scales = (None, None)
    if layer.dtype == torch.float8_e4m3fn:  # codes move as they are: any scales describe the layer
        one = torch.empty(layer.shape[3], dtype=torch.float32, device=layer.device)
        scales = (one, one)
    return _lib.paged_kv_desc(layer, *scales), kv_cache.stride(0) if kv_cache.dim() == 6 else 0, 0


def evict_kv_cache(kv_cache: torch.Tensor | MXKVLayer | MXKVCache, weights: torch.Tensor, kv_indptr: torch.Tensor,
                   kv_indices: torch.Tensor, last_page_len: torch.Tensor, keep: int, recent: int = 0, sinks: int = 0,
                   out_weights: torch.Tensor | None = None) -> torch.Tensor:
    """Hold every request of a batch to ``keep`` tokens; returns the places that stayed.

    Of a request with more than ``keep`` tokens each layer and kv head keeps the first ``sinks``, the
    last ``recent`` and the heaviest of the others by ``weights`` (ties: the lowest place; NaN counts less than any number),
    ``keep`` in all.  Their K, V and weights move to the request's first ``keep`` places, in their order; places
    behind them are left as they were.  Shorter requests are left as they are.  The caller goes on with
    ``min(length, keep)`` tokens a request, and may free the pages behind them.  Windowed runs count places: they
    go on as if nothing had been cut where ``recent`` is at least ``window_left`` and ``sinks`` at least ``sink_tokens``.

    ``kv_cache``: one layer, or a pool of layers (``[num_layers, ...]`` or an ``MXKVCache``) whose ``weights`` (:func:`kv_weights`)
    have the same leading dimension.  The index tensors are those a wrapper plans with; CPU ones are
    copied to the cache's device.  Requests must not share pages.  ``out_weights``: where the kept tokens' weights are
    written, of all requests, instead of in place; ``weights`` then stays as it was, and they must not overlap.

    Returns int32 ``[(num_layers,) batch, num_kv_heads, keep]``: the places in the request that stayed,
    ascending, -1 behind those of a shorter request.
    """
    shape, dev = _pool_shape(kv_cache), kv_cache.device
    if dev.type != "cuda":
        raise ValueError("kv_cache must be on a GPU")
    for name, w in (("weights", weights), ("out_weights", out_weights)):
        if w is not None and (w.dtype is not torch.float32 or w.shape != shape or not w.is_contiguous() or w.get_device() != dev.index
                              or w.data_ptr() % 16):
            raise ValueError(f"{name} must be a contiguous, 16-byte aligned float32 tensor {shape} on {dev}, got {tuple(w.shape)}, "
                             f"{w.dtype} on {w.device}")
    if out_weights is not None and 0 < abs(out_weights.data_ptr() - weights.data_ptr()) < 4 * weights.numel():
        raise ValueError("out_weights must not overlap weights, unless it is the same tensor")
    keep, recent, sinks = int(keep), int(recent), int(sinks)
    if keep < 1 or recent < 0 or sinks < 0 or recent + sinks > keep:
        raise ValueError(f"keep {keep} must be positive and hold recent {recent} and sinks {sinks}")
    if keep > _KEEP_MAX:
        raise ValueError(f"keep {keep} is beyond {_KEEP_MAX}")
    indptr, indices, last = _index(kv_indptr, dev), _index(kv_indices, dev), _index(last_page_len, dev)
    batch = indptr.shape[0] - 1
    if batch < 0 or last.shape[0] != batch:
        raise ValueError("index tensors disagree on the number of requests")
    layers = shape[0] if len(shape) == 4 else 1
    desc, layer_stride, scale_stride = _layers(kv_cache, layers) if layers else (None, 0, 0)
    kept = torch.empty((*shape[:-3], batch, shape[-2], keep), dtype=torch.int32, device=dev)
    if kept.numel() == 0:
        return kept
    if indices.shape[0] == 0:
        return kept.fill_(-1)
    out = weights if out_weights is None else out_weights
    status = _lib.lib().mi_kv_evict_block(_lib.KV_EVICT_ARGS.pack(
        ctypes.addressof(desc), weights.data_ptr(), out.data_ptr(), indptr.data_ptr(), indices.data_ptr(), last.data_ptr(),
        kept.data_ptr(), _lib.stream_ptr(dev), layer_stride, scale_stride, weights.stride(0) if len(shape) == 4 else 0, layers, batch,
        indices.shape[0], keep, recent, sinks))
    if status:
        _lib.check(status, "mi_kv_evict")
    return kept


_KEEP_MAX = 1 << 30  # beyond any context
