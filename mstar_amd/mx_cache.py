"""The microscaled KV cache: 8- or 4-bit codes that share a power-of-two scale per 32 elements.

The fp8 cache of the wrappers needs one scale per kv-head, found beforehand; here the
scales come from the values as they are appended, a byte for each block of 32 consecutive
elements of a (token, kv-head) row of K or V.  A cached element takes 8.25 or 4.25 bits.
The formats are the OCP microscaling ones: e4m3 or e2m1 codes, E8M0 scales.

* :class:`MXKVLayer` -- one layer's codes and scales, given to the wrappers' ``set_kv_cache``
  and ``run`` in the place of a KV layer tensor;
* :class:`MXKVCache` -- a pool of layers, given to ``BatchedCacheManager`` and
  ``PagedAllocationManager`` in the place of the ``kv_cache`` tensor;
* :func:`read_kv_cache` -- a batch's contexts back as values, from any cache format.

No counterpart in the reference, whose cache is 16- or 32-bit (``kv_cache_engine.py:132-136``).
"""

from __future__ import annotations

import torch

from . import _lib

__all__ = ["MXKVLayer", "MXKVCache", "read_kv_cache", "MX_BLOCK"]

MX_BLOCK = 32  # elements that share a scale

_BYTES = {torch.uint8, torch.float8_e4m3fn}
_SCALES = {torch.uint8, torch.float8_e8m0fnu}
_OUT = {torch.bfloat16: _lib.MI_BF16, torch.float16: _lib.MI_F16, torch.float32: _lib.MI_F32}


class MXKVLayer:
    """One KV layer in a microscaled format.

    ``codes``: ``[max_pages, 2, page_size, num_kv_heads, head_dim]`` bytes (uint8 or
    float8_e4m3fn) at 8 bits, ``[..., head_dim // 2]`` (uint8) at 4, the even element in a
    byte's low four bits; any strides that are whole multiples of 16 bytes, the last
    dimension contiguous.  ``scales``: ``[max_pages, 2, num_kv_heads, head_dim // 32,
    page_size]`` (uint8 or float8_e8m0fnu), contiguous: tokens innermost, so that four
    tokens' scales are one load.  A scale byte s stands for 2^(s - 127), 255 for a block
    of NaN.  The tensors are the caller's; the layer describes them as they are now.
    """

    __slots__ = ("codes", "scales", "bits", "head_dim", "desc", "device")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        if codes.dim() != 5 or codes.shape[1] != 2 or scales.dim() != 5:
            raise ValueError("codes must be [max_pages, 2, page_size, num_kv_heads, bytes] and scales "
                             f"[max_pages, 2, num_kv_heads, blocks, page_size], got {tuple(codes.shape)}, {tuple(scales.shape)}")
        if codes.dtype not in _BYTES or scales.dtype not in _SCALES:
            raise ValueError(f"codes must be uint8 or float8_e4m3fn and scales uint8 or float8_e8m0fnu, got {codes.dtype}, "
                             f"{scales.dtype}")
        pages, _, page_size, heads, width = codes.shape
        if tuple(scales.shape) != (pages, 2, heads, scales.shape[3], page_size) or scales.shape[3] < 1:
            raise ValueError(f"scales {tuple(scales.shape)} do not fit codes {tuple(codes.shape)}")
        self.head_dim = MX_BLOCK * scales.shape[3]
        if width not in (self.head_dim, self.head_dim // 2) or (width != self.head_dim and codes.dtype != torch.uint8):
            raise ValueError(f"{width} code bytes a row are neither 8 nor 4 bits for head_dim {self.head_dim}")
        self.bits = 8 if width == self.head_dim else 4
        if codes.device != scales.device:
            raise ValueError("codes and scales must live on one device")
        if codes.stride(4) != 1 or any(s % 16 for s in codes.stride()[:4]) or codes.data_ptr() % 16:
            raise ValueError("codes: rows must be contiguous and 16-byte aligned")
        if not scales.is_contiguous() or scales.data_ptr() % 4 or page_size % 4:
            raise ValueError("scales must be contiguous and 4-byte aligned")
        self.codes, self.scales, self.device = codes, scales, codes.device
        d = self.desc = _lib.MiPagedKV()
        d.data = codes.data_ptr()
        d.dtype = _lib.MI_MXFP8 if self.bits == 8 else _lib.MI_MXFP4
        d.page_size, d.num_kv_heads, d.head_dim, d.max_pages = page_size, heads, self.head_dim, pages
        d.page_stride, d.kv_stride, d.token_stride, d.head_stride = codes.stride()[:4]
        d.k_scale = scales.data_ptr()
        d.v_scale = scales.data_ptr() + heads * scales.shape[3] * page_size

    @property
    def shape(self) -> torch.Size:
        """``[max_pages, 2, page_size, num_kv_heads, head_dim]``, as the shape of a KV layer tensor."""
        return torch.Size((*self.codes.shape[:4], self.head_dim))


class MXKVCache:
    """A pool of :class:`MXKVLayer`, indexed by layer.

    ``codes`` ``[num_layers, max_pages, 2, page_size, num_kv_heads, head_dim * bits // 8]`` and
    ``scales`` ``[num_layers, max_pages, 2, num_kv_heads, head_dim // 32, page_size]``, uint8,
    all zeros.
    """

    def __init__(self, num_layers: int, max_pages: int, page_size: int, num_kv_heads: int, head_dim: int,
                 bits: int = 8, device: torch.device | str = "cuda"):
        if bits not in (8, 4):
            raise ValueError(f"a microscaled cache holds 8 or 4 bits an element, not {bits}")
        if head_dim % MX_BLOCK or head_dim <= 0:
            raise ValueError(f"head_dim {head_dim} must be a multiple of {MX_BLOCK}")
        if page_size <= 0 or page_size % 16:
            raise ValueError(f"page_size {page_size} must be a positive multiple of 16")
        self.bits = bits
        self.codes = torch.zeros(num_layers, max_pages, 2, page_size, num_kv_heads, head_dim * bits // 8,
                                 dtype=torch.uint8, device=device)
        self.scales = torch.zeros(num_layers, max_pages, 2, num_kv_heads, head_dim // MX_BLOCK, page_size,
                                  dtype=torch.uint8, device=device)
        self._layers = [MXKVLayer(c, s) for c, s in zip(self.codes, self.scales)]

    def __getitem__(self, layer: int) -> MXKVLayer:
        return self._layers[layer]

    def __len__(self) -> int:
        return len(self._layers)

    @property
    def device(self) -> torch.device:
        return self.codes.device

    @property
    def is_cuda(self) -> bool:
        return self.codes.is_cuda


def _index(t: torch.Tensor, dev: torch.device) -> torch.Tensor:
    """A contiguous int32 vector on ``dev``."""
    if t.dim() != 1:
        raise ValueError("index tensors must have one dimension")
    return t if t.dtype is torch.int32 and t.device == dev and t.is_contiguous() else t.to(dev, torch.int32).contiguous()


def read_kv_cache(kv_cache_layer: torch.Tensor | MXKVLayer, kv_indptr: torch.Tensor, kv_indices: torch.Tensor,
                  last_page_len: torch.Tensor, total_tokens: int, dtype: torch.dtype = torch.bfloat16,
                  k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                  out: tuple[torch.Tensor, torch.Tensor] | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """K and V of a batch's whole contexts, ``[total_tokens, num_kv_heads, head_dim]`` each, requests one after the other.

    The index tensors are those a wrapper plans with (int32; CPU ones are copied to the
    layer's device).  ``total_tokens``, the sum of the requests' lengths, is the caller's
    knowledge (nothing is read back); rows beyond the batch's own are left as they were,
    and so are rows beyond ``total_tokens``.  Values come in ``dtype`` (bf16, fp16 or
    fp32), rounded to nearest; microscaled values past fp16's range are ±65504.  ``out``: contiguous tensors to write instead of new ones.
    Reads 16-bit, fp32, fp8 (with its per-head ``k_scale`` / ``v_scale``) and microscaled
    layers.
    """
    desc = _lib.paged_kv_desc(kv_cache_layer, k_scale, v_scale)
    dev = kv_cache_layer.device
    if dev.type != "cuda":
        raise ValueError("kv_cache_layer must be on a GPU")
    code = _OUT.get(dtype)
    if code is None:
        raise ValueError(f"dtype {dtype} is not bf16, fp16 or fp32")
    indptr, indices, last = _index(kv_indptr, dev), _index(kv_indices, dev), _index(last_page_len, dev)
    batch = indptr.shape[0] - 1
    if batch < 0 or last.shape[0] != batch:
        raise ValueError("index tensors disagree on the number of requests")
    if total_tokens < 0:
        raise ValueError(f"total_tokens {total_tokens} is negative")
    shape = (total_tokens, desc.num_kv_heads, desc.head_dim)
    if out is None:
        k, v = torch.empty(shape, dtype=dtype, device=dev), torch.empty(shape, dtype=dtype, device=dev)
    else:
        k, v = out
        for t in (k, v):
            if t.shape != shape or t.dtype != dtype or t.device != dev or not t.is_contiguous():
                raise ValueError(f"out must be contiguous {shape} tensors of {dtype} on {dev}")
    _lib.check(_lib.lib().mi_kv_read(desc, indptr.data_ptr(), indices.data_ptr(), last.data_ptr(), batch,
                                     indices.shape[0], k.data_ptr(), v.data_ptr(), code, total_tokens,
                                     _lib.stream_ptr(dev)), "mi_kv_read")
    return k, v
