"""Rotary position embedding on the packed batch (gfx950 kernels).

Mirrors the two ``flashinfer.rope`` calls M* makes from
``BatchedCacheManager.apply_rope`` (``mstar/engine/cache_manager.py:702-760``):
``apply_rope_pos_ids_inplace`` and ``apply_llama31_rope_pos_ids_inplace``, same
argument names and defaults.  q ``[tokens, Hq, D]`` and k ``[tokens, Hkv, D]``
(bf16 or fp16, last dim contiguous) are rotated in place by ``mi_rope_apply``;
there is no CPU fallback.  ``rope_append`` fuses the rotation with the paged
K/V append that follows it in ``run_attention`` (``mi_rope_append``).
``apply_qk_norm_rope_pos_ids_inplace`` and ``qk_norm_rope_append`` normalise q and k head
by head before the rotation, in the same pass (``mi_qk_norm_rope``).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

_DTYPES = {torch.bfloat16: _lib.MI_BF16, torch.float16: _lib.MI_F16}
_POS = {torch.int32: _lib.MI_I32, torch.int64: _lib.MI_I64}


def _check(x: torch.Tensor, name: str) -> None:
    if x.dim() != 3:
        raise ValueError(f"{name} must be [tokens, heads, head_dim], got {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{name}: RoPE runs on bf16 or fp16 tensors, got {x.dtype}")
    if x.device.type != "cuda":
        raise ValueError(f"{name} must be a GPU tensor")
    if x.stride(2) != 1:
        raise ValueError(f"{name}: head_dim must be contiguous")


def _apply(q, k, pos_ids, rotary_dim, interleave, rope_scale, rope_theta, llama31, low, high, old) -> None:
    _check(q, "q")
    _check(k, "k")
    if q.dtype != k.dtype or q.shape[0] != k.shape[0] or q.shape[2] != k.shape[2] or q.device != k.device:
        raise ValueError("q and k must agree on dtype, device, token count and head_dim")
    d = q.shape[2]
    rd = d if rotary_dim is None else int(rotary_dim)
    if rd <= 0 or rd > d or rd % 8 or d % 8:
        raise ValueError(f"rotary_dim {rd} and head_dim {d} must be multiples of 8 with rotary_dim <= head_dim")
    if pos_ids.dtype not in _POS or pos_ids.dim() != 1 or pos_ids.shape[0] < q.shape[0]:
        raise ValueError("pos_ids must be an int32/int64 vector with one position per token")
    pos_ids = pos_ids.to(q.device).contiguous()
    _lib.check(
        _lib.lib().mi_rope_apply(
            q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], k.data_ptr(), k.stride(0), k.stride(1), k.shape[1],
            _DTYPES[q.dtype], d, rd, pos_ids.data_ptr(), _POS[pos_ids.dtype], q.shape[0], 1 if interleave else 0,
            float(rope_scale), float(rope_theta), 1 if llama31 else 0, float(low), float(high), float(old),
            _lib.stream_ptr(q.device),
        ),
        "mi_rope_apply",
    )


def apply_rope_pos_ids_inplace(q: torch.Tensor, k: torch.Tensor, pos_ids: torch.Tensor,
                               rotary_dim: int | None = None, interleave: bool = False,
                               rope_scale: float = 1, rope_theta: float = 1e4) -> None:
    """Rotate q and k in place at the given positions (flashinfer.rope semantics)."""
    _apply(q, k, pos_ids, rotary_dim, interleave, rope_scale, rope_theta, False, 1.0, 4.0, 8192.0)


def apply_llama31_rope_pos_ids_inplace(q: torch.Tensor, k: torch.Tensor, pos_ids: torch.Tensor,
                                       rotary_dim: int | None = None, interleave: bool = False,
                                       rope_scale: float = 8, rope_theta: float = 5e5,
                                       low_freq_factor: float = 1, high_freq_factor: float = 4,
                                       old_context_len: int = 8192) -> None:
    """Llama-3.1 frequency-smoothed RoPE in place (flashinfer.rope semantics)."""
    _apply(q, k, pos_ids, rotary_dim, interleave, rope_scale, rope_theta, True, low_freq_factor,
           high_freq_factor, old_context_len)


def rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, kv_cache_layer: torch.Tensor,
                pos_ids: torch.Tensor, page_idx: torch.Tensor, slot_idx_ptr: int, idx_stride: int,
                num_append: int, num_append_device_ptr: int | None, *, rotary_dim: int | None = None,
                interleave: bool = False, rope_scale: float = 1, rope_theta: float = 1e4,
                k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None, keep_k: bool = True,
                llama31: dict | None = None) -> None:
    """Rotate q (and k) in place and write the rotated k and v to the paged cache, in one launch.

    The result equals ``apply_rope_pos_ids_inplace`` (or the Llama-3.1 variant
    when ``llama31`` holds its factors) followed by the wrapper's
    ``set_kv_cache`` on the same page map: token ``t < num_append`` (and below
    the device count at ``num_append_device_ptr`` when given) goes to page
    ``page_idx[t * idx_stride]``, slot ``slot_idx[t * idx_stride]``.  With
    ``keep_k=False`` the rotated k only reaches the cache and ``k`` keeps its
    input values.
    """
    _check(q, "q")
    _check(k, "k")
    _check(v, "v")
    if q.dtype != k.dtype or v.dtype != k.dtype:
        raise ValueError("q, k and v must share one dtype")
    if q.shape[0] != k.shape[0] or v.shape != k.shape or q.shape[2] != k.shape[2]:
        raise ValueError(f"shapes q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} do not agree")
    desc = _lib.paged_kv_desc(kv_cache_layer, k_scale, v_scale)
    if k.shape[1:] != (desc.num_kv_heads, desc.head_dim):
        raise ValueError(f"k/v shape {tuple(k.shape)} does not match the cache heads/head_dim")
    if num_append > k.shape[0]:
        raise ValueError(f"k/v hold {k.shape[0]} tokens, {num_append} planned")
    for name, x in (("k", k), ("v", v)):
        if x.stride(0) % 8 or x.stride(1) % 8 or x.data_ptr() % 16:
            raise ValueError(f"{name}: rows must be 16-byte aligned")
    d = q.shape[2]
    rd = d if rotary_dim is None else int(rotary_dim)
    if rd <= 0 or rd > d or rd % 8 or d % 8:
        raise ValueError(f"rotary_dim {rd} and head_dim {d} must be multiples of 8 with rotary_dim <= head_dim")
    if pos_ids.dtype not in _POS or pos_ids.dim() != 1 or pos_ids.shape[0] < q.shape[0]:
        raise ValueError("pos_ids must be an int32/int64 vector with one position per token")
    pos_ids = pos_ids.to(q.device).contiguous()
    l31 = llama31 or {}
    _lib.check(
        _lib.lib().mi_rope_append(
            q.data_ptr(), q.stride(0), q.stride(1), q.shape[1], k.data_ptr(), k.stride(0), k.stride(1),
            v.data_ptr(), v.stride(0), v.stride(1), _DTYPES[q.dtype], 1 if keep_k else 0, desc,
            page_idx.data_ptr(), slot_idx_ptr, idx_stride, num_append, num_append_device_ptr, rd,
            pos_ids.data_ptr(), _POS[pos_ids.dtype], q.shape[0], 1 if interleave else 0, float(rope_scale),
            float(rope_theta), 1 if llama31 else 0, float(l31.get("low_freq_factor", 1.0)),
            float(l31.get("high_freq_factor", 4.0)), float(l31.get("old_context_len", 8192.0)),
            _lib.stream_ptr(q.device),
        ),
        "mi_rope_append",
    )


def _norm_weight(w: torch.Tensor, name: str, dtype: torch.dtype, d: int, at: int) -> int:
    """The type code of a norm's weight; refuses what the kernel does not read."""
    if w.shape != (d,) or not w.is_contiguous():
        raise ValueError(f"{name} must be a contiguous vector of head_dim {d} elements, got {tuple(w.shape)}")
    wd = w.dtype
    if wd is not dtype and wd is not torch.float32:
        raise ValueError(f"{name} must be {dtype} or float32, got {wd}")
    if w.get_device() != at:
        raise ValueError(f"{name} must be on cuda:{at}, not on {w.device}")
    return _DTYPES.get(wd, _lib.MI_F32)


def _norm_rows(x: torch.Tensor, name: str) -> tuple[torch.Size, int, int, int]:
    """(shape, address, token stride, head stride) of q, k or v, in rows that the kernel reads."""
    shape = x.shape
    if len(shape) != 3 or x.dtype not in _DTYPES or not x.is_cuda:
        _check(x, name)
    (st, sh, sd), ptr = x.stride(), x.data_ptr()
    if sd != 1:
        _check(x, name)
    if (st | sh) % 8 or ptr % 16:
        raise ValueError(f"{name}: rows must be 16-byte aligned")
    return shape, ptr, st, sh


def _qk_norm_rope(q, k, v, q_weight, k_weight, pos_ids, eps, rotary_dim, interleave, rope_scale, rope_theta, llama31, keep_k,
                  layer=None, k_scale=None, v_scale=None, page_idx=None, slot_at=None, idx_stride=0, n_append=0, n_device_at=None):
    # in a decode step the launch is over before these checks are: each attribute is read once
    (n, hq, d), q_at, q_st, q_sh = _norm_rows(q, "q")
    (n_k, hkv, d_k), k_at, k_st, k_sh = _norm_rows(k, "k")
    dtype, at = q.dtype, q.get_device()
    if k.dtype is not dtype or n_k != n or d_k != d or k.get_device() != at:
        raise ValueError("q and k must agree on dtype, device, token count and head_dim")
    v_at = v_st = v_sh = desc_at = page_at = 0
    if page_idx is not None:
        v_shape, v_at, v_st, v_sh = _norm_rows(v, "v")
        if v.dtype is not dtype or v_shape != (n, hkv, d) or v.get_device() != at:
            raise ValueError(f"v {tuple(v_shape)}, {v.dtype} does not agree with k {tuple(k.shape)}, {k.dtype}")
        desc = _lib.paged_kv_desc(layer, k_scale, v_scale)
        if layer.device != k.device:
            raise ValueError(f"kv_cache_layer must be on {k.device}, not on {layer.device}")
        if desc.num_kv_heads != hkv or desc.head_dim != d:
            raise ValueError(f"k/v shape {tuple(k.shape)} does not match the cache heads/head_dim")
        if n_append > n:
            raise ValueError(f"k/v hold {n} tokens, {n_append} planned")
        desc_at, page_at = ctypes.addressof(desc), page_idx.data_ptr()
    rd = d if rotary_dim is None else int(rotary_dim)
    least = 8 if interleave else 16
    if rd <= 0 or rd > d or rd % least or d % 8 or d > 512:
        raise ValueError(f"rotary_dim {rd} must be a multiple of {least} and head_dim {d} one of 8 up to 512, rotary_dim <= head_dim")
    wd = _norm_weight(q_weight, "q_weight", dtype, d, at)
    if _norm_weight(k_weight, "k_weight", dtype, d, at) != wd:
        raise ValueError("q_weight and k_weight must share one dtype")
    if not eps >= 0:
        raise ValueError(f"eps {eps} must not be negative")
    pos_type, pos_shape = _POS.get(pos_ids.dtype), pos_ids.shape
    if pos_type is None or len(pos_shape) != 1 or pos_shape[0] < n:
        raise ValueError("pos_ids must be an int32/int64 vector with one position per token")
    if pos_ids.get_device() != at or not pos_ids.is_contiguous():
        pos_ids = pos_ids.to(q.device).contiguous()
    smooth, low, high, old = 0, 1.0, 4.0, 8192.0
    if llama31:
        smooth = 1
        low, high = llama31.get("low_freq_factor", low), llama31.get("high_freq_factor", high)
        old = llama31.get("old_context_len", old)
    status = _lib.lib().mi_qk_norm_rope_block(_lib.QK_NORM_ROPE_ARGS.pack(
        q_at, k_at, v_at, q_weight.data_ptr(), k_weight.data_ptr(), pos_ids.data_ptr(), desc_at, page_at, slot_at or 0,
        n_device_at or 0, _lib.stream_at(at), q_st, q_sh, k_st, k_sh, v_st, v_sh, idx_stride, hq, hkv, _DTYPES[dtype], d, wd,
        1 if keep_k else 0, n_append, rd, pos_type, n, 1 if interleave else 0, smooth, eps, rope_scale, rope_theta, low, high, old))
    if status:
        _lib.check(status, "mi_qk_norm_rope")


def apply_qk_norm_rope_pos_ids_inplace(q: torch.Tensor, k: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                                       pos_ids: torch.Tensor, eps: float = 1e-6, rotary_dim: int | None = None,
                                       interleave: bool = False, rope_scale: float = 1, rope_theta: float = 1e4,
                                       llama31: dict | None = None) -> None:
    """Normalise every head's row of q and k, then rotate it, in place and in one pass.

    A row x becomes ``x * rsqrt(mean(x^2) + eps) * weight`` (``q_weight``, ``k_weight``: ``[head_dim]``, in q's dtype
    or fp32), rotated as :func:`apply_rope_pos_ids_inplace` rotates (with ``llama31``'s factors as
    :func:`apply_llama31_rope_pos_ids_inplace`, ``rope_scale`` given).  fp32 throughout, rounded once; angles are formed in 64
    bits, so far positions turn more exactly than in the calls without a norm.
    """
    _qk_norm_rope(q, k, None, q_weight, k_weight, pos_ids, eps, rotary_dim, interleave, rope_scale, rope_theta, llama31, True)


def qk_norm_rope_append(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor, k_weight: torch.Tensor,
                        kv_cache_layer, pos_ids: torch.Tensor, page_idx: torch.Tensor, slot_idx_ptr: int, idx_stride: int,
                        num_append: int, num_append_device_ptr: int | None, *, eps: float = 1e-6,
                        rotary_dim: int | None = None, interleave: bool = False, rope_scale: float = 1,
                        rope_theta: float = 1e4, k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                        keep_k: bool = True, llama31: dict | None = None) -> None:
    """:func:`apply_qk_norm_rope_pos_ids_inplace`, and k and v to the paged cache, in one launch.

    Page map and ``keep_k`` as in :func:`rope_append`; any cache type, microscaled layers among them.  k is rounded
    once, from fp32 to the cache's type.
    """
    if page_idx is None:
        raise ValueError("page_idx must be a tensor of page ids")
    _qk_norm_rope(q, k, v, q_weight, k_weight, pos_ids, eps, rotary_dim, interleave, rope_scale, rope_theta, llama31, keep_k,
                  kv_cache_layer, k_scale, v_scale, page_idx, slot_idx_ptr, idx_stride, num_append, num_append_device_ptr)


def rope_positions(qo_indptr: torch.Tensor, position_id_start: torch.Tensor, out: torch.Tensor,
                   num_tokens: int) -> torch.Tensor:
    """``out[t] = position_id_start[r] + t - qo_indptr[r]`` for t < num_tokens (int64, on the GPU)."""
    batch = position_id_start.shape[0]
    if qo_indptr.dtype != torch.int32 or position_id_start.dtype != torch.int32 or out.dtype != torch.int64:
        raise ValueError("qo_indptr/position_id_start must be int32 and out int64")
    if out.shape[0] < num_tokens or qo_indptr.shape[0] != batch + 1:
        raise ValueError("rope_positions: inconsistent sizes")
    _lib.check(
        _lib.lib().mi_rope_positions(qo_indptr.data_ptr(), position_id_start.data_ptr(), batch, out.data_ptr(),
                                     num_tokens, _lib.stream_ptr(out.device)),
        "mi_rope_positions",
    )
    return out
