"""Attention behind a sliding window with sinks, one request, in 64 bits, and how far a kernel may be off.

Query j of a request stands at position i = kv_len - qo_len + j and sees key t iff
t >= i - window_left or t < sinks (window_left < 0: all), and t <= i where causal.
"""

from __future__ import annotations

import torch


def visible(kv_len: int, qo_len: int, window_left: int, sinks: int, causal: bool) -> torch.Tensor:
    """``[qo_len, kv_len]``: which keys each query sees."""
    i = torch.arange(kv_len - qo_len, kv_len)[:, None]
    t = torch.arange(kv_len)[None]
    seen = torch.ones(qo_len, kv_len, dtype=torch.bool)
    if window_left >= 0:
        seen &= (t >= i - window_left) | (t < sinks)
    return seen & (t <= i) if causal else seen


def _product(w: torch.Tensor, v: torch.Tensor, seen: torch.Tensor) -> torch.Tensor:
    """sum_t w_jt v_t over the keys that row j sees; the others take no part, also where v is NaN or infinite."""
    if torch.isfinite(v).all():
        return w @ v  # w is zero elsewhere
    return torch.stack([w[j, see] @ v[see] for j, see in enumerate(seen)])


def attend(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, seen: torch.Tensor,
           out_eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    """(outputs, bound) of q ``[n, Hq, D]`` over k, v ``[kv_len, Hkv, D]``, both in 64 bits.

    Keys that a query does not see take no part, whatever they hold (the kernels
    keep to that but for V rows that are not finite: those may make NaN the elements they
    hold in rows that another row of their tile sees them for).  ``bound`` is
    how far from it a kernel with 32-bit sums and probabilities and outputs rounded
    to a type of half-step ``out_eps`` (``torch.finfo(t).eps / 2``) may be:

    * the output's own rounding, out_eps |o|;
    * every probability's rounding, out_eps each, in the sum with V and in the row
      sum: 2 out_eps A, A = sum_t w_t |v_t|;
    * fp16 probabilities below 2^-14 are off by up to 2^-25 where the largest of
      the row is at least 1: 2 * 2^-25 sum_t |v_t| (bf16 has fp32's range);
    * scores: a sum of D products in fp32 is off by at most (D + 2) 2^-24
      sum_d |q_d k_d| / sqrt(D) =: d, which changes every weight by a factor within
      1 +- 2 d: 4 d A with the normalisation; the exponential and the sums over
      keys and pieces in fp32 add less than 2^-16 A.
    """
    n, hq, dim = q.shape
    hkv = k.shape[1]
    out = torch.zeros(n, hq, dim, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for h in range(hq):
        kk, vv = k[:, h // (hq // hkv)].double(), v[:, h // (hq // hkv)].double()
        used = seen.any(0)
        kk, vv, see = kk[used], vv[used], seen[:, used]
        if see.shape[1] == 0:
            continue
        qq = q[:, h].double()
        s = (qq @ kk.T) * dim ** -0.5
        delta = (qq.abs() @ kk.abs().T) * dim ** -0.5 * (dim + 2) * 2.0 ** -24
        s = torch.where(see, s, -torch.inf)
        delta = torch.where(see, delta, 0.0).amax(-1, keepdim=True)
        rows = see.any(1)
        w = torch.zeros_like(s)
        w[rows] = torch.softmax(s[rows], -1)
        out[:, h] = _product(w, vv, see)
        a = _product(w, vv.abs(), see)
        small = 2.0 ** -24 * _product(see.double(), vv.abs(), see) if out_eps == torch.finfo(torch.float16).eps / 2 else 0.0
        bound[:, h] = out_eps * out[:, h].abs() + (2 * out_eps + 4 * delta + 2.0 ** -16) * a + small
    return out, bound
