"""Attention weights of cached tokens and eviction by them, in 64 bits and by the definitions."""

from __future__ import annotations

import numpy as np
import torch


def probabilities(q: torch.Tensor, k: torch.Tensor, seen: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """One request: (weights, bound) ``[keys, kv_heads]`` of q ``[n, Hq, D]`` over k ``[keys, Hkv, D]``; ``seen`` ``[n, keys]``.

    The sum over queries and the q heads of a kv head of their softmax probabilities.  ``bound``: a score is a sum of D products
    in fp32, off by at most (D + 4) 2^-24 sum_d |q_d k_d| / sqrt(D) =: e (its scaling included), an exponential by that of the
    score and of the row's log-sum-exp (at most the row's largest e), the rounding of their difference in the log2 domain
    and two units of the function's: p (2 e + (|s| + |lse| + 4) 2^-23); sums in fp32 are at most keys / 16 + 32 and rows + 32
    additions after one another: p (keys / 16 + rows + 64) 2^-24.
    """
    n, hq, dim = q.shape
    keys, hkv = k.shape[0], k.shape[1]
    g = hq // hkv
    out = torch.zeros(keys, hkv, dtype=torch.float64)
    bound = torch.zeros_like(out)
    for h in range(hkv):
        kk = k[:, h].double()
        for j in range(h * g, (h + 1) * g):
            qq = q[:, j].double()
            s = qq @ kk.T * dim ** -0.5
            e = (qq.abs() @ kk.abs().T) * dim ** -0.5 * (dim + 4) * 2.0 ** -24
            s = torch.where(seen, s, -torch.inf)
            rows = seen.any(-1)
            if not rows.any():
                continue
            s, e, see = s[rows], e[rows], seen[rows]
            lse = torch.logsumexp(s, -1, keepdim=True)
            p = torch.exp(s - lse)
            worst = torch.where(see, e, 0.0).amax(-1, keepdim=True)
            size = torch.where(see, s.abs(), 0.0) + lse.abs()
            out[:, h] += p.sum(0)
            bound[:, h] += (p * (2 * worst + (size + 4) * 2.0 ** -23 + (keys / 16 + n * g + 64) * 2.0 ** -24)).sum(0)
    return out, bound


def kept_places(weights: np.ndarray, keep: int, recent: int, sinks: int) -> np.ndarray:
    """The places of one (request, head) that stay, ascending: weights ``[length]``, NaN below every number."""
    n = len(weights)
    if n <= keep:
        return np.arange(n)
    middle = sorted(range(sinks, n - recent), key=lambda t: (np.isnan(weights[t]), -weights[t] if weights[t] == weights[t] else 0.0, t))
    return np.array(sorted([*range(sinks), *range(n - recent, n), *middle[: keep - sinks - recent]]), dtype=np.int64)
