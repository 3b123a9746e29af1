"""Paged caches of every format for the window and microscaled tests: a pool on the GPU beside the 64-bit values it holds."""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

from mstar_amd.mx_cache import MXKVLayer
from oracle import microscaled as M
from oracle import window as W

KINDS = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.bfloat16, "mx8": torch.bfloat16, "mx4": torch.bfloat16,
         "fp8_f16": torch.float16, "mx8_f16": torch.float16, "mx4_f16": torch.float16}  # -> q's type


@dataclass
class Paged:
    kind: str
    layer: object          # tensor or MXKVLayer on the GPU
    scales: tuple          # k_scale, v_scale of an fp8 layer
    values: torch.Tensor   # float64 [pool, 2, ps, hkv, d] on the CPU
    kv_indptr: np.ndarray
    kv_indices: np.ndarray
    last: np.ndarray
    lens: list
    ps: int

    def rows(self, r: int, which: int) -> torch.Tensor:
        pages = torch.as_tensor(self.kv_indices[self.kv_indptr[r]:self.kv_indptr[r + 1]]).long()
        return self.values[pages, which].flatten(0, 1)[: self.lens[r]]

    def index(self):
        return tuple(torch.as_tensor(x) for x in (self.kv_indptr, self.kv_indices, self.last))


def poison_layer(layer, page: int, slots, nan_bytes: bool = True) -> None:
    """NaN in K and V of a page's slots, in the layer's own format."""
    if isinstance(layer, MXKVLayer):
        layer.scales[page][:, :, :, slots] = 255
        layer.codes[page][:, slots] = 0x77
    elif layer.dtype == torch.float8_e4m3fn:
        layer.view(torch.uint8)[page][:, slots] = 0x7F
    else:
        layer[page][:, slots] = float("nan")


def make(gpu, kind: str, lens, ps: int, hkv: int, d: int, seed: int, spread: float = 1.0) -> Paged:
    g = torch.Generator().manual_seed(seed)
    lens = [int(x) for x in lens]
    npages = [-(-n // ps) for n in lens]
    pool = sum(npages) + 5
    perm = torch.randperm(pool, generator=g).numpy().astype(np.int32)
    indptr = np.concatenate([[0], np.cumsum(npages)]).astype(np.int32)
    last = np.array([n - (p - 1) * ps if p else ps for n, p in zip(lens, npages)], dtype=np.int32)
    x = torch.randn(pool, 2, ps, hkv, d, generator=g) * spread
    scales = (None, None)
    base = kind.split("_")[0]
    if base in ("mx8", "mx4"):
        bits = int(base[2])
        codes, sc = M.quantize(x, bits)
        values = M.values(codes, sc, bits)
        layer = MXKVLayer(M.pack(codes, bits).to(gpu), sc.permute(0, 1, 3, 4, 2).contiguous().to(gpu))
    elif base == "fp8":
        ks, vs = torch.rand(hkv, generator=g) * 0.01 + 0.01, torch.rand(hkv, generator=g) * 0.01 + 0.01
        both = torch.stack([ks, vs]).view(1, 2, 1, hkv, 1)
        q8 = (x / both).clamp(-448, 448).to(torch.float8_e4m3fn)
        layer, values, scales = q8.to(gpu), q8.double() * both.double(), (ks.to(gpu), vs.to(gpu))
    else:
        q16 = x.to(KINDS[kind])
        layer, values = q16.to(gpu), q16.double()
    return Paged(kind, layer, scales, values, indptr, perm[: indptr[-1]].copy(), last, lens, ps)


def check(p: Paged, q: torch.Tensor, new, out: torch.Tensor, window_left: int, sinks: int, causal: bool, what="") -> float:
    """Every row of out against 64 bits; returns the largest share of the bound."""
    worst, at = 0.0, 0
    o = out.double().cpu()
    for r, n in enumerate(new):
        if n == 0:
            continue
        if p.lens[r] == 0:
            assert (o[at:at + n] == 0).all(), f"{what} request {r}: a request without keys gives zeros"
            at += n
            continue
        seen = W.visible(p.lens[r], n, window_left, sinks, causal)
        ref, bound = W.attend(q[at:at + n], p.rows(r, 0), p.rows(r, 1), seen, torch.finfo(out.dtype).eps / 2)
        err = (o[at:at + n] - ref).abs()
        assert torch.isfinite(o[at:at + n]).all(), f"{what} request {r} ({p.lens[r]} keys): not finite"
        share = (err / (bound + 1e-30)).max().item()
        assert share <= 1, f"{what} request {r} ({p.lens[r]} keys, {n} queries): {share:.2f} of the bound"
        worst = max(worst, share)
        at += n
    return worst


def hide(p: Paged, new, window_left: int, sinks: int) -> None:
    """NaN wherever every query's window hides a key, and past each request's end; pages hidden whole become one
    page of NaN."""
    free = [i for i in range(p.values.shape[0]) if i not in set(p.kv_indices.tolist())]
    poison_layer(p.layer, free[0], slice(None))
    for r, n in enumerate(new):
        if p.lens[r] == 0:
            continue
        lo = p.lens[r] - max(n, 1) - window_left
        for e in range(p.kv_indptr[r], p.kv_indptr[r + 1]):
            first = (e - p.kv_indptr[r]) * p.ps
            bad = [s for s in range(p.ps) if (sinks <= first + s < lo) or first + s >= p.lens[r]]
            if len(bad) == p.ps:
                p.kv_indices[e] = free[0]
            elif bad:
                poison_layer(p.layer, int(p.kv_indices[e]), bad)
