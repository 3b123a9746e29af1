"""GPU: NaN and infinities in keys that some rows of a tile see and others do not.

* K: only rows that see the key are touched, whatever its bits.
* V: rows that see the key get what 64 bits give.  Of the rows that do not, those of a tile
  (or of a short request) that reaches the key may get NaN in the elements that are not finite, and in
  no others; rows of tiles that do not reach it, of other kv-heads and of other requests
  get nothing.  Runs of single tokens have one position a request: nothing hidden reaches them.
"""

import pytest
import torch

import mx_helpers as H
from gpu_helpers import workspace
from mstar_amd.mx_cache import MXKVLayer
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper
from oracle import window as W

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 128), (8, 1, 256), (16, 4, 64)]
STEP = 32  # keys that a tile takes at a time


def _poison(p: H.Paged, r: int, token: int, head: int, which: int, value: float) -> list:
    """value in K (0) or V (1) of a key, in the layer and in its values; the elements that hold it."""
    page, slot = int(p.kv_indices[p.kv_indptr[r] + token // p.ps]), token % p.ps
    if isinstance(p.layer, MXKVLayer):  # a block of NaN
        p.layer.scales[page, which, head, 1, slot] = 255
        elements = list(range(32, 64))
        p.values[page, which, slot, head, 32:64] = float("nan")
    else:
        elements = [37]
        p.layer[page, which, slot, head, 37] = value
        p.values[page, which, slot, head, 37] = value
    return elements


def _check(p, q, new, out, wl, sinks, at, which, elements, reached):
    """at: (request, token, head) of the key; reached(j): its tile reaches the key, for a row that does not see it."""
    o, first = out.double().cpu(), 0
    group = q.shape[1] // p.values.shape[3]
    for r, n in enumerate(new):
        seen = W.visible(p.lens[r], n, wl, sinks, True)
        ref, bound = W.attend(q[first:first + n], p.rows(r, 0), p.rows(r, 1), seen, torch.finfo(out.dtype).eps / 2)
        got = o[first:first + n]
        first += n
        may = torch.zeros_like(ref, dtype=torch.bool)  # elements that may be NaN though the reference is finite
        if r == at[0] and which == 1:
            for j in range(n):
                if not seen[j, at[1]] and reached(j):
                    may[j, at[2] * group:(at[2] + 1) * group, elements] = True
        fin = torch.isfinite(ref)
        if r == at[0]:
            assert not fin.all(), "no row sees the key"
        assert not torch.isfinite(got[~fin]).any(), f"request {r}: a row that sees the key is finite"
        ok = ((got - ref).abs() <= bound) | ~fin
        assert (ok | may).all(), f"request {r}: {(~(ok | may)).nonzero()[:4].tolist()}"
        assert (ok | got.isnan()).all(), f"request {r}: neither right nor NaN"


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("kind", ["bf16", "f16", "mx8", "mx4"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_chunks(gpu, hq, hkv, d, kind, which, value):
    """A chunk of several tiles and a short request, poisoned in turn at a key whose windows end inside a tile."""
    new, lens, wl, sinks, group = [330, 3], [520, 90], 40, 3, hq // hkv
    tile = (128 if d == 256 else 256) // group  # tokens of a tile
    for at in ((0, 190 + tile + 17, hkv - 1), (1, 90 - 3 - 40, 0)):
        p = H.make(gpu, kind, lens, 16, hkv, d, seed=d)
        q = torch.randn(sum(new), hq, d, generator=torch.Generator().manual_seed(1)).to(H.KINDS[kind])
        elements = _poison(p, *at, which, value)
        w = PagedPrefillWrapper(workspace(gpu, 64 << 20), hq, hkv, d, 16, device=gpu)
        w.plan(torch.tensor([0, 330, 333], dtype=torch.int32), *p.index(), dtype=H.KINDS[kind])

        def reached(j):
            if at[0] == 1:
                return True
            a = j // tile * tile  # the tile's first row; keys from its window to its last row's step
            last = lens[0] - new[0] + min(a + tile, new[0]) - 1
            return lens[0] - new[0] + a - wl <= at[1] < (last // STEP + 1) * STEP

        assert not all(reached(j) for j in range(330)) or at[0] == 1
        out = w.run(q.to(gpu), p.layer, window_left=wl, sink_tokens=sinks)
        _check(p, q, new, out, wl, sinks, at, which, elements, reached)


@pytest.mark.parametrize("kind", ["bf16", "f16", "mx8", "mx4"])
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_single_tokens(gpu, hq, hkv, d, kind):
    """NaN in K and V of the last hidden key and of the first behind the sinks: nothing of it arrives."""
    lens, wl, sinks = [300, 45, 1025, 2000], 30, 3
    p = H.make(gpu, kind, lens, 16, hkv, d, seed=d)
    for r, n in enumerate(lens):
        for token in (sinks, n - 1 - wl - 1):
            for which in (0, 1):
                _poison(p, r, token, hkv - 1, which, float("nan"))
    q = torch.randn(4, hq, d, generator=torch.Generator().manual_seed(2)).to(H.KINDS[kind])
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, 16, device=gpu)
    w.plan(*p.index(), dtype=H.KINDS[kind])
    H.check(p, q, [1] * 4, w.run(q.to(gpu), p.layer, window_left=wl, sink_tokens=sinks), wl, sinks, True, kind)
