"""GPU: requests so long that the product of their tiles and their pieces passes 2^31.

The page list names few pages again and again, and five pages of keys that the queries
favour once each, spread over the request's pieces: a piece that is left out, read twice or read from
elsewhere moves every output.  The reference counts how often each (page, slot) is seen and
is exact in 64 bits.
"""

import numpy as np
import pytest
import torch

from gpu_helpers import log, workspace
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper

pytestmark = pytest.mark.gpu

PS, PLAIN = 1024, 3


def _inputs(gpu, keys, hq, d, rows, seed):
    """(layer, values, q, page list): one kv-head."""
    g = torch.Generator().manual_seed(seed)
    pages = -(-keys // PS)
    u = torch.randn(d, generator=g)
    u /= u.norm()
    # logits of the favoured keys: their 1024 weigh about as much as a sixth of all the others
    a = (np.log(pages / 6) * d ** 0.5) ** 0.5
    kv = torch.randn(PLAIN + 5, 2, PS, 1, d, generator=g)
    kv[PLAIN:, 0] = a * u + 0.1 * kv[PLAIN:, 0]
    kv[PLAIN:, 1] += 50 * torch.tensor([1.0, -2.0, 3.0, -4.0, 5.0]).view(5, 1, 1, 1)
    q = (a * u + 0.3 * torch.randn(rows, hq, d, generator=g)).to(torch.bfloat16)
    kv = kv.to(torch.bfloat16)
    indices = np.arange(pages, dtype=np.int32) % PLAIN
    indices[[pages // 50, pages // 3, pages // 2, pages - pages // 5, pages - 2]] = PLAIN + np.arange(5)
    return kv.to(gpu), kv.double(), q, indices


def _reference(values, q, indices, keys, window_left, sinks, steps):
    """(outputs, bound) of queries at the end of the request, causal."""
    n, hq, d = q.shape
    k, v = values[:, 0, :, 0].flatten(0, 1), values[:, 1, :, 0].flatten(0, 1)
    pool = len(values)

    def count(a, b):  # how often keys [a, b) of the request are each (page, slot)
        c = np.zeros((pool, PS))
        for page, lo, hi in ((a // PS, a % PS, PS), (b // PS, 0, b % PS)) if a // PS < b // PS else ((a // PS, a % PS, b % PS),):
            if lo < hi:
                c[indices[page], lo:hi] += 1
        if a // PS < b // PS:
            c += np.bincount(indices[a // PS + 1:b // PS], minlength=pool)[:, None]
        return torch.from_numpy(c.reshape(-1))

    out, bound = torch.empty(n, hq, d, dtype=torch.float64), torch.empty(n, hq, d, dtype=torch.float64)
    for j in range(n):
        at = keys - n + j
        first = max(0, at - window_left) if window_left >= 0 else 0
        c = count(first, at + 1) + (count(0, min(sinks, first)) if min(sinks, first) else 0)
        s = q[j].double() @ k.T * d ** -0.5
        delta = (q[j].double().abs() @ k.abs().T * d ** -0.5).amax(-1, keepdim=True) * (d + 2) * 2.0 ** -24
        w = c * torch.exp(s - s.amax(-1, keepdim=True))
        w /= w.sum(-1, keepdim=True)
        out[j] = w @ v
        # as oracle/window.py: output, probabilities, scores; and a wavefront's sums in 32 bits, the row sum's and the
        # products', to which `steps` groups of four keys are added one after the other: steps 2^-24 of the magnitudes each
        eps = torch.finfo(torch.bfloat16).eps / 2
        bound[j] = eps * out[j].abs() + (2 * eps + 4 * delta + 2.0 ** -16 + 2 * steps * 2.0 ** -24) * (w @ v.abs())
    return out, bound


@pytest.mark.parametrize("window_left,sinks", [(1 << 30, 0), (70_000_001, 5)])
def test_decode(gpu, window_left, sinks):
    """One request at one kv-head: 512 items of its 4.5 million tiles."""
    keys, hq, d = 72_000_777, 8, 64
    layer, values, q, indices = _inputs(gpu, keys, hq, d, 1, seed=1)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, 1, d, PS, device=gpu)
    w.plan(torch.tensor([0, len(indices)], dtype=torch.int32), torch.from_numpy(indices),
           torch.tensor([keys - (len(indices) - 1) * PS], dtype=torch.int32))
    out = w.run(q.to(gpu), layer, window_left=window_left, sink_tokens=sinks).double().cpu()
    ref, bound = _reference(values, q, indices, keys, window_left, sinks, steps=keys // (512 * 4) // 4 + 32)
    log(f"decode of {keys} keys: {((out - ref).abs() / bound).max():.3f} of the bound")
    assert ((out - ref).abs() <= bound).all()


@pytest.mark.parametrize("d,new", [(64, 20), (256, 10)])
@pytest.mark.parametrize("window_left,sinks", [(1 << 30, 0), (590_000_001, 5), (-1, 0)])
def test_chunk(gpu, d, new, window_left, sinks):
    """One tile of rows, which the plan cuts into more than a hundred pieces of its 18.75 million steps."""
    keys, hq = 600_000_777, 8
    layer, values, q, indices = _inputs(gpu, keys, hq, d, new, seed=d)
    w = PagedPrefillWrapper(workspace(gpu, 256 << 20), hq, 1, d, PS, device=gpu)
    w.plan(torch.tensor([0, new], dtype=torch.int32), torch.tensor([0, len(indices)], dtype=torch.int32),
           torch.from_numpy(indices), torch.tensor([keys - (len(indices) - 1) * PS], dtype=torch.int32))
    pieces = int(w._workspace[:32].cpu().view(torch.int32)[2])
    assert pieces * -(-keys // 32) > 2**31, f"{pieces} pieces: the products stay in 32 bits"
    out = w.run(q.to(gpu), layer, window_left=window_left, sink_tokens=sinks).double().cpu()
    ref, bound = _reference(values, q, indices, keys, window_left, sinks, steps=keys // pieces // 4 + 64)
    log(f"chunk over {keys} keys in {pieces} pieces: {((out - ref).abs() / bound).max():.3f} of the bound")
    assert ((out - ref).abs() <= bound).all()
