"""GPU: what microscaled codes are read as, over every code and scale, and blocks that are hard to quantise.

* every (code, scale byte) pair of both formats, in every output type of the read;
* ties between codes and the limits of a block's scale, at every head_dim, each of them counted;
* magnitudes at the top of fp16's range, whose nearest codes lie past it: read back and attended
  to in fp16 as its largest value, by every kernel.
"""

import pytest
import torch

import mx_helpers as H
from gpu_helpers import log, workspace
from mstar_amd.mx_cache import MXKVCache, MXKVLayer, read_kv_cache
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper
from oracle import microscaled as M

pytestmark = pytest.mark.gpu

F16_TOP = 65504.0


def _as(values: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """64-bit values in dtype, rounded once, finite ones past fp16's range as its largest.  Code values have at most four
    significant bits and exponents from -136, so fp32 holds them exactly wherever it does not overflow."""
    if dtype == torch.float16:
        values = values.clamp(-F16_TOP, F16_TOP)
    return values.float().to(dtype)


def _same(got: torch.Tensor, want: torch.Tensor) -> bool:
    a, b = got.cpu(), want
    return torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(nan=0.0, posinf=1e38, neginf=-1e38),
                                                             b.nan_to_num(nan=0.0, posinf=1e38, neginf=-1e38))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("bits", [8, 4])
def test_every_code_under_every_scale(gpu, bits, dtype):
    """Token s holds every code in blocks of scale byte s; K in this order, V in the opposite one."""
    n, d = 256, 256
    codes = torch.arange(256, dtype=torch.uint8)
    if bits == 4:  # 256 bytes of two codes each
        codes = M.unpack(codes, 4)
    width = codes.numel() // d
    c = codes.view(width, d).expand(n, width, d)  # heads x head_dim hold all of them
    s = torch.arange(256, dtype=torch.uint8).view(n, 1, 1).expand(n, width, d // 32)
    kv = torch.stack([c, c.flip(2)]), torch.stack([s, s.flip(0)])
    rows = M.pack(kv[0].contiguous(), bits).view(2, n // 16, 16, width, -1).permute(1, 0, 2, 3, 4).contiguous()
    scales = kv[1].reshape(2, n // 16, 16, width, d // 32).permute(1, 0, 3, 4, 2).contiguous()
    layer = MXKVLayer(rows.to(gpu), scales.to(gpu))
    idx = torch.tensor([0, n // 16], dtype=torch.int32), torch.arange(n // 16, dtype=torch.int32), torch.tensor([16], dtype=torch.int32)
    got = read_kv_cache(layer, *idx, n, dtype)
    for which, x in enumerate(got):
        assert _same(x, _as(M.values(kv[0][which], kv[1][which], bits), dtype)), ("K", "V")[which]


def _ties(bits: int) -> torch.Tensor:
    """Every code's value, every midpoint between two and the block's limits, of both signs, in 64 bits."""
    grid, lim = (M.E4M3[:127] if bits == 8 else M.E2M1[:8]), M.LIMIT[bits]
    t = torch.cat([grid, (grid[1:] + grid[:-1]) / 2, torch.tensor([lim, lim * (1 + 2 ** -7), lim * (1 - 2 ** -7)], dtype=torch.float64)])
    return torch.cat([t, -t])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 4])
def test_append_ties_and_limits(gpu, bits, d, dtype):
    """Each value beside the largest code, so that its block's scale is 1, and the same blocks 2^-9 as large."""
    ties = _ties(bits)
    ties = ties.to(dtype).double().unique()  # what the source type holds of them
    per = 31 * (2 * d // 32)
    n = -(-len(ties) // per)
    flat = torch.zeros(n * per, dtype=torch.float64)
    flat[: len(ties)] = ties
    x = torch.empty(n * 2 * d // 32, 32, dtype=torch.float64)
    x[:, 0] = M.LIMIT[bits] - (16 if bits == 8 else 1)  # the largest code: 448, 6
    x[:, 1:] = flat.view(-1, 31)
    x = torch.cat([x, x * 2.0 ** -9]).view(2 * n, 2, d)
    k = x.to(dtype)
    assert (k.double() == x)[:n].all()
    assert set(ties.tolist()) <= set(k[:n].double().flatten().tolist()), "a value is not among the rows"
    v = k.flip(0).contiguous()
    tokens, pages = 2 * n, -(-2 * n // 16)
    layer = MXKVCache(1, pages, 16, 2, d, bits=bits, device=gpu)[0]
    idx = torch.tensor([0, pages], dtype=torch.int32), torch.arange(pages, dtype=torch.int32), \
        torch.tensor([tokens - (pages - 1) * 16], dtype=torch.int32)
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), 4, 2, d, 16, device=gpu)
    w.plan(torch.tensor([0, tokens], dtype=torch.int32), *idx)
    w.set_kv_cache(layer, k.to(gpu), v.to(gpu))
    rows, scales = layer.codes.cpu(), layer.scales.cpu()
    for which, src in enumerate((k, v)):
        c, s = M.quantize(src, bits)
        got_c = rows[:, which].flatten(0, 1)[:tokens]
        got_s = scales[:, which].permute(0, 3, 1, 2).flatten(0, 1)[:tokens]
        assert torch.equal(got_s, s), "scale bytes differ"
        a, b = M.unpack(got_c, bits), c
        bad = (a != b).nonzero()
        assert len(bad) == 0, f"{len(bad)} codes differ: {src[tuple(bad[0])]} gives {a[tuple(bad[0])]}, not {b[tuple(bad[0])]}"


TOP = {8: (63488.0, 63500.0, 65504.0, 61440.0), 4: (57344.0, 57500.0, 60000.0, 65504.0)}


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 4])
def test_fp16_values_at_the_top_of_their_range(gpu, bits, d):
    """Appended from fp16 and read back in fp16: finite, what the codes stand for or fp16's largest."""
    n = 20
    k = torch.randn(n, 2, d, generator=torch.Generator().manual_seed(d)).to(torch.float16)
    for i, t in enumerate(TOP[bits]):
        k[i::4, :, i] = t
        k[i::4, :, d - 1 - i] = -t
    v = -k.flip(0)
    layer = MXKVCache(1, 2, 16, 2, d, bits=bits, device=gpu)[0]
    idx = torch.tensor([0, 2], dtype=torch.int32), torch.tensor([1, 0], dtype=torch.int32), torch.tensor([4], dtype=torch.int32)
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), 4, 2, d, 16, device=gpu)
    w.plan(torch.tensor([0, n], dtype=torch.int32), *idx, dtype=torch.float16)
    w.set_kv_cache(layer, k.to(gpu), v.to(gpu))
    past = 0
    for got, src in zip(read_kv_cache(layer, *idx, n, torch.float16), (k, v)):
        ref = M.values(*M.quantize(src, bits), bits)
        past += int((ref.abs() > F16_TOP).sum())
        assert torch.isfinite(got).all()
        assert torch.equal(got.cpu(), _as(ref, torch.float16))
    assert past > 0, "no value's code lies past the range"


CHUNKS = [(1, 1), (1, 700), (3, 50), (40, 40), (129, 400), (300, 2500)]


@pytest.mark.parametrize("kw", [{}, {"window_left": 150, "sink_tokens": 21}])
@pytest.mark.parametrize("kind", ["mx8_f16", "mx4_f16"])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 1, 256), (16, 4, 64)])
def test_fp16_attention_past_the_range(gpu, hq, hkv, d, kind, kw):
    """K and V of up to 10^5 under fp16 queries: what is past the range takes part as 65504."""
    wl, sinks = kw.get("window_left", -1), kw.get("sink_tokens", 0)
    g = torch.Generator().manual_seed(d)
    for new, lens in (tuple(zip(*CHUNKS)), ((1,) * 6, (1, 17, 300, 511, 1025, 3001)), ((1,) * 80, (260,) * 80)):
        p = H.make(gpu, kind, lens, 16, hkv, d, seed=d, spread=2e4)
        assert (p.values.abs() > F16_TOP).any()
        p.values.clamp_(-F16_TOP, F16_TOP)
        q = (torch.randn(sum(new), hq, d, generator=g) * 1e-4).to(torch.float16)
        if max(new) == 1:
            w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, 16, device=gpu)
            w.plan(*p.index(), dtype=torch.float16)
        else:
            w = PagedPrefillWrapper(workspace(gpu, 128 << 20), hq, hkv, d, 16, device=gpu)
            w.plan(torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32), *p.index(), dtype=torch.float16)
        share = H.check(p, q, new, w.run(q.to(gpu), p.layer, **kw), wl, sinks, True, kind)
        log(f"{kind} {len(lens)} requests: {share:.2f} of the bound")
