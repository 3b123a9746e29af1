"""GPU: the microscaled KV cache against its definition in 64 bits (oracle/microscaled.py).

What an append writes is compared byte for byte, what a read gives value for value: blocks
of every magnitude the source types hold, ties and the largest codes, zeros, subnormals,
NaN and infinities; strided sources; tokens that are skipped; contexts of no token, one,
part of a page; every cache format and output type of the read.  Attention over the cache
without a window is compared like the windowed runs (tests/test_gpu_window.py).
"""

import pytest
import torch

import mx_helpers as H
from gpu_helpers import log, workspace
from mstar_amd import _lib
from mstar_amd.mx_cache import MXKVCache, read_kv_cache
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper
from oracle import microscaled as M

pytestmark = pytest.mark.gpu


def _edge_rows(bits: int, dtype: torch.dtype, d: int, seed: int) -> torch.Tensor:
    """[tokens, heads, d] of blocks that are hard to quantise."""
    g = torch.Generator().manual_seed(seed)
    info = torch.finfo(dtype)
    lim = M.LIMIT[bits]
    rows = [torch.randn(8, d, generator=g)]
    for e in (-140, -130, -127, -120, -60, -20, -3, 0, 5, 12, 60, 110, 118, 120):  # magnitudes across the type's range
        rows.append(torch.randn(2, d, generator=g).double() * 2.0 ** e)
    grid = (M.E4M3[:127] if bits == 8 else M.E2M1[:8])
    ties = torch.cat([grid, (grid[1:] + grid[:-1]) / 2, torch.tensor([lim, lim * (1 + 2 ** -7), lim * (1 - 2 ** -7)])])
    ties = torch.cat([ties, -ties])
    t = torch.zeros(-(-len(ties) // 31) * 32, dtype=torch.float64)  # each block beside the largest code: its scale stays 1
    t.view(-1, 32)[:, 0] = grid[-1]
    flat = t.view(-1, 32)[:, 1:]
    idx = torch.arange(flat.numel())
    flat.copy_(ties[idx % len(ties)].view(flat.shape))
    n = t.numel() // d * d
    rows += [t[:n].view(-1, d), t[:n].view(-1, d) * 2.0 ** -9]
    z = torch.zeros(6, d, dtype=torch.float64)
    z[0, 3] = 1.0  # alone in its block, the others zero
    z[1, :32] = -0.0
    z[2, 5], z[2, 40] = float("nan"), 1.5
    z[3, 33] = float("inf")
    z[4, 0], z[4, 1] = float("-inf"), 7.0
    z[5] = float(info.max)
    z[5, ::2] *= -1
    rows.append(z)
    x = torch.cat([r.double() for r in rows])
    x = torch.where(x.abs() > info.max, x.sign() * float("inf"), x) if dtype == torch.float16 else x
    x = x.to(dtype)
    if x.shape[0] % 2:
        x = x[:-1]
    return x.view(-1, 2, d)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("bits", [8, 4])
def test_append_is_the_definition(gpu, bits, d, dtype):
    k = _edge_rows(bits, dtype, d, seed=d + bits)
    v = k.flip(0).contiguous()
    n, ps = k.shape[0], 16
    pages = -(-n // ps)
    cache = MXKVCache(2, pages + 3, ps, 2, d, bits=bits, device=gpu)
    cache.codes.fill_(0x11)
    cache.scales.fill_(0x22)
    perm = torch.randperm(pages + 3, generator=torch.Generator().manual_seed(1))[:pages].int()
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), 4, 2, d, ps, device=gpu)
    w.plan(torch.tensor([0, n], dtype=torch.int32), torch.tensor([0, pages], dtype=torch.int32), perm,
           torch.tensor([n - (pages - 1) * ps], dtype=torch.int32))
    w.set_kv_cache(cache[1], k.to(gpu), v.to(gpu))
    want_c, want_s = cache.codes[1].clone().cpu().fill_(0x11), cache.scales[1].clone().cpu().fill_(0x22)
    for i in range(n):
        page, slot = int(perm[i // ps]), i % ps
        for which, x in enumerate((k, v)):
            c, s = M.quantize(x[i], bits)
            want_c[page, which, slot] = M.pack(c, bits)
            want_s[page, which, :, :, slot] = s
    got_s, got_c = cache.scales[1].cpu(), cache.codes[1].cpu()
    assert torch.equal(got_s, want_s), "scale bytes differ"
    a, b = M.unpack(got_c, bits), M.unpack(want_c, bits)
    bad = (a != b).nonzero()
    assert len(bad) == 0, f"{len(bad)} codes differ, first at {bad[0].tolist()}: {a[tuple(bad[0])]} for {b[tuple(bad[0])]}"
    assert (cache.codes[0] == 0x11).all() and (cache.scales[0] == 0x22).all(), "another layer was written"
    # and back: every value, the last block of tokens included
    kk, vv = read_kv_cache(cache[1], *_one(n, pages, perm, ps), n, dtype=torch.float32)
    for got, x in ((kk, k), (vv, v)):
        c, s = M.quantize(x, bits)
        ref = M.values(c, s, bits)
        assert torch.equal(torch.nan_to_num(got.cpu().double(), nan=-1e300), torch.nan_to_num(ref, nan=-1e300))


def _one(n, pages, perm, ps):
    return torch.tensor([0, pages], dtype=torch.int32), perm, torch.tensor([n - (pages - 1) * ps], dtype=torch.int32)


@pytest.mark.parametrize("bits", [8, 4])
def test_append_strided_and_skipped(gpu, bits):
    """k and v as views of a fused projection; tokens with pages or slots out of range, and those past the device's
    count, are skipped."""
    ps, h, d, n = 16, 3, 128, 21
    qkv = torch.randn(n, 8 * d + 2 * h * d, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16).to(gpu)
    k, v = (qkv[:, 8 * d + i * h * d: 8 * d + (i + 1) * h * d].view(n, h, d) for i in (0, 1))
    layer = MXKVCache(1, 4, ps, h, d, bits=bits, device=gpu)[0]
    page = torch.tensor([(0, 3, 1, -1, 4, 2)[i % 6] for i in range(n)], dtype=torch.long)
    slot = torch.tensor([(i * 5) % 17 for i in range(n)], dtype=torch.long)
    count = torch.tensor([18], dtype=torch.int32, device=gpu)
    pg, sl = page.to(gpu), slot.to(gpu)
    _lib.check(_lib.lib().mi_kv_append(layer.desc, k.data_ptr(), v.data_ptr(), _lib.MI_BF16, k.stride(0), k.stride(1),
                                       v.stride(0), v.stride(1), pg.data_ptr(), sl.data_ptr(), 1, n, count.data_ptr(),
                                       _lib.stream_ptr(gpu)), "mi_kv_append")
    wc, ws = torch.zeros_like(layer.codes).cpu(), torch.zeros_like(layer.scales).cpu()
    for i in range(18):
        if 0 <= page[i] < 4 and slot[i] < ps:
            for which, x in enumerate((k, v)):
                c, s = M.quantize(x[i].cpu(), bits)
                wc[page[i], which, slot[i]] = M.pack(c, bits)
                ws[page[i], which, :, :, slot[i]] = s
    assert torch.equal(layer.scales.cpu(), ws)
    assert torch.equal(layer.codes.cpu(), wc)


LENS = [33, 0, 1, 16, 200, 0, 0, 47, 130, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("kind", ["bf16", "f16", "fp8", "mx8", "mx4", "f32"])
@pytest.mark.parametrize("ps,h,d", [(16, 2, 128), (48, 1, 256), (64, 5, 64)])
def test_read_contexts(gpu, ps, h, d, kind, dtype):
    p = H.make(gpu, "bf16" if kind == "f32" else kind, LENS, ps, h, d, seed=ps + d)
    if kind == "f32":
        p.layer = torch.randn(p.values.shape, generator=torch.Generator().manual_seed(3)).to(gpu)
        p.values = p.layer.cpu().double()
    total, extra = sum(LENS), 3
    for index in (p.index(), tuple(t.to(gpu) for t in p.index())):
        k = torch.full((total + extra, h, d), 7.0, dtype=dtype, device=gpu)
        v = torch.full_like(k, 8.0)
        got = read_kv_cache(p.layer, *index, total + extra, dtype, *p.scales, out=(k, v))
        assert got[0] is k and got[1] is v
        for which, x in enumerate((k, v)):
            ref = torch.cat([p.rows(r, which) for r in range(len(LENS))])
            # fp8: the product with the scale is rounded to fp32 before the output's type
            want = (ref.float() if kind == "fp8" else ref).to(dtype)
            assert torch.equal(x[:total].cpu(), want), (which, (x[:total].cpu().double() - ref).abs().max())
            assert (x[total:] == 7.0 + which).all(), "rows behind the last sequence were written"
    # fewer rows than the batch has: the rest is not written
    k, v = read_kv_cache(p.layer, *p.index(), 40, dtype, *p.scales)
    ref = torch.cat([p.rows(r, 0) for r in range(len(LENS))])[:40]
    assert torch.equal(k.cpu(), (ref.float() if kind == "fp8" else ref).to(dtype))


def test_read_long_list_and_empty(gpu):
    """More pages than the launch has workgroups, many requests; and batches without any token."""
    lens = [(i * 7919) % 97 for i in range(1500)]
    p = H.make(gpu, "mx4", lens, 16, 1, 64, seed=4)
    assert len(p.kv_indices) > 2048
    k, v = read_kv_cache(p.layer, *p.index(), sum(lens), torch.float32)
    for which, x in enumerate((k, v)):
        assert torch.equal(x.cpu().double(), torch.cat([p.rows(r, which) for r in range(len(lens))]))
    zero, none = torch.zeros(1, dtype=torch.int32), torch.empty(0, dtype=torch.int32)
    assert read_kv_cache(p.layer, zero, none, none, 0)[0].shape == (0, 1, 64)
    assert read_kv_cache(p.layer, torch.zeros(3, dtype=torch.int32), none, torch.ones(2, dtype=torch.int32), 0)[1].numel() == 0


CHUNKS = [(1, 1), (1, 700), (3, 50), (40, 40), (129, 400), (300, 2500), (0, 30), (517, 517)]


@pytest.mark.parametrize("kind", ["mx8", "mx4", "mx8_f16", "mx4_f16"])
@pytest.mark.parametrize("hq,hkv,d,ps", [(8, 2, 128, 16), (28, 4, 128, 64), (8, 1, 256, 16), (16, 4, 64, 48), (16, 1, 64, 16)])
def test_attention(gpu, hq, hkv, d, ps, kind):
    """Decode and chunks over the cache without a window; slots past the end hold NaN."""
    new, lens = zip(*CHUNKS)
    p = H.make(gpu, kind, lens, ps, hkv, d, seed=ps + d)
    H.hide(p, new, 1 << 20, 0)
    dt = H.KINDS[kind]
    q = torch.randn(sum(new), hq, d, generator=torch.Generator().manual_seed(5)).to(dt)
    qo = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    for causal in (True, False):
        w = PagedPrefillWrapper(workspace(gpu, 128 << 20), hq, hkv, d, ps, device=gpu)
        w.plan(qo, *p.index(), causal=causal, dtype=dt)
        H.check(p, q, new, w.run(q.to(gpu), p.layer), -1, 0, causal, "chunk")
    lens = [1, 2, 15, 16, 17, 33, 0, 511, 1025, 3001] + [20] * 4
    p = H.make(gpu, kind, lens, ps, hkv, d, seed=ps + d)
    H.hide(p, [1] * len(lens), 1 << 20, 0)
    q = torch.randn(len(lens), hq, d, generator=torch.Generator().manual_seed(6)).to(dt)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu)
    w.plan(*p.index(), dtype=dt)
    H.check(p, q, [1] * len(lens), w.run(q.to(gpu), p.layer), -1, 0, True, "decode")


@pytest.mark.parametrize("kind", ["mx8", "mx4"])
def test_decode_full_batch(gpu, kind):
    """At 128 requests the plan pairs kv-heads; these caches take the per-head kernels on it."""
    lens = [(53 * i) % 700 + 1 for i in range(140)]
    p = H.make(gpu, kind, lens, 16, 4, 128, seed=7)
    q = torch.randn(140, 32, 128, generator=torch.Generator().manual_seed(8)).to(torch.bfloat16)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), 32, 4, 128, 16, device=gpu)
    w.plan(*p.index())
    log(f"{H.check(p, q, [1] * 140, w.run(q.to(gpu), p.layer), -1, 0, True, kind):.2f} of the bound")


def test_nan_block_reaches_its_rows_only(gpu):
    """A NaN appended to one head's K makes that head's rows NaN and no others."""
    cache = MXKVCache(1, 8, 16, 2, 128, bits=4, device=gpu)
    k = torch.randn(40, 2, 128, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    v = torch.randn(40, 2, 128, generator=torch.Generator().manual_seed(10)).to(torch.bfloat16)
    k[11, 1, 70] = float("nan")
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), 8, 2, 128, 16, device=gpu)
    w.plan(torch.tensor([0, 40], dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32),
           torch.tensor([5, 1, 3], dtype=torch.int32), torch.tensor([8], dtype=torch.int32))
    w.set_kv_cache(cache[0], k.to(gpu), v.to(gpu))
    q = torch.randn(40, 8, 128, generator=torch.Generator().manual_seed(11)).to(torch.bfloat16).to(gpu)
    out = w.run(q, cache[0]).cpu()
    assert torch.isfinite(out[:, :4]).all() and torch.isfinite(out[:11]).all()
    assert torch.isnan(out[11:, 4:]).all()
    out = w.run(q, cache[0], window_left=4).cpu()  # behind the window nothing of it is left
    assert torch.isnan(out[11:16, 4:]).all() and torch.isfinite(out[16:]).all() and torch.isfinite(out[:, :4]).all()


def test_refusals(gpu):
    cache = MXKVCache(1, 4, 16, 2, 128, device=gpu)
    w = PagedDecodeWrapper(workspace(gpu, 32 << 20), 8, 2, 128, 16, device=gpu)
    one = torch.ones(2, device=gpu)
    w.plan(torch.tensor([0, 1], dtype=torch.int32), torch.tensor([2], dtype=torch.int32), torch.tensor([5], dtype=torch.int32))
    q, k = torch.zeros(1, 8, 128, dtype=torch.bfloat16, device=gpu), torch.zeros(1, 2, 128, dtype=torch.bfloat16, device=gpu)
    with pytest.raises(ValueError):
        w.run(q, cache[0], one, one)
    with pytest.raises(ValueError):
        w.set_kv_cache(cache[0], k, k, one, one)
    with pytest.raises(ValueError):
        w.run(q, MXKVCache(1, 4, 16, 2, 64, device=gpu)[0])
    with pytest.raises(ValueError):
        w.set_kv_cache(cache[0], k[:, :1], k[:, :1])
    w.plan(torch.tensor([0, 1], dtype=torch.int32), torch.tensor([2], dtype=torch.int32), torch.tensor([5], dtype=torch.int32),
           dtype=torch.float32)
    with pytest.raises(RuntimeError):
        w.run(q.float(), cache[0])
    with pytest.raises(ValueError):
        read_kv_cache(cache[0], torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                      torch.ones(1, dtype=torch.int32), 16, dtype=torch.float64)
    with pytest.raises(ValueError):
        read_kv_cache(cache[0], torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                      torch.ones(3, dtype=torch.int32), 16)
    with pytest.raises(ValueError):
        read_kv_cache(cache[0], torch.zeros(2, dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
                      torch.ones(1, dtype=torch.int32), 16, out=(q[0], q[0]))
