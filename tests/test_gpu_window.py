"""GPU: attention behind a sliding window with sinks, against 64 bits (oracle/window.py).

Every cache format, head layouts, windows and sinks that end inside tiles and pages,
contexts from none to several thousand keys, single queries, short and long chunks, with
and without causal.  Keys that the window hides hold NaN, and pages that it hides whole
are replaced by a page of NaN, so whatever reads them shows.
"""

import pytest
import torch

import mx_helpers as H
from gpu_helpers import log, workspace
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper

pytestmark = pytest.mark.gpu

HEADS = [(8, 2, 128), (28, 4, 128), (8, 1, 256), (16, 4, 64), (16, 1, 64), (3, 3, 128)]
WINDOWS = [(0, 0), (1, 0), (15, 1), (16, 4), (30, 16), (100, 40), (63, 100), (1023, 4), (5000, 7)]
LENS = [1, 2, 15, 16, 17, 33, 100, 0, 511, 1025, 3001]


def _decode(gpu, p, hq, hkv, d, dtype, seed, wl, sinks, **kw):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(len(p.lens), hq, d, generator=g).to(dtype)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, p.ps, device=gpu)
    w.plan(*p.index(), dtype=dtype)
    out = w.run(q.to(gpu), p.layer, *p.scales, window_left=wl, sink_tokens=sinks, **kw)
    torch.cuda.synchronize()
    return q, out


@pytest.mark.parametrize("wl,sinks", WINDOWS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_decode_windows(gpu, hq, hkv, d, wl, sinks):
    p = H.make(gpu, "bf16", LENS, 16, hkv, d, seed=wl + d)
    H.hide(p, [1] * len(LENS), wl, sinks)
    q, out = _decode(gpu, p, hq, hkv, d, torch.bfloat16, 1, wl, sinks)
    log(f"{H.check(p, q, [1] * len(LENS), out, wl, sinks, True, 'decode'):.2f} of the bound")


@pytest.mark.parametrize("ps", [16, 48, 128])
@pytest.mark.parametrize("kind", sorted(H.KINDS))
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 1, 256), (16, 4, 64)])
def test_decode_formats(gpu, hq, hkv, d, kind, ps):
    p = H.make(gpu, kind, LENS, ps, hkv, d, seed=ps + d)
    for wl, sinks in ((200, 20), (40, 0)):
        H.hide(p, [1] * len(LENS), 200, 20)
        q, out = _decode(gpu, p, hq, hkv, d, H.KINDS[kind], 2, wl, sinks)
        H.check(p, q, [1] * len(LENS), out, wl, sinks, True, kind)


def test_decode_one_request_split(gpu):
    """One request: its window is cut into items whose partials are merged; a small workspace leaves fewer."""
    p = H.make(gpu, "bf16", [9000], 16, 2, 128, seed=3)
    H.hide(p, [1], 4095, 4)
    for ws in (64 << 20, 1 << 20, 200 << 10):
        q = torch.randn(1, 16, 128, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
        w = PagedDecodeWrapper(workspace(gpu, ws), 16, 2, 128, 16, device=gpu)
        w.plan(*p.index())
        out = w.run(q.to(gpu), p.layer, window_left=4095, sink_tokens=4)
        H.check(p, q, [1], out, 4095, 4, True, f"workspace {ws}")


def test_window_beyond_context_is_full_attention(gpu):
    """A window longer than every context sees what the run without one sees."""
    p = H.make(gpu, "bf16", LENS, 16, 2, 128, seed=5)
    for wl in (4000, 2 ** 31 - 1, 2 ** 40):
        q, out = _decode(gpu, p, 8, 2, 128, torch.bfloat16, 6, wl, 0)
        H.check(p, q, [1] * len(LENS), out, -1, 0, True, f"window {wl}")
    q, out = _decode(gpu, p, 8, 2, 128, torch.bfloat16, 6, -1, 2 ** 40)
    H.check(p, q, [1] * len(LENS), out, -1, 0, True, "no window")
    q, out = _decode(gpu, p, 8, 2, 128, torch.bfloat16, 6, 3, 2 ** 40)
    H.check(p, q, [1] * len(LENS), out, -1, 0, True, "all sinks")


CHUNKS = [(1, 1), (1, 700), (2, 2), (3, 50), (40, 40), (129, 400), (300, 2500), (0, 30), (517, 517), (5, 1000)]


def _prefill(gpu, p, hq, hkv, d, dtype, new, seed, wl, sinks, causal, ws=128 << 20):
    g = torch.Generator().manual_seed(seed)
    q = torch.randn(sum(new), hq, d, generator=g).to(dtype)
    qo = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    w = PagedPrefillWrapper(workspace(gpu, ws), hq, hkv, d, p.ps, device=gpu)
    w.plan(qo, *p.index(), causal=causal, dtype=dtype)
    out = w.run(q.to(gpu), p.layer, *p.scales, window_left=wl, sink_tokens=sinks)
    torch.cuda.synchronize()
    return q, out


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("wl,sinks", WINDOWS)
@pytest.mark.parametrize("hq,hkv,d", HEADS)
def test_chunk_windows(gpu, hq, hkv, d, wl, sinks, causal):
    new, lens = zip(*CHUNKS)
    p = H.make(gpu, "bf16", lens, 16, hkv, d, seed=wl + d)
    H.hide(p, new, wl, sinks)
    q, out = _prefill(gpu, p, hq, hkv, d, torch.bfloat16, new, 7, wl, sinks, causal)
    log(f"{H.check(p, q, new, out, wl, sinks, causal, 'chunk'):.2f} of the bound")


@pytest.mark.parametrize("ps", [16, 48, 128])
@pytest.mark.parametrize("kind", sorted(H.KINDS))
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (8, 1, 256), (16, 4, 64)])
def test_chunk_formats(gpu, hq, hkv, d, kind, ps):
    new, lens = zip(*CHUNKS)
    p = H.make(gpu, kind, lens, ps, hkv, d, seed=ps + d)
    H.hide(p, new, 150, 21)
    q, out = _prefill(gpu, p, hq, hkv, d, H.KINDS[kind], new, 8, 150, 21, True)
    H.check(p, q, new, out, 150, 21, True, kind)


@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (8, 1, 256), (16, 4, 64)])
@pytest.mark.parametrize("wl", [600, 2000, 70000])
def test_chunk_cut_tiles(gpu, hq, hkv, d, wl):
    """Few tiles over a long context: the plan cuts them into pieces, the window leaves some of those without work."""
    new, lens = [300, 40], [6000, 2600]
    p = H.make(gpu, "bf16", lens, 16, hkv, d, seed=9)
    for ws in (128 << 20, 24 << 20):
        q, out = _prefill(gpu, p, hq, hkv, d, torch.bfloat16, new, 10, wl, 5, True, ws)
        H.check(p, q, new, out, wl, 5, True, f"workspace {ws}")


def test_many_requests_paired_plan(gpu):
    """From 128 requests on a plan pairs kv-heads, which halves the rows of its short requests: windowed runs follow it."""
    lens = [(37 * i) % 300 + 12 for i in range(140)]
    new = [(1, 2, 3, 12)[i % 4] for i in range(140)]
    p = H.make(gpu, "bf16", lens, 16, 2, 128, seed=11)
    H.hide(p, new, 64, 2)
    q, out = _prefill(gpu, p, 8, 2, 128, torch.bfloat16, new, 12, 64, 2, True)
    H.check(p, q, new, out, 64, 2, True, "paired plan")
    p = H.make(gpu, "bf16", lens, 16, 2, 128, seed=11)
    H.hide(p, [1] * 140, 64, 2)
    q, out = _decode(gpu, p, 8, 2, 128, torch.bfloat16, 13, 64, 2)
    H.check(p, q, [1] * 140, out, 64, 2, True, "paired decode plan")


def test_one_plan_for_windowed_and_full_layers(gpu):
    """Layers with and without a window in turn over one plan; each run equals itself bit for bit."""
    new, lens = zip(*CHUNKS)
    p = H.make(gpu, "bf16", lens, 16, 4, 128, seed=14)
    q = torch.randn(sum(new), 28, 128, generator=torch.Generator().manual_seed(15)).to(torch.bfloat16)
    qo = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    w = PagedPrefillWrapper(workspace(gpu, 128 << 20), 28, 4, 128, 16, device=gpu)
    w.plan(qo, *p.index())
    runs = [w.run(q.to(gpu), p.layer, **({} if i % 2 else {"window_left": 50, "sink_tokens": 3})) for i in range(6)]
    torch.cuda.synchronize()
    H.check(p, q, new, runs[0], 50, 3, True, "windowed")
    H.check(p, q, new, runs[1], -1, 0, True, "full")
    for i in range(2, 6):
        assert torch.equal(runs[i], runs[i % 2])


def test_refusals(gpu):
    p = H.make(gpu, "bf16", [40], 16, 2, 128, seed=16)
    w = PagedDecodeWrapper(workspace(gpu, 32 << 20), 8, 2, 128, 16, device=gpu)
    w.plan(*p.index())
    q = torch.randn(1, 8, 128, device=gpu, dtype=torch.bfloat16)
    for kw in ({"window_left": -2}, {"window_left": 3, "sink_tokens": -1}, {"sink_tokens": -1}):
        with pytest.raises(ValueError):
            w.run(q, p.layer, **kw)
    w.plan(*p.index(), dtype=torch.float32)
    with pytest.raises(ValueError):
        w.run(q.float(), p.layer.float(), window_left=3)
