"""GPU: windowed and microscaled runs as a serving program issues them.

Captured and replayed with other lengths, through the cache manager with rotation, append
and snapshots, on other streams than their plan's, side by side, from strided queries and
other cache layouts, over large batches, over pools whose offsets pass 32 bits, and without
a workspace.  Values are compared with 64 bits as in tests/test_gpu_window.py.
"""

import ctypes
import math

import numpy as np
import pytest
import torch

import mx_helpers as H
from gpu_helpers import custom_batch, log, workspace
from mstar_amd import _lib
from mstar_amd.cache_manager import BatchedCacheManager, WorkspaceBufferManager
from mstar_amd.kv_store import KVCacheConfig, PagedAllocationManager
from mstar_amd.mx_cache import MXKVCache, MXKVLayer, read_kv_cache
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper
from mstar_amd.rope import apply_rope_pos_ids_inplace
from oracle import microscaled as M
from oracle import window as W

pytestmark = pytest.mark.gpu


def _index(lens, ps, pool, seed, new=None):
    qo, indptr, indices, last = custom_batch(lens, ps, pool, seed, new_lens=new)
    return tuple(torch.as_tensor(x) for x in (qo, indptr, indices, last))


@pytest.mark.parametrize("bits", [8, 4])
def test_captured_decode(gpu, bits):
    """append + windowed and full runs captured once, replayed for other lengths and values: each replay equals the eager calls."""
    b, hq, hkv, d, ps, pool = 6, 16, 4, 128, 16, 700
    g = torch.Generator().manual_seed(1)
    cache = MXKVCache(1, pool, ps, hkv, d, bits=bits, device=gpu)
    eager_cache = MXKVCache(1, pool, ps, hkv, d, bits=bits, device=gpu)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, batch_size=b, max_num_pages=pool, device=gpu,
                           use_cuda_graph=True)
    e = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu)
    q = torch.zeros(b, hq, d, dtype=torch.bfloat16, device=gpu)
    k, v = (torch.zeros(b, hkv, d, dtype=torch.bfloat16, device=gpu) for _ in range(2))

    def step(wrapper, layer):
        wrapper.set_kv_cache(layer, k, v)
        return wrapper.run(q, layer, window_left=200, sink_tokens=5), wrapper.run(q, layer)

    _, *idx = _index([900] * b, ps, pool, 2)
    w.plan(*idx)
    step(w, cache[0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(w, cache[0])
    base = torch.randint(0, 256, cache.codes.shape, dtype=torch.uint8, generator=g)
    if bits == 8:
        base[(base & 127) == 127] = 0
    for c in (cache, eager_cache):
        c.codes.copy_(base)
        c.scales.fill_(125)
    for i, lens in enumerate(([1] * b, [17, 900, 300, 16, 211, 5], [205, 206, 207, 1000, 2, 33], [1800, 1, 1, 1, 1, 1])):
        for t in (q, k, v):
            t.copy_(torch.randn(t.shape, generator=g).to(t.dtype))
        _, *idx = _index(lens, ps, pool, 3 + i)
        w.plan(*idx)
        graph.replay()
        e.plan(*idx)
        want = step(e, eager_cache[0])
        torch.cuda.synchronize()
        assert torch.equal(cache.codes, eager_cache.codes) and torch.equal(cache.scales, eager_cache.scales)
        for a, o in zip(outs, want):
            assert torch.isfinite(a).all() and torch.equal(a, o), lens


def test_captured_chunks_with_padding(gpu):
    """A captured windowed run over a ragged batch replayed with fewer tokens and empty requests; rows behind stay."""
    b, hq, hkv, d, ps, pool, most = 4, 28, 4, 128, 16, 900, 600
    p = H.make(gpu, "bf16", [1], ps, hkv, d, seed=1)  # for its helpers
    g = torch.Generator().manual_seed(5)
    values = torch.randn(pool, 2, ps, hkv, d, generator=g).to(torch.bfloat16)
    layer = values.to(gpu)
    w = PagedPrefillWrapper(workspace(gpu, 128 << 20), hq, hkv, d, ps, batch_size=b, max_total_tokens=most,
                            max_num_pages=pool, device=gpu, use_cuda_graph=True)
    q = torch.zeros(most, hq, d, dtype=torch.bfloat16, device=gpu)
    out = torch.empty(most, hq, d, dtype=torch.bfloat16, device=gpu)
    qo, *idx = _index([300] * b, ps, pool, 2, new=[150] * b)
    w.plan(qo, *idx)
    w.run(q, layer, out=out, window_left=90, sink_tokens=3)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.run(q, layer, out=out, window_left=90, sink_tokens=3)
    for i, (lens, new) in enumerate((([700, 40, 300, 90], [300, 1, 120, 2]), ([64, 2000, 0, 0], [64, 3, 0, 0]),
                                     ([500, 500, 500, 500], [150, 150, 150, 150]), ([9, 0, 0, 0], [9, 0, 0, 0]))):
        q.copy_(torch.randn(q.shape, generator=g).to(q.dtype))
        qo, *idx = _index(lens, ps, pool, 20 + i, new=new)
        w.plan(qo, *idx)
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        p.values, p.lens = values.double(), lens
        p.kv_indptr, p.kv_indices, p.last = (t.numpy() for t in idx)
        H.check(p, q.cpu(), new, out, 90, 3, True, f"replay {i}")
        assert (out[sum(new):] == 3.0).all(), "rows behind the last sequence were written"


@pytest.mark.parametrize("bits", [8, 4])
def test_manager_steps(gpu, bits):
    """Chunks, then decode steps, through BatchedCacheManager over an MXKVCache: rotation, append, a full and a windowed layer;
    every output against 64 bits over the quantised rotated history, then a snapshot continued on another label."""
    hq, hkv, d, ps, layers = 16, 4, 128, 16, 2
    cfg = KVCacheConfig(num_layers=layers, num_kv_heads=hkv, head_dim=d, max_seq_len=2048, max_num_pages=300, page_size=ps,
                        num_qo_heads=hq)
    kv = MXKVCache(layers, 300, ps, hkv, d, bits=bits, device=gpu)
    mgr = PagedAllocationManager(cfg, kv)
    bufs = WorkspaceBufferManager(64 << 20, gpu)
    rids = [f"r{i}" for i in range(4)]
    for r in rids:
        mgr.add_request(r, ["main"])
    hist = {(r, l): [torch.empty(0, hkv, d, dtype=torch.float64)] * 2 for r in rids for l in range(layers)}
    g = torch.Generator().manual_seed(0)
    label = "main"
    for step, new in enumerate([[70, 1, 200, 16], [1] * 4, [1] * 4, [3, 40, 1, 17], [1] * 4]):
        cm = BatchedCacheManager(rids, {r: label for r in rids}, kv, mgr, bufs, cfg, gpu)
        cm.plan_attention(new)
        cm.plan_rope(new)
        n = sum(new)
        for layer in range(layers):
            q = torch.randn(n, hq, d, generator=g).to(torch.bfloat16)
            k, v = (torch.randn(n, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2))
            wl, sinks = ((-1, 0), (30, 3))[layer]
            qr, kr = q.to(gpu), k.to(gpu)
            pos = torch.cat([torch.arange(len(hist[r, layer][0]), len(hist[r, layer][0]) + m) for r, m in zip(rids, new)]).to(gpu)
            apply_rope_pos_ids_inplace(qr, kr, pos, rope_theta=1e5)
            kg = k.to(gpu)
            out = cm.apply_rope_and_run_attention(q.to(gpu), kg, v.to(gpu), rope_theta=1e5, layer_idx=layer, keep_k=False,
                                                  window_left=wl, sink_tokens=sinks)
            assert torch.equal(kg.cpu(), k), "keep_k=False changed k"
            at = 0
            for r, m in zip(rids, new):
                for i, x in enumerate((kr.cpu(), v)):
                    c, s = M.quantize(x[at:at + m], bits)
                    hist[r, layer][i] = torch.cat([hist[r, layer][i], M.values(c, s, bits)])
                kk, vv = hist[r, layer]
                ref, bound = W.attend(qr[at:at + m].cpu(), kk, vv, W.visible(len(kk), m, wl, sinks, True), 2.0 ** -8)
                err = (out[at:at + m].double().cpu() - ref).abs()
                assert (err <= bound).all(), (step, layer, r, (err / bound).max())
                at += m
        cm.advance_seq_lens()
        if step == 2:  # the same history under another label, whose pages are copies
            cm.snapshot_all("main", "copy")
            old, label = label, "copy"
            for r in rids:
                a, b = mgr.get_state(r, old).page_indices, mgr.get_state(r, label).page_indices
                assert len(a) == len(b) and not set(a) & set(b)
                assert torch.equal(kv.codes[:, a], kv.codes[:, b]) and torch.equal(kv.scales[:, a], kv.scales[:, b])
    with pytest.raises(ValueError):
        mgr.kv_transfer_engine  # noqa: B018


def test_run_attention_window(gpu):
    """run_attention's window over a 16-bit pool."""
    cfg = KVCacheConfig(num_layers=1, num_kv_heads=2, head_dim=64, max_seq_len=512, max_num_pages=64, page_size=16, num_qo_heads=8)
    kv = torch.zeros(1, 64, 2, 16, 2, 64, dtype=torch.bfloat16, device=gpu)
    mgr = PagedAllocationManager(cfg, kv, device=gpu)
    mgr.add_request("r", ["main"])
    cm = BatchedCacheManager(["r"], {"r": "main"}, kv, mgr, WorkspaceBufferManager(64 << 20, gpu), cfg, gpu)
    g = torch.Generator().manual_seed(2)
    q = torch.randn(100, 8, 64, generator=g).to(torch.bfloat16)
    k, v = (torch.randn(100, 2, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    cm.plan_attention([100])
    out = cm.run_attention(q.to(gpu), k.to(gpu), v.to(gpu), layer_idx=0, window_left=20, sink_tokens=2)
    ref, bound = W.attend(q, k, v, W.visible(100, 100, 20, 2, True), 2.0 ** -8)
    assert ((out.double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("captured", [False, True])
def test_both_parts_on_two_streams(gpu, captured):
    """A ragged batch large enough for its chunks and decodes to fork: equal to the parts in turn, eager and replayed."""
    hq, hkv, d, ps = 16, 2, 128, 16
    lens, new = [4300, 4200] + [3000] * 300, [4200, 4100] + [1] * 300
    pool = sum(-(-n // ps) for n in lens)
    qo, *idx = _index(lens, ps, pool, 31, new=new)
    g = torch.Generator().manual_seed(31)
    layer = torch.randn(pool, 2, ps, hkv, d, generator=g).to(torch.bfloat16).to(gpu)
    n = sum(new)
    q = torch.randn(n, hq, d, generator=g).to(torch.bfloat16).to(gpu)
    kw = dict(batch_size=len(lens), max_total_tokens=n, max_num_pages=pool, use_cuda_graph=True) if captured else {}
    w = PagedPrefillWrapper(workspace(gpu, 256 << 20), hq, hkv, d, ps, device=gpu, **kw)
    w.plan(qo, *idx)
    out = torch.empty_like(q)

    def run():
        return w.run(q, layer, out=out, window_left=2900, sink_tokens=5)

    forked = []
    wait = w._side.wait_stream
    w._side.wait_stream = lambda s: (forked.append(1), wait(s))[1]
    run()
    assert forked, "the parts did not fork"
    if captured:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run()
    for _ in range(3 if captured else 1):
        out.fill_(7.0)
        graph.replay() if captured else run()
        torch.cuda.synchronize()
        got = out.clone()
        w._serial = True
        assert torch.equal(got, w.run(q, layer, window_left=2900, sink_tokens=5))
        w._serial = False


def test_other_streams_and_two_at_once(gpu):
    """Two wrappers with workspaces of their own, planned on the default stream and run on two others at the same time."""
    ps = [H.make(gpu, kind, [3000, 40, 700, 1], 16, 4, 128, seed=i) for i, kind in enumerate(("bf16", "mx4"))]
    q = torch.randn(4, 32, 128, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    qg, ws, outs = q.to(gpu), [], []
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for p in ps:
        w = PagedDecodeWrapper(workspace(gpu, 64 << 20), 32, 4, 128, 16, device=gpu)
        w.plan(*p.index())
        ws.append(w)
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(5):
        for p, w, s in zip(ps, ws, streams):
            with torch.cuda.stream(s):
                outs.append(w.run(qg, p.layer, window_left=500, sink_tokens=9))
                outs[-1].record_stream(s)
    torch.cuda.synchronize()
    for i, o in enumerate(outs):
        H.check(ps[i % 2], q, [1] * 4, o, 500, 9, True, f"stream {i % 2}")


@pytest.mark.parametrize("kind", ["bf16", "mx8", "mx4"])
def test_layouts(gpu, kind):
    """Queries and outputs as views of wider rows; a pool whose pages hold heads before tokens."""
    lens, new = [300, 33, 1, 90], [120, 1, 1, 40]
    p = H.make(gpu, kind, lens, 16, 2, 128, seed=4)
    if kind == "bf16":
        hnd = p.layer.permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)
        assert hnd.stride(3) > hnd.stride(2)
        p.layer = hnd
    else:
        c = p.layer.codes.permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)
        p.layer = MXKVLayer(c, p.layer.scales)
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(sum(new) + 2, 12 * 128, generator=g).to(torch.bfloat16).to(gpu)
    q = wide[: sum(new), 128:9 * 128].view(sum(new), 8, 128)
    out = torch.full((sum(new) + 2, 10, 128), 2.0, dtype=torch.bfloat16, device=gpu)
    qo = torch.tensor([0] + list(torch.tensor(new).cumsum(0)), dtype=torch.int32)
    w = PagedPrefillWrapper(workspace(gpu, 64 << 20), 8, 2, 128, 16, device=gpu)
    w.plan(qo, *p.index())
    for kw in ({"window_left": 50, "sink_tokens": 2}, {}):
        view = out[:, 1:9]
        w.run(q, p.layer, out=view, **kw)
        torch.cuda.synchronize()
        H.check(p, q.cpu(), new, view, kw.get("window_left", -1), kw.get("sink_tokens", 0), True, kind)
        assert (out[:, 0] == 2).all() and (out[:, 9] == 2).all() and (out[sum(new):] == 2).all()
    # appended through the same layout
    k, v = (torch.randn(sum(new), 2, 128, generator=g).to(torch.bfloat16) for _ in range(2))
    w.set_kv_cache(p.layer, k.to(gpu), v.to(gpu))
    kk, _ = read_kv_cache(p.layer, *p.index(), sum(lens), torch.float32)
    at = np.cumsum([0] + lens)
    got = torch.cat([kk[at[r + 1] - n:at[r + 1]] for r, n in enumerate(new)]).cpu().double()
    want = k.double() if kind == "bf16" else M.values(*M.quantize(k, int(kind[2])), int(kind[2]))
    assert torch.equal(got, want)


@pytest.mark.parametrize("batch", [300, 1024, 1025, 1500])
def test_large_batches(gpu, batch):
    """Batches that are taken longest first, and those beyond what is sorted."""
    r = np.random.default_rng(batch)
    lens = np.where(r.random(batch) < 0.1, r.integers(200, 900, batch), r.integers(0, 60, batch)).tolist()
    p = H.make(gpu, "bf16", lens, 16, 2, 64, seed=batch)
    q = torch.randn(batch, 4, 64, generator=torch.Generator().manual_seed(6)).to(torch.bfloat16)
    w = PagedDecodeWrapper(workspace(gpu, 128 << 20), 4, 2, 64, 16, device=gpu)
    w.plan(*p.index())
    out = w.run(q.to(gpu), p.layer, window_left=300, sink_tokens=1)
    log(f"{H.check(p, q, [1] * batch, out, 300, 1, True, 'large batch'):.2f} of the bound")


@pytest.mark.parametrize("batch", [1, 5, 300])
def test_window_wider_than_every_context(gpu, batch):
    """Requests are cut and ordered by their own lengths where the window is far wider, up to the largest one."""
    r = np.random.default_rng(batch)
    lens = r.integers(1, 5000 if batch < 10 else 400, batch).tolist()
    p = H.make(gpu, "bf16", lens, 16, 4, 128, seed=batch)
    q = torch.randn(batch, 16, 128, generator=torch.Generator().manual_seed(11)).to(torch.bfloat16)
    w = PagedDecodeWrapper(workspace(gpu, 128 << 20), 16, 4, 128, 16, device=gpu)
    w.plan(*p.index())
    outs = [w.run(q.to(gpu), p.layer, window_left=wl, sink_tokens=sinks) for wl, sinks in
            ((5000, 0), (1 << 20, 7), (2**31 - 1, 2**31 - 1), (0, 2**31 - 1))]
    for out in outs:
        H.check(p, q, [1] * batch, out, -1, 0, True, "wide window")


@pytest.mark.parametrize("kind,hkv,d", [("bf16", 4, 128), ("mx4", 2, 256), ("bf16", 2, 256), ("mx8", 4, 64), ("fp8", 2, 128)])
@pytest.mark.parametrize("batch,wl,sinks", [(1, 2100, 3), (1, 300, 20), (3, 640, 0), (45, 900, 40), (100, 900, 0), (60, 33, 5)])
def test_cut_and_whole_requests(gpu, kind, hkv, d, batch, wl, sinks):
    """Requests in many items, in few, and whole to one workgroup of four or of eight wavefronts."""
    r = np.random.default_rng(batch + wl)
    lens = r.integers(1, 2600 if batch < 10 else 1200, batch).tolist()
    p = H.make(gpu, kind, lens, 16, hkv, d, seed=wl)
    q = torch.randn(batch, 4 * hkv, d, generator=torch.Generator().manual_seed(wl)).to(torch.bfloat16)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), 4 * hkv, hkv, d, 16, device=gpu)
    w.plan(*p.index())
    H.check(p, q, [1] * batch, w.run(q.to(gpu), p.layer, *p.scales, window_left=wl, sink_tokens=sinks), wl, sinks, True, kind)


@pytest.mark.parametrize("wl,sinks", [(100, 0), (700, 20)])
def test_paired_heads_cut_in_two(gpu, wl, sinks):
    """One kv-head pair a request: its window is cut in two items of the pair, which are merged."""
    lens = np.random.default_rng(wl).integers(1, 1200, 128).tolist()
    p = H.make(gpu, "bf16", lens, 16, 2, 128, seed=wl)
    q = torch.randn(128, 14, 128, generator=torch.Generator().manual_seed(wl)).to(torch.bfloat16)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), 14, 2, 128, 16, device=gpu)
    w.plan(*p.index())
    H.check(p, q, [1] * 128, w.run(q.to(gpu), p.layer, window_left=wl, sink_tokens=sinks), wl, sinks, True, "pair")


@pytest.mark.parametrize("hq,hkv,d", [(16, 2, 128), (8, 1, 256), (4, 4, 64)])
@pytest.mark.parametrize("wl,sinks", [(0, 0), (128, 4), (150, 32), (200, 0), (320, 0), (380, 0), (400, 33), (440, 0), (470, 0), (520, 64)])
def test_short_windows_of_cut_tiles(gpu, hq, hkv, d, wl, sinks):
    """Tiles that the plan cut for all their keys, behind windows that leave pieces to share them or do not."""
    new, lens = [290, 37], [6000, 2600]
    p = H.make(gpu, "bf16", lens, 16, hkv, d, seed=wl)
    H.hide(p, new, wl, sinks)
    q = torch.randn(sum(new), hq, d, generator=torch.Generator().manual_seed(wl)).to(torch.bfloat16)
    w = PagedPrefillWrapper(workspace(gpu, 128 << 20), hq, hkv, d, 16, device=gpu)
    for causal in (True, False):
        w.plan(torch.tensor([0, 290, 327], dtype=torch.int32), *p.index(), causal=causal)
        out = torch.full((sum(new), hq, d), 5.0, dtype=torch.bfloat16, device=gpu)
        w.run(q.to(gpu), p.layer, out=out, window_left=wl, sink_tokens=sinks)
        H.check(p, q, new, out, wl, sinks, causal, f"causal {causal}")


def test_read_from_pages_behind_others(gpu):
    """A list whose first request begins behind entries of none: those are not read; pages past the pool leave their rows."""
    p = H.make(gpu, "mx4", [40, 70], 16, 2, 64, seed=12)
    indptr, indices, last = p.index()
    want = read_kv_cache(p.layer, indptr, indices, last, 110)
    shifted = torch.cat([torch.tensor([-1, 10**6, 0], dtype=torch.int32), indices])
    got = read_kv_cache(p.layer, indptr + 3, shifted, last, 110)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    bad = indices.clone()
    bad[1], bad[4] = -5, p.layer.shape[0]
    out = tuple(torch.full_like(x, 9.0) for x in want)
    read_kv_cache(p.layer, indptr, bad, last, 110, out=out)
    for a, b in zip(out, want):
        assert (a[16:32] == 9).all() and (a[56:72] == 9).all()
        keep = [i for i in range(110) if not (16 <= i < 32 or 56 <= i < 72)]
        assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("kind", ["bf16", "mx8"])
def test_pool_past_32_bits(gpu, kind):
    """Pages whose byte offsets pass 2^32 (and, in the scales, 2^31): append, read, decode and chunks."""
    hq, hkv, d, ps = 16, 8, 256, 128
    pages = (5 << 30) // (2 * ps * hkv * d)
    lens, new = [300, 140], [200, 1]
    need = 5
    idx = torch.tensor([pages - 1, 3, pages - 2, pages // 2, pages - 3], dtype=torch.int32)
    indptr, last = torch.tensor([0, 3, 5], dtype=torch.int32), torch.tensor([44, 12], dtype=torch.int32)
    assert need == idx.numel()
    g = torch.Generator().manual_seed(7)
    if kind == "mx8":
        layer = MXKVLayer(torch.empty(pages, 2, ps, hkv, d, dtype=torch.uint8, device=gpu),
                          torch.empty(pages, 2, hkv, d // 32, ps, dtype=torch.uint8, device=gpu))
    else:
        layer = torch.empty(pages, 2, ps, hkv, d, dtype=torch.bfloat16, device=gpu)
    kv = [[torch.randn(n, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2)] for n in lens]
    full = PagedPrefillWrapper(workspace(gpu, 128 << 20), hq, hkv, d, ps, device=gpu)
    full.plan(torch.tensor([0, 300, 440], dtype=torch.int32), indptr, idx, last)
    full.set_kv_cache(layer, *(torch.cat([kv[r][i] for r in range(2)]).to(gpu) for i in range(2)))
    vals = [[M.values(*M.quantize(x, 8), 8) if kind == "mx8" else x.double() for x in pair] for pair in kv]
    got = read_kv_cache(layer, indptr, idx, last, 440, torch.float32)
    for i in range(2):
        assert torch.equal(got[i].cpu().double(), torch.cat([vals[r][i] for r in range(2)]))
    q = torch.randn(201, hq, d, generator=g).to(torch.bfloat16)
    w = PagedPrefillWrapper(workspace(gpu, 128 << 20), hq, hkv, d, ps, device=gpu)
    w.plan(torch.tensor([0, 200, 201], dtype=torch.int32), indptr, idx, last)
    for wl, sinks in ((150, 4), (-1, 0)):
        out = w.run(q.to(gpu), layer, window_left=wl, sink_tokens=sinks).double().cpu()
        for r, (a, b) in enumerate(((0, 200), (200, 201))):
            ref, bound = W.attend(q[a:b], *vals[r], W.visible(lens[r], new[r], wl, sinks, True), 2.0 ** -8)
            assert ((out[a:b] - ref).abs() <= bound).all()


@pytest.mark.parametrize("kind", ["mx8", "mx4"])
def test_decode_without_a_workspace(gpu, kind):
    p = H.make(gpu, kind, [700, 3, 64], 16, 4, 128, seed=8)
    q = torch.randn(3, 32, 128, generator=torch.Generator().manual_seed(9)).to(torch.bfloat16)
    qg, out = q.to(gpu), torch.empty(3, 32, 128, dtype=torch.bfloat16, device=gpu)
    idx = [t.to(gpu) for t in p.index()]
    _lib.check(_lib.lib().mi_decode_noalloc(qg.data_ptr(), 0, 32 * 128, 128, ctypes.byref(p.layer.desc), None,
                                            *(t.data_ptr() for t in idx), 3, 32, 0, 1 / math.sqrt(128), out.data_ptr(), 32 * 128,
                                            128, None, _lib.stream_ptr(gpu)), "mi_decode_noalloc")
    H.check(p, q, [1] * 3, out, -1, 0, True, kind)


def test_windowed_run_checks_its_tensors(gpu):
    p = H.make(gpu, "bf16", [40, 9], 16, 2, 128, seed=10)
    w = PagedDecodeWrapper(workspace(gpu, 32 << 20), 8, 2, 128, 16, device=gpu)
    w.plan(*p.index())
    q = torch.randn(2, 8, 128, device=gpu, dtype=torch.bfloat16)
    for bad in (torch.empty(1, 8, 128, device=gpu, dtype=torch.bfloat16), torch.empty(2, 8, 128, device=gpu, dtype=torch.float16),
                torch.empty(2, 8, 64, device=gpu, dtype=torch.bfloat16)):
        with pytest.raises(ValueError):
            w.run(q, p.layer, out=bad, window_left=3)
    f = PagedPrefillWrapper(workspace(gpu, 64 << 20), 8, 2, 128, 16, device=gpu)
    f.plan(torch.tensor([0, 30, 39], dtype=torch.int32), *p.index())
    with pytest.raises(ValueError):
        f.run(torch.randn(38, 8, 128, device=gpu, dtype=torch.bfloat16), p.layer, window_left=3)


def test_tensors_of_another_device_are_refused(gpu):
    """A tensor in host memory reaches no kernel."""
    p = H.make(gpu, "mx8", [40, 9], 16, 2, 128, seed=13)
    cpu = MXKVCache(1, 8, 16, 2, 128, device="cpu")[0]
    q, k = torch.zeros(2, 8, 128, dtype=torch.bfloat16), torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    w = PagedDecodeWrapper(workspace(gpu, 32 << 20), 8, 2, 128, 16, device=gpu)
    w.plan(*p.index())
    f = PagedPrefillWrapper(workspace(gpu, 64 << 20), 8, 2, 128, 16, device=gpu)
    f.plan(torch.tensor([0, 1, 2], dtype=torch.int32), *p.index())
    pool = torch.zeros(8, 2, 16, 2, 128, dtype=torch.bfloat16)
    for x in (w, f):
        for bad in (lambda: x.run(q, p.layer), lambda: x.run(q.to(gpu), cpu), lambda: x.run(q.to(gpu), pool, window_left=3),
                    lambda: x.run(q, pool.to(gpu), window_left=3), lambda: x.set_kv_cache(p.layer, k, k.to(gpu)),
                    lambda: x.set_kv_cache(p.layer, k.to(gpu), k), lambda: x.set_kv_cache(cpu, k.to(gpu), k.to(gpu)),
                    lambda: x.run(q.to(gpu), p.layer, out=torch.empty_like(q), window_left=3)):
            with pytest.raises(ValueError):
                bad()


def test_two_graphs_share_a_workspace(gpu):
    """A windowed and a full run captured apart on one wrapper, replayed by turns over replans with eager work between."""
    lens, new = [900, 300, 40, 7], [260, 1, 33, 1]
    p = H.make(gpu, "mx4", lens, 16, 4, 128, seed=14)
    pool = p.layer.shape[0]
    n = sum(new)
    w = PagedPrefillWrapper(workspace(gpu, 128 << 20), 16, 4, 128, 16, batch_size=4, max_total_tokens=n, max_num_pages=pool,
                            device=gpu, use_cuda_graph=True)
    g = torch.Generator().manual_seed(15)
    q = torch.randn(n, 16, 128, generator=g).to(torch.bfloat16).to(gpu)
    qo = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    w.plan(qo, *p.index())
    kws, outs, graphs = ({"window_left": 70, "sink_tokens": 2}, {}), [], []
    for kw in kws:
        w.run(q, p.layer, **kw)
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(w.run(q, p.layer, **kw))
    for i in range(6):
        if i % 2 == 0:
            q.copy_(torch.randn(n, 16, 128, generator=g).to(torch.bfloat16))
            w.plan(qo, *p.index())
        for j in (i % 2, 1 - i % 2):
            outs[j].zero_()
            graphs[j].replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[j], w.run(q, p.layer, **kws[j]))
            H.check(p, q.cpu(), new, outs[j], kws[j].get("window_left", -1), kws[j].get("sink_tokens", 0), True, f"{i} {j}")
