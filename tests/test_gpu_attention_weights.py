"""GPU: accumulated attention weights of cached tokens (mi_attention_weights) against 64 bits.

Bounds are oracle.eviction's (fp32 scores, exponentials and sums), and the rounding of adding to what was there.
"""

import ctypes

import numpy as np
import pytest
import torch

import mx_helpers as H
from gpu_helpers import custom_batch, log, workspace
from mstar_amd import _lib
from mstar_amd.eviction import kv_weights
from mstar_amd.mx_cache import MXKVLayer
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper
from oracle import eviction as E
from oracle import window as W

pytestmark = pytest.mark.gpu


def _start(p, gpu, seed=1):
    """Weights of every slot, NaN where no token lies or the step's own token does: those must not count."""
    g = torch.Generator().manual_seed(seed)
    hkv = p.values.shape[3]
    return torch.rand(p.values.shape[0], hkv, p.ps, generator=g) * 3


def _expect(p, q, new, causal, start):
    """(weights, bound) of every slot, in 64 bits."""
    want, bound = start.double().clone(), torch.zeros(start.shape, dtype=torch.float64)
    at = 0
    for r, n in enumerate(new):
        length = p.lens[r]
        if n and length:
            add, b = E.probabilities(q[at:at + n], p.rows(r, 0), W.visible(length, n, -1, 0, causal))
            pages = torch.as_tensor(p.kv_indices[p.kv_indptr[r]:p.kv_indptr[r + 1]]).long()
            t = torch.arange(length)
            page, slot = pages[t // p.ps], t % p.ps
            old = want[page, :, slot]
            old[max(0, length - n):] = 0
            want[page, :, slot] = old + add
            bound[page, :, slot] = b + (old + add).abs() * 2.0 ** -23
        at += n
    return want, bound


def _poison(p, start, new):
    """NaN in K and V past each request's end, and in the weights of its own tokens and past its end."""
    for r, n in enumerate(new):
        for e in range(p.kv_indptr[r], p.kv_indptr[r + 1]):
            first = (e - p.kv_indptr[r]) * p.ps
            page = int(p.kv_indices[e])
            past = [s for s in range(p.ps) if first + s >= p.lens[r]]
            if past:
                H.poison_layer(p.layer, page, past)
            if n:
                fresh = [s for s in range(p.ps) if first + s >= p.lens[r] - n]
                start[page][:, fresh] = float("nan")


def _same_or_near(got, want, bound, what):
    got = got.double().cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan), f"{what}: NaN elsewhere"
    err = (got - want).abs()[~nan]
    share = (err / (bound[~nan] + 1e-30)).max().item()
    log(f"  {what}: {share:.3f} of the bound")
    assert share <= 1, what


def _wrapper(p, gpu, hq, new, causal=True, dtype=torch.bfloat16, **kw):
    hkv, d = p.values.shape[3], p.values.shape[4]
    indptr, indices, last = p.index()
    if new is None:
        w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, p.ps, device=gpu, **kw)
        w.plan(indptr, indices, last, dtype=dtype)
    else:
        w = PagedPrefillWrapper(workspace(gpu, 64 << 20), hq, hkv, d, p.ps, device=gpu, **kw)
        w.plan(torch.as_tensor(np.concatenate([[0], np.cumsum(new)]).astype(np.int32)), indptr, indices, last, causal=causal,
               dtype=dtype)
    return w


def _run(p, gpu, hq, new, causal=True, dtype=None, seed=3):
    dtype = dtype or H.KINDS.get(p.kind, torch.bfloat16)
    counts = [1] * len(p.lens) if new is None else new
    d = p.values.shape[4]
    q = torch.randn(sum(counts), hq, d, generator=torch.Generator().manual_seed(seed)).to(dtype)
    start = _start(p, gpu)
    _poison(p, start, counts)
    want, bound = _expect(p, q, counts, causal, start)
    w = _wrapper(p, gpu, hq, new, causal, dtype)
    weights = start.to(gpu)
    w.accumulate_weights(q.to(gpu), p.layer, weights, *p.scales)
    torch.cuda.synchronize()
    # slots past a request's end keep what they held: NaN here
    _same_or_near(weights, want, bound, f"{p.kind} {hq} heads, {len(p.lens)} requests")
    return weights


@pytest.mark.parametrize("kind,hq,hkv,d,ps,lens", [
    ("bf16", 8, 2, 128, 16, [1, 2, 15, 16, 17, 300]),
    ("f16", 7, 1, 64, 32, [1, 31, 32, 33, 1000]),
    ("bf16", 16, 1, 256, 16, [5, 700, 64]),
    ("bf16", 28, 4, 128, 48, [47, 48, 49, 2000]),
    ("bf16", 4, 4, 64, 128, [1, 127, 500]),
    ("fp8", 32, 4, 128, 16, [3, 999, 256]),
    ("fp8_f16", 4, 1, 64, 16, [40, 777]),
    ("mx8", 6, 2, 256, 16, [33, 600]),
    ("mx8", 4, 1, 64, 16, [33, 600]),
    ("mx4", 8, 2, 128, 16, [1, 450]),
    ("mx4", 8, 8, 64, 16, [18, 450]),
    ("mx4", 2, 1, 256, 16, [18, 450]),
    ("mx8_f16", 8, 1, 128, 16, [100, 20]),
    ("mx4_f16", 8, 1, 64, 16, [100, 20]),
])
def test_decode(gpu, kind, hq, hkv, d, ps, lens):
    _run(H.make(gpu, kind, lens, ps, hkv, d, seed=hq + d), gpu, hq, None)


@pytest.mark.parametrize("kind,hq,hkv,d,ps,ctx,new,causal", [
    ("bf16", 8, 2, 128, 16, [0, 5, 300, 17], [40, 128, 33, 20], True),
    ("bf16", 8, 2, 128, 16, [0, 5, 300, 17], [40, 128, 33, 20], False),
    ("f16", 7, 1, 64, 32, [100, 0], [257, 5], True),           # one long, one short of 35 rows
    ("bf16", 16, 1, 256, 16, [500, 3], [9, 70], True),
    ("bf16", 4, 4, 64, 128, [0, 0, 1000], [300, 17, 16], True),  # a kv head's rows are its queries: 16 are short
    ("bf16", 28, 4, 128, 48, [100, 7], [50, 90], False),
    ("fp8", 32, 4, 128, 16, [900, 3], [32, 33], True),
    ("fp8_f16", 4, 1, 64, 16, [90], [120], True),
    ("mx8", 6, 2, 256, 16, [200, 0], [64, 31], True),
    ("mx8_f16", 4, 1, 64, 16, [200, 0], [64, 31], False),
    ("mx4", 8, 2, 128, 16, [333, 2], [64, 100], True),
    ("mx4", 8, 2, 256, 16, [333, 2], [20, 30], True),
    ("mx4_f16", 8, 1, 64, 16, [50, 1], [40, 60], True),
])
def test_chunks(gpu, kind, hq, hkv, d, ps, ctx, new, causal):
    _run(H.make(gpu, kind, [c + n for c, n in zip(ctx, new)], ps, hkv, d, seed=hq + d), gpu, hq, new, causal)


def test_mixed_batch_with_empty_requests(gpu):
    """Chunks, decodes, requests of a few tokens (short by rows), one without new tokens, one without keys."""
    new = [100, 1, 1, 3, 0, 4, 2, 1]
    ctx = [50, 400, 0, 77, 90, 0, 15, 2047]
    p = H.make(gpu, "bf16", [c + n for c, n in zip(ctx, new)], 16, 2, 128, seed=4)
    _run(p, gpu, 8, new)


def test_queries_before_the_first_key(gpu):
    """More queries than keys: the first queries see nothing and add nothing."""
    for hq, lens, new in ((4, [20, 3], [50, 64]), (4, [2, 1], [4, 3])):
        p = H.make(gpu, "bf16", lens, 16, 1, 128, seed=6)
        _run(p, gpu, hq, new)


def test_fp32(gpu):
    g = torch.Generator().manual_seed(7)
    for d, hq, hkv in ((64, 4, 2), (128, 6, 2), (256, 5, 1)):
        for new in (None, [1, 60, 30]):
            lens = [100, 200, 33]
            p = H.make(gpu, "bf16", lens, 16, hkv, d, seed=d)
            x = torch.randn(p.values.shape, generator=g)
            p.kind, p.layer, p.values = "f32", x.to(gpu), x.double()
            _run(p, gpu, hq, new, dtype=torch.float32)


def test_large_scores_and_long_contexts(gpu):
    """Scores of some hundreds (one key takes all) and one request over many runs of pages."""
    p = H.make(gpu, "bf16", [9000, 300], 16, 1, 128, seed=8, spread=12.0)
    _run(p, gpu, 4, None)
    p = H.make(gpu, "bf16", [3000, 700], 16, 1, 128, seed=9, spread=12.0)
    _run(p, gpu, 4, [40, 200])


def test_many_short_requests(gpu):
    """More requests than a wavefront's lanes: units are found by a search in steps."""
    g = np.random.default_rng(3)
    lens = g.integers(1, 60, 150).tolist()
    _run(H.make(gpu, "bf16", lens, 16, 2, 64, seed=2), gpu, 4, None)
    new = g.integers(0, 20, 150)
    _run(H.make(gpu, "bf16", (np.array(lens) + new).tolist(), 16, 2, 64, seed=2), gpu, 4, new.tolist())


def test_not_finite(gpu):
    """A NaN key makes its request's weights NaN for its kv head, an infinite query those of what it sees; others stay."""
    p = H.make(gpu, "bf16", [200, 200, 300], 16, 2, 128, seed=5)
    for new in (None, [50, 60, 70]):
        counts = new or [1, 1, 1]
        q = torch.randn(sum(counts), 8, 128, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
        start = _start(p, gpu)
        want, bound = _expect(p, q, counts, True, start)
        layer = p.layer.clone()
        page = int(p.kv_indices[p.kv_indptr[1]])
        layer[page, 0, 3, 1, 7] = float("nan")  # request 1, key 3, kv head 1
        w = _wrapper(p, gpu, 8, new)
        weights = start.to(gpu)
        w.accumulate_weights(q.to(gpu), layer, weights)
        torch.cuda.synchronize()
        pages = torch.as_tensor(p.kv_indices[p.kv_indptr[1]:p.kv_indptr[2]]).long()
        got = weights.cpu()[pages, 1].flatten()[:200]
        assert torch.isnan(got).all()
        want[pages[:, None], 1, torch.arange(16)] = torch.where(torch.arange(len(pages) * 16).view(-1, 16) < 200, float("nan"),
                                                                want[pages[:, None], 1, torch.arange(16)])
        _same_or_near(weights, want, bound, f"beside a NaN, {'decode' if new is None else 'chunks'}")


def test_steps_add_up_and_repeat_bit_for_bit(gpu):
    """Two steps over one request: the first step's tokens keep their weight; the same calls give the same bits."""
    ps, hq, hkv, d = 16, 8, 2, 128
    p = H.make(gpu, "bf16", [180, 33], ps, hkv, d, seed=3)
    g = torch.Generator().manual_seed(2)
    q1 = torch.randn(170 + 20, hq, d, generator=g).to(torch.bfloat16)
    q2 = torch.randn(10 + 13, hq, d, generator=g).to(torch.bfloat16)
    results = []
    for _ in range(2):
        weights = torch.full((p.values.shape[0], hkv, ps), float("nan"), device=gpu)
        one = H.make(gpu, "bf16", [180, 33], ps, hkv, d, seed=3)
        # the first step saw fewer tokens: the same pages, shorter
        first = PagedPrefillWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu)
        indptr = np.concatenate([[0], np.cumsum([-(-170 // ps), -(-20 // ps)])]).astype(np.int32)
        indices = np.concatenate([one.kv_indices[: indptr[1]], one.kv_indices[one.kv_indptr[1]:one.kv_indptr[1] + indptr[2] - indptr[1]]])
        last = np.array([170 - (indptr[1] - 1) * ps, 20 - (indptr[2] - indptr[1] - 1) * ps], np.int32)
        first.plan(torch.tensor([0, 170, 190], dtype=torch.int32), *(torch.as_tensor(a) for a in (indptr, indices, last)))
        first.accumulate_weights(q1.to(gpu), one.layer, weights)
        second = _wrapper(one, gpu, hq, [10, 13])
        second.accumulate_weights(q2.to(gpu), one.layer, weights)
        torch.cuda.synchronize()
        results.append(weights.cpu())
    assert torch.equal(results[0].view(torch.int32), results[1].view(torch.int32))
    for r, (length, old, at1, at2) in enumerate(((180, 170, 0, 0), (33, 20, 170, 10))):
        a, ba = E.probabilities(q1[at1:at1 + (170 if r == 0 else 20)], p.rows(r, 0)[:old], W.visible(old, old, -1, 0, True))
        n = length - old
        b, bb = E.probabilities(q2[at2:at2 + n], p.rows(r, 0), W.visible(length, n, -1, 0, True))
        b[:old] += a
        bb[:old] += ba
        pages = torch.as_tensor(p.kv_indices[p.kv_indptr[r]:p.kv_indptr[r + 1]]).long()
        got = results[0][pages].transpose(0, 1).flatten(1)[:, :length].T
        assert ((got.double() - b).abs() <= bb + b * 2.0 ** -22).all()


def test_strided_queries_other_layouts_and_a_side_stream(gpu):
    """q as a view of a projection, a pool whose heads come before its tokens, and a call on another stream than the plan's."""
    hq, hkv, d, ps = 8, 2, 128, 16
    p = H.make(gpu, "bf16", [300, 20, 111], ps, hkv, d, seed=5)
    hnd = p.layer.permute(0, 1, 3, 2, 4).contiguous().permute(0, 1, 3, 2, 4)
    for new in (None, [30, 1, 100]):
        counts = new or [1, 1, 1]
        wide = torch.randn(sum(counts), (hq + 2) * d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
        q = wide[:, d:d + hq * d].unflatten(1, (hq, d))
        start = _start(p, gpu)
        want, bound = _expect(p, q.cpu(), counts, True, start)
        w = _wrapper(p, gpu, hq, new)
        weights, side = start.to(gpu), torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            w.accumulate_weights(q, hnd, weights)
        torch.cuda.current_stream().wait_stream(side)
        torch.cuda.synchronize()
        _same_or_near(weights, want, bound, "strided")


def test_captured_and_replayed(gpu):
    """Captured with the largest sizes, replayed for other lengths, beside eager work: each replay equals the eager call."""
    hq, hkv, d, ps, b, pool = 8, 2, 128, 16, 4, 200
    layer = torch.randn(pool, 2, ps, hkv, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
    for ragged in (False, True):
        kw = dict(batch_size=b, max_num_pages=pool, device=gpu, use_cuda_graph=True)
        cls = PagedPrefillWrapper if ragged else PagedDecodeWrapper
        w = cls(workspace(gpu, 64 << 20), hq, hkv, d, ps, **kw, **(dict(max_total_tokens=256) if ragged else {}))
        e = cls(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu)
        q = torch.zeros(256 if ragged else b, hq, d, dtype=torch.bfloat16, device=gpu)
        weights = torch.zeros(pool, hkv, ps, device=gpu)

        def index(lens, new, seed):
            qo, *rest = (torch.as_tensor(a) for a in custom_batch(lens, ps, pool, seed, new_lens=new))
            return (qo, *rest) if ragged else rest

        w.plan(*index([200] * b, [10] * b, 1))
        w.accumulate_weights(q, layer, weights)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            w.accumulate_weights(q, layer, weights)
        for i, (lens, new) in enumerate((([1, 700, 30, 200], [1, 90, 3, 100]), ([64, 64, 64, 64], [64, 64, 64, 64]),
                                         ([1500, 2, 1, 9], [200, 2, 1, 0]))):
            q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
            start = torch.rand(weights.shape, generator=torch.Generator().manual_seed(i)).to(gpu)
            weights.copy_(start)
            w.plan(*index(lens, new, 5 + i))
            graph.replay()
            e.plan(*index(lens, new, 5 + i))
            e.accumulate_weights(q, layer, start)
            torch.cuda.synchronize()
            # the cuts of the work follow the call's bounds, which differ: near, and equal in what was not touched
            assert torch.allclose(weights, start, rtol=1e-4, atol=1e-6), (ragged, lens)
            assert bool(((weights - start).abs() <= 2e-5 * start + 1e-6).all())


def test_pages_out_of_range_and_past_the_list(gpu):
    """An id out of range gets no weights and breaks nothing; a graph's list longer than the batch's is not read."""
    hq, hkv, d, ps, pool = 4, 1, 64, 16, 12
    layer = torch.randn(pool, 2, ps, hkv, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
    for ids in ([3, pool, 5], [3, -1, 5]):
        for new in (None, [40]):
            cls = PagedDecodeWrapper if new is None else PagedPrefillWrapper
            w = cls(workspace(gpu, 16 << 20), hq, hkv, d, ps, device=gpu)
            idx = (torch.tensor([0, 3], dtype=torch.int32), torch.tensor([3, 4, 5], dtype=torch.int32), torch.tensor([10], dtype=torch.int32))
            w.plan(*(idx if new is None else (torch.tensor([0, 40], dtype=torch.int32), *idx)))
            w._indices.copy_(torch.tensor(ids, dtype=torch.int32))
            weights = torch.zeros(pool, hkv, ps, device=gpu)
            w.accumulate_weights(torch.ones(1 if new is None else 40, hq, d, dtype=torch.bfloat16, device=gpu), layer, weights)
            torch.cuda.synchronize()
            got = weights.cpu()
            assert bool((got[3] > 0).all()) and bool((got[5, :, :10] > 0).all()) and not bool(got[5, :, 10:].any())
            assert not bool(got[[i for i in range(pool) if i not in (3, 5)]].any())


def test_pool_past_4_gib(gpu):
    """Offsets past 32 bits: a pool of 5 GiB, the request's pages at its end."""
    hq, hkv, d, ps = 8, 4, 128, 16
    pool = (5 << 30) // (2 * ps * hkv * d * 2)
    layer = torch.zeros(pool, 2, ps, hkv, d, dtype=torch.bfloat16, device=gpu)
    ids = torch.tensor([pool - 1, 0, pool - 2, 7], dtype=torch.int32)
    part = torch.randn(4, 2, ps, hkv, d, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16)
    layer[ids.long().to(gpu)] = part.to(gpu)
    k = part[:, 0].flatten(0, 1)[:61]
    for new in (1, 30):
        q = torch.randn(new, hq, d, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
        w = PagedPrefillWrapper(workspace(gpu, 16 << 20), hq, hkv, d, ps, device=gpu)
        w.plan(torch.tensor([0, new], dtype=torch.int32), torch.tensor([0, 4], dtype=torch.int32), ids, torch.tensor([13], dtype=torch.int32))
        weights = kv_weights(layer)
        w.accumulate_weights(q.to(gpu), layer, weights)
        want, bound = E.probabilities(q, k, W.visible(61, new, -1, 0, True))
        got = weights[ids.long().to(gpu)].cpu().transpose(1, 2).flatten(0, 1)[:61]
        assert ((got.double() - want).abs() <= bound + want * 2.0 ** -23).all()
        assert float(weights.sum()) == pytest.approx(new * hq, rel=1e-5)


def test_refusals(gpu):
    hq, hkv, d, ps, pool = 8, 2, 128, 16, 8
    layer = torch.zeros(pool, 2, ps, hkv, d, dtype=torch.bfloat16, device=gpu)
    q = torch.zeros(2, hq, d, dtype=torch.bfloat16, device=gpu)
    weights = kv_weights(layer)
    w = PagedDecodeWrapper(workspace(gpu, 16 << 20), hq, hkv, d, ps, device=gpu)
    with pytest.raises(RuntimeError):
        w.accumulate_weights(q, layer, weights)
    w.plan(torch.tensor([0, 1, 3], dtype=torch.int32), torch.tensor([0, 1, 2], dtype=torch.int32), torch.tensor([5, 6], dtype=torch.int32))
    call = w.accumulate_weights
    for bad in (lambda: call(q[:1], layer, weights), lambda: call(q[:, :4], layer, weights), lambda: call(q, layer[:, :, :, :1], weights),
                lambda: call(q, layer, weights[:4]), lambda: call(q, layer, weights.double()), lambda: call(q, layer, weights.cpu()),
                lambda: call(q, layer.cpu(), weights), lambda: call(q, layer, weights.transpose(1, 2).contiguous().transpose(1, 2)),
                lambda: call(q, layer, torch.zeros(weights.numel() + 1, device=gpu)[1:].view(weights.shape)),
                lambda: call(q, layer.to(torch.float8_e4m3fn), weights), lambda: call(q.cpu(), layer, weights)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):  # an fp16 layer under a bf16 plan
        call(q, layer.half(), weights)
    assert not bool(weights.any())


@pytest.mark.parametrize("kind,hq,hkv,d", [("bf16", 8, 2, 128), ("f16", 8, 8, 64), ("mx4", 16, 1, 64), ("fp8", 6, 2, 256), ("mx8_f16", 3, 1, 128),
                                           ("bf16", 2, 2, 256), ("mx4", 9, 1, 128), ("mx8", 12, 1, 64), ("fp8_f16", 5, 1, 64)])
@pytest.mark.parametrize("lens", [[1], [512], [513], [1000, 8], [1024, 1], [500, 300, 100, 0, 16], [1900, 1, 1, 1, 1], [9000], [12000, 5, 0, 16]])
def test_either_side_of_one_launch(gpu, kind, hq, hkv, d, lens):
    """Batches whose scores fit a workgroup's LDS, and those past it, with many runs of pages to join."""
    _run(H.make(gpu, kind, lens, 16, hkv, d, seed=hq + d), gpu, hq, None)


@pytest.mark.parametrize("lens", [[100, 33], [9000, 20], [700, 900]])
def test_short_fp32(gpu, lens):
    """One query a request, either side of one launch."""
    g = torch.Generator().manual_seed(8)
    for d, hq, hkv in ((64, 4, 2), (128, 6, 2), (256, 5, 1)):
        p = H.make(gpu, "bf16", lens, 16, hkv, d, seed=d)
        x = torch.randn(p.values.shape, generator=g)
        p.kind, p.layer, p.values = "f32", x.to(gpu), x.double()
        _run(p, gpu, hq, None, dtype=torch.float32)


@pytest.mark.parametrize("row", [0, 7, 49])
def test_a_query_that_is_not_finite_reaches_what_it_sees(gpu, row):
    """Rows past the last of a tile are read as another's: a NaN there must stay with the keys that its query sees."""
    for ctx, n in ((40, 50), (300, 50), (0, 50)):
        p = H.make(gpu, "bf16", [ctx + n], 16, 2, 128, seed=5)
        q = torch.randn(n, 6, 128, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
        q[row, 1, 3] = float("nan")  # of kv head 0
        weights = kv_weights(p.layer)
        _wrapper(p, gpu, 6, [n]).accumulate_weights(q.to(gpu), p.layer, weights)
        pages = torch.as_tensor(p.kv_indices).long()
        got = weights.cpu()[pages].permute(1, 0, 2).flatten(1)[:, :ctx + n]
        assert bool(got[0, :ctx + row + 1].isnan().all()) and bool(got[0, ctx + row + 1:].isfinite().all())
        assert bool(got[1].isfinite().all())


def test_one_launch_captured_and_replayed(gpu):
    """A static page list small enough for one launch: replays equal eager calls over other lengths, requests of no keys among them."""
    hq, hkv, d, ps, b, pool = 8, 2, 128, 16, 4, 120
    layer = torch.randn(pool, 2, ps, hkv, d, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(gpu)
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, batch_size=b, max_num_pages=pool, device=gpu, use_cuda_graph=True)
    e = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu)
    q, weights = torch.zeros(b, hq, d, dtype=torch.bfloat16, device=gpu), torch.zeros(pool, hkv, ps, device=gpu)
    w.plan(*(torch.as_tensor(a) for a in custom_batch([200] * b, ps, pool, 1)[1:]))
    w.accumulate_weights(q, layer, weights)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.accumulate_weights(q, layer, weights)
    for i, lens in enumerate(([1, 700, 30, 200], [1800, 1, 2, 16], [64, 0, 64, 0], [1, 700, 30, 200])):
        q.copy_(torch.randn(q.shape, generator=torch.Generator().manual_seed(i)))
        start = torch.rand(weights.shape, generator=torch.Generator().manual_seed(i)).to(gpu)
        weights.copy_(start)
        index = [torch.as_tensor(a) for a in custom_batch(lens, ps, pool, 5 + i)[1:]]
        w.plan(*index)
        graph.replay()
        e.plan(*index)
        e.accumulate_weights(q, layer, start)
        torch.cuda.synchronize()
        assert bool(((weights - start).abs() <= 2e-5 * start + 1e-6).all()), lens
