"""GPU: norms of q and k with rotation and append (mi_qk_norm_rope) against 64 bits.

Bounds are oracle.qk_norm's: fp32 arithmetic, one rounding to the q / k type or the cache's.
"""

import numpy as np
import pytest
import torch

from gpu_helpers import custom_batch, log, workspace
from mstar_amd import rope as MR
from mstar_amd.mx_cache import MXKVCache, MXKVLayer
from mstar_amd.paged_attention import PagedDecodeWrapper, PagedPrefillWrapper
from oracle import microscaled as M
from oracle import qk_norm as N

pytestmark = pytest.mark.gpu

L31 = dict(low_freq_factor=1.0, high_freq_factor=4.0, old_context_len=8192)
BF, F16 = torch.bfloat16, torch.float16


def _fused(t, hq, hkv, d, dtype, seed, spread=1.0):
    """q, k, v as views of one projection, on the CPU."""
    x = (torch.randn(t, (hq + 2 * hkv) * d, generator=torch.Generator().manual_seed(seed)) * spread).to(dtype)
    return x, lambda y: tuple(p.unflatten(1, (-1, d)) for p in y.split([hq * d, hkv * d, hkv * d], 1))


def _weights(d, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple((1 + 0.3 * torch.randn(d, generator=g)).to(dtype) for _ in range(2))


def _check(got, out, bound, dtype, what):
    b = N.rounded(out, bound, dtype)
    share = ((got.double().cpu() - out).abs() / b).max().item()
    log(f"  {what}: {share:.3f} of the bound")
    assert share <= 1, what


CASES = [
    # dtype, weight dtype, hq, hkv, d, rotary_dim, interleave, llama31, tokens, farthest position
    (BF, BF, 32, 4, 128, 128, False, None, 1, 131072),
    (BF, BF, 8, 2, 128, 128, False, None, 300, 40000),
    (F16, F16, 16, 4, 64, 32, True, None, 77, 2000000),
    (F16, torch.float32, 5, 1, 256, 256, False, L31, 130, 300000),
    (BF, torch.float32, 3, 3, 256, 64, False, L31, 65, 100000),
    (BF, BF, 28, 4, 128, 64, True, L31, 2000, 60000),
    (F16, F16, 7, 1, 64, 16, False, None, 33, 1000),
    (BF, BF, 2, 5, 96, 96, False, None, 50, 5000),
    (BF, BF, 1, 1, 512, 512, False, None, 9, 5000),
    (F16, F16, 3, 2, 40, 16, True, None, 19, 5000),
    (BF, BF, 4, 1, 8, 8, True, None, 100, 5000),
]


@pytest.mark.parametrize("dtype,wdt,hq,hkv,d,rd,interleave,llama31,t,far", CASES)
def test_in_place(gpu, dtype, wdt, hq, hkv, d, rd, interleave, llama31, t, far):
    x, views = _fused(t, hq, hkv, d, dtype, d + rd + t)
    qw, kw = _weights(d, wdt, d)
    pos = torch.randint(0, far, (t,), generator=torch.Generator().manual_seed(t))
    pos[0] = far - 1
    y = x.to(gpu)
    q, k, v = views(y)
    rope = dict(rotary_dim=rd, interleave=interleave, rope_scale=8.0 if llama31 else 1.0, rope_theta=1e6, llama31=llama31)
    log(f"{dtype} {hq}/{hkv} x {d}, {rd} rotated, {t} tokens")
    MR.apply_qk_norm_rope_pos_ids_inplace(q, k, qw.to(gpu), kw.to(gpu), pos.to(gpu).to(torch.int32 if t % 2 else torch.int64),
                                          eps=1e-5, **rope)
    torch.cuda.synchronize()
    for name, got, src, w in (("q", q, views(x)[0], qw), ("k", k, views(x)[1], kw)):
        _check(got, *N.norm_rope(src, w, pos, 1e-5, **rope), dtype, name)
    assert torch.equal(v.cpu(), views(x)[2])


def _layer(kind, pool, ps, hkv, d, gpu):
    """(layer, scales, values(page, which, slot) -> float64 rows) of a cache full of ones."""
    if kind in ("mx8", "mx4"):
        layer = MXKVCache(1, pool, ps, hkv, d, bits=int(kind[2]), device=gpu)[0]
        layer.scales.fill_(3)

        def values(page, which, slot):
            codes = M.unpack(layer.codes.cpu()[page, which, slot], layer.bits)
            return M.values(codes, layer.scales.cpu()[page, which, :, :, slot], layer.bits)

        return layer, (None, None), values
    dtype = {"bf16": BF, "f16": F16, "f32": torch.float32, "fp8": torch.float8_e4m3fn}[kind]
    layer = torch.ones(pool, 2, ps, hkv, d, device=gpu).to(dtype)
    scales = (None, None)
    if kind == "fp8":
        scales = tuple((torch.rand(hkv, generator=torch.Generator().manual_seed(i)) * 0.01 + 0.008).to(gpu) for i in range(2))

    def values(page, which, slot):
        rows = layer.cpu()[page, which, slot].double()
        return rows * scales[which].double().cpu()[:, None] if kind == "fp8" else rows

    return layer, scales, values


def _cache_bound(kind, out, bound):
    """How far a cached value may be from ``out``: its half step (of the value, or of the least one) and ``bound``."""
    if kind in ("bf16", "f16", "f32"):
        return N.rounded(out, bound, {"bf16": BF, "f16": F16, "f32": torch.float32}[kind])
    if kind == "fp8":  # relative to the head's scale: normal values half a step of 2^-4, subnormal ones 2^-10
        return bound + (out.abs() + bound) * 2.0 ** -4 + 0.018 * 2.0 ** -10
    # a block's scale is at most its peak / (T / 2), twice that if the peak is within `bound` of the limit; clipping (16 of 464, 1 of
    # 7) is within the half step of the value
    step, low, limit = (2.0 ** -4, 2.0 ** -10, 464.0) if kind == "mx8" else (2.0 ** -2, 0.25, 7.0)
    peak = (out.abs() + bound).unflatten(-1, (-1, 32)).amax(-1, keepdim=True).expand(*out.shape[:-1], -1, 32).flatten(-2)
    return bound + (out.abs() + bound) * step + low * peak * 4 / limit


@pytest.mark.parametrize("dtype,kind,hq,hkv,d,rd,interleave,llama31,keep_k,idx_stride", [
    (BF, "bf16", 8, 2, 128, 128, False, None, True, 1),
    (F16, "f16", 6, 3, 64, 32, True, None, False, 2),
    (BF, "f16", 7, 1, 128, 64, False, L31, True, 1),
    (F16, "bf16", 5, 1, 256, 256, False, None, False, 1),
    (BF, "f32", 4, 2, 256, 128, False, None, True, 2),
    (BF, "fp8", 32, 4, 128, 128, False, None, False, 1),
    (F16, "fp8", 3, 1, 64, 64, True, L31, True, 1),
    (BF, "mx8", 16, 2, 256, 256, False, None, False, 1),
    (F16, "mx8", 4, 4, 64, 64, False, None, True, 2),
    (BF, "mx4", 8, 2, 128, 64, False, None, False, 1),
    (F16, "mx4", 2, 1, 64, 32, True, None, True, 1),
    (BF, "mx4", 2, 1, 96, 32, False, None, True, 1),
    (BF, "bf16", 2, 3, 80, 80, False, None, True, 1),
])
def test_append(gpu, dtype, kind, hq, hkv, d, rd, interleave, llama31, keep_k, idx_stride):
    t, pool, ps = 203, 64, 16
    n_append, n_dev = 190, 170  # tokens from 170 on are a graph's padding: rotated, not written
    x, views = _fused(t, hq, hkv, d, dtype, d + hq)
    qw, kw = _weights(d, dtype, d)
    g = torch.Generator().manual_seed(5)
    places = torch.randperm(pool * ps, generator=g)[:t]
    page, slot = places // ps, places % ps
    page[3], slot[5], page[7] = -1, ps, pool  # left out
    pos = torch.randint(0, 100000, (t,), generator=g)
    layer, scales, values = _layer(kind, pool, ps, hkv, d, gpu)
    before = [s.clone() for s in ((layer.codes, layer.scales) if isinstance(layer, MXKVLayer) else (layer,))]
    if idx_stride == 2:
        loc = torch.stack([page, slot], 1).contiguous().to(gpu)
        idx = (loc, loc.data_ptr() + 8)
    else:
        on = page.to(gpu), slot.to(gpu)
        idx = (on[0], on[1].data_ptr())
    count = torch.tensor([n_dev], dtype=torch.int32, device=gpu)
    rope = dict(rotary_dim=rd, interleave=interleave, rope_scale=8.0 if llama31 else 1.0, rope_theta=5e5, llama31=llama31)
    y = x.to(gpu)
    q, k, v = views(y)
    log(f"{dtype} -> {kind} {hq}/{hkv} x {d}")
    MR.qk_norm_rope_append(q, k, v, qw.to(gpu), kw.to(gpu), layer, pos.to(gpu), *idx, idx_stride, n_append, count.data_ptr(),
                           k_scale=scales[0], v_scale=scales[1], keep_k=keep_k, eps=1e-6, **rope)
    torch.cuda.synchronize()
    xq, xk, xv = views(x)
    _check(q, *N.norm_rope(xq, qw, pos, 1e-6, **rope), dtype, "q")
    out, bound = N.norm_rope(xk, kw, pos, 1e-6, **rope)
    if keep_k:
        _check(k, out, bound, dtype, "k")
    else:
        assert torch.equal(k.cpu(), xk)
    assert torch.equal(v.cpu(), xv)
    ok = [i for i in range(n_dev) if i not in (3, 5, 7)]
    got_k, got_v = (values(page[ok], i, slot[ok]) for i in (0, 1))
    if kind == "fp8":  # an append clamps to the largest code
        top = 448 * scales[0].double().cpu()[:, None]
        out = out.clamp(-top, top)
    share = ((got_k - out[ok]).abs() / _cache_bound(kind, out, bound)[ok]).max().item()
    log(f"  cached k: {share:.3f} of the bound")
    assert share <= 1
    if kind in ("mx8", "mx4"):
        bits = int(kind[2])
        assert torch.equal(got_v, M.values(*M.quantize(xv[ok].double(), bits), bits))  # v is quantised as set_kv_cache does
        same = (got_k == M.values(*M.quantize(out[ok], bits), bits)).double().mean()
        # fp32 noise of a few 1e-6 moves a value over a code's border, or a peak over a scale's, in far fewer than a thousandth
        assert same > 0.999
    elif kind == "fp8":
        want = (xv[ok].float() * (1 / scales[1].cpu())[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn).double()
        assert torch.equal(got_v, want * scales[1].double().cpu()[:, None])
    else:
        assert torch.equal(got_v, xv[ok].to(layer.dtype).double())
    # nothing else was written
    after = (layer.codes, layer.scales) if isinstance(layer, MXKVLayer) else (layer,)
    for a, b in zip(after, before):
        a, b = a.cpu().view(torch.uint8).clone(), b.cpu().view(torch.uint8).clone()
        if a.shape[2] == ps:
            a[page[ok], :, slot[ok]] = b[page[ok], :, slot[ok]] = 0
        else:
            a[page[ok], :, :, :, slot[ok]] = b[page[ok], :, :, :, slot[ok]] = 0
        assert torch.equal(a, b)


def test_rows_that_are_not_finite_stay_alone(gpu):
    """A row of zeros gives zeros, one with a NaN is NaN, one with an infinity is no other row's matter."""
    t, hq, hkv, d = 6, 4, 2, 128
    x, views = _fused(t, hq, hkv, d, BF, 3)
    q, k, _ = views(x)
    q[1, 2], q[2, 0, 5], k[3, 1, 100] = 0, float("nan"), float("inf")
    qw, kw = _weights(d, BF, 1)
    pos = torch.arange(t) * 1000
    gq, gk = q.to(gpu).contiguous(), k.to(gpu).contiguous()
    MR.apply_qk_norm_rope_pos_ids_inplace(gq, gk, qw.to(gpu), kw.to(gpu), pos.to(gpu), eps=1e-6)
    torch.cuda.synchronize()
    gq, gk = gq.cpu(), gk.cpu()
    assert (gq[1, 2] == 0).all() and torch.isnan(gq[2, 0]).all()
    rope = dict(rotary_dim=d, interleave=False, rope_scale=1.0, rope_theta=1e4, llama31=None)
    for got, src, w, bad in ((gq, q, qw, (2, 0)), (gk, k, kw, (3, 1))):
        src = src.clone()
        src[bad] = 1
        out, bound = N.norm_rope(src, w, pos, 1e-6, **rope)
        got = got.clone()
        got[bad] = out[bad].to(BF)
        _check(got, out, bound, BF, "the others")


def test_no_tokens_one_side_only_and_zero_eps(gpu):
    d = 64
    qw, kw = (w.to(gpu) for w in _weights(d, BF, 1))
    q, k = torch.randn(0, 4, d, device=gpu).to(BF), torch.randn(0, 2, d, device=gpu).to(BF)
    MR.apply_qk_norm_rope_pos_ids_inplace(q, k, qw, kw, torch.zeros(0, dtype=torch.long, device=gpu))
    x = torch.randn(5, 3, d, generator=torch.Generator().manual_seed(1)).to(BF)
    q = x.to(gpu)
    MR.apply_qk_norm_rope_pos_ids_inplace(q, q[:, :0], qw, kw, torch.arange(5, device=gpu), eps=0.0)
    out, bound = N.norm_rope(x, qw.cpu(), torch.arange(5), 0.0, d, False, 1.0, 1e4, None)
    _check(q, out, bound, BF, "q alone")


def _plan(cls, gpu, new, ctx, ps, hq, hkv, d, **kw):
    lens = [c + n for c, n in zip(ctx, new)]
    pool = sum(-(-n // ps) for n in lens) + 3
    qo, indptr, indices, last = (torch.as_tensor(a) for a in custom_batch(lens, ps, pool, 4, new_lens=new))
    w = cls(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu, **kw)
    w.plan(*((indptr, indices, last) if cls is PagedDecodeWrapper else (qo, indptr, indices, last)))
    return w, pool


@pytest.mark.parametrize("cls,new", [(PagedDecodeWrapper, [1] * 5), (PagedPrefillWrapper, [3, 1, 40, 0, 17])])
@pytest.mark.parametrize("kind", ["bf16", "mx8"])
def test_wrappers_write_where_set_kv_cache_writes(gpu, cls, new, kind):
    """The same slots as the plan's set_kv_cache of the normed, rotated k, and the same rows where the cache is k's type."""
    hq, hkv, d, ps = 8, 2, 128, 16
    w, pool = _plan(cls, gpu, new, [30, 0, 5, 64, 100], ps, hq, hkv, d)
    t = sum(new)
    x, views = _fused(t, hq, hkv, d, BF, 9)
    qw, kw = (a.to(gpu) for a in _weights(d, BF, 2))
    pos = torch.arange(t, device=gpu) + 70000
    a, b = x.to(gpu), x.to(gpu)
    layers = [_layer(kind, pool, ps, hkv, d, gpu)[0] for _ in range(2)]
    q, k, v = views(a)
    w.qk_norm_rope_set_kv_cache(layers[0], q, k, v, qw, kw, pos, rope_theta=1e6)
    q2, k2, v2 = views(b)
    MR.apply_qk_norm_rope_pos_ids_inplace(q2, k2, qw, kw, pos, rope_theta=1e6)
    w.set_kv_cache(layers[1], k2, v2)
    torch.cuda.synchronize()
    assert torch.equal(q, q2) and torch.equal(k, k2)
    if kind == "bf16":
        assert torch.equal(layers[0], layers[1])
    else:
        written = [layer.scales != 3 for layer in layers]  # what was not written is 3
        assert torch.equal(written[0], written[1])


def test_captured_and_replayed(gpu):
    """A captured call replayed for other values, positions and places, the padding left out: each replay equals the eager call."""
    hq, hkv, d, ps, b = 8, 2, 128, 16, 4
    pool = 80
    w = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, batch_size=b, max_num_pages=pool, device=gpu, use_cuda_graph=True)
    e = PagedDecodeWrapper(workspace(gpu, 64 << 20), hq, hkv, d, ps, device=gpu)
    qw, kw = (a.to(gpu) for a in _weights(d, BF, 2))
    x, views = _fused(b, hq, hkv, d, BF, 1)
    static, pos = x.to(gpu), torch.zeros(b, dtype=torch.long, device=gpu)
    layer, want = (torch.zeros(pool, 2, ps, hkv, d, dtype=BF, device=gpu) for _ in range(2))

    def index(lens, seed):
        return tuple(torch.as_tensor(a) for a in custom_batch(lens, ps, pool, seed)[1:])

    w.plan(*index([20] * b, 1))
    w.qk_norm_rope_set_kv_cache(layer, *views(static), qw, kw, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.qk_norm_rope_set_kv_cache(layer, *views(static), qw, kw, pos)
    for i, lens in enumerate(([1, 16, 17, 300], [5, 5, 5, 5], [100, 1, 64, 33])):
        x, _ = _fused(b, hq, hkv, d, BF, 20 + i)
        layer.zero_(), want.zero_()
        static.copy_(x), pos.copy_(torch.arange(b) * 11111 + i)
        w.plan(*index(lens, 30 + i))
        graph.replay()
        e.plan(*index(lens, 30 + i))
        y = x.to(gpu)
        e.qk_norm_rope_set_kv_cache(want, *views(y), qw, kw, pos)
        torch.cuda.synchronize()
        assert torch.equal(static, y) and torch.equal(layer, want) and bool(layer.any())


def test_refusals(gpu):
    d, t = 128, 4
    q, k = torch.zeros(t, 4, d, dtype=BF, device=gpu), torch.zeros(t, 2, d, dtype=BF, device=gpu)
    w, pos = torch.ones(d, dtype=BF, device=gpu), torch.arange(t, device=gpu)
    call = MR.apply_qk_norm_rope_pos_ids_inplace
    for bad in (
        lambda: call(q, k.half(), w, w, pos), lambda: call(q.float(), k.float(), w, w, pos), lambda: call(q, k[:3], w, w, pos),
        lambda: call(q, k, w[:64], w, pos), lambda: call(q, k, w.half(), w, pos), lambda: call(q, k, w.float(), w, pos),
        lambda: call(q, k, w.cpu(), w, pos), lambda: call(q, k, w, w, pos[:3]), lambda: call(q, k, w, w, pos.float()),
        lambda: call(q, k, w, w, pos, rotary_dim=24), lambda: call(q, k, w, w, pos, rotary_dim=256),
        lambda: call(q, k, w, w, pos, rotary_dim=12, interleave=True), lambda: call(q, k, w, w, pos, eps=-1.0),
        lambda: call(q, k, w, w, pos, eps=float("nan")), lambda: call(q, k, w, w, pos, rope_theta=0.0),
        lambda: call(q[..., 4:68], k[..., 4:68], w[:64], w[:64], pos), lambda: call(q, k, torch.ones(2 * d, dtype=BF, device=gpu)[::2], w, pos),
        lambda: call(q, k, w, w, pos, llama31=dict(low_freq_factor=4.0, high_freq_factor=1.0)),
        lambda: call(torch.zeros(t, 1, 520, dtype=BF, device=gpu), torch.zeros(t, 1, 520, dtype=BF, device=gpu),
                     torch.ones(520, dtype=BF, device=gpu), torch.ones(520, dtype=BF, device=gpu), pos, rotary_dim=16),
    ):
        with pytest.raises(ValueError):
            bad()
    idx = torch.zeros(t, dtype=torch.long, device=gpu)
    cache = torch.zeros(2, 2, 16, 2, d, dtype=BF, device=gpu)

    def append(q=q, k=k, v=k, cache=cache, n=t, **kw):
        MR.qk_norm_rope_append(q, k, v, w, w, cache, pos, idx, idx.data_ptr(), 1, n, None, **kw)

    for bad in (lambda: append(v=k.half()), lambda: append(v=k[:3]), lambda: append(cache=cache[:, :, :, :1]), lambda: append(n=t + 1),
                lambda: append(cache=cache.cpu()), lambda: append(cache=cache.to(torch.float8_e4m3fn)), lambda: append(cache=object())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):  # not planned
        PagedDecodeWrapper(workspace(gpu, 1 << 20), 4, 2, d, 16, device=gpu).qk_norm_rope_set_kv_cache(cache, q, k, k, w, w, pos)
    assert not bool(cache.any())
