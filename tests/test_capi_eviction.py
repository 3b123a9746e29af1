"""Normed rotation, attention weights and eviction without a GPU: arguments are checked before any HIP call."""

import ctypes

import pytest
import torch

from mstar_amd import _lib
from mstar_amd.eviction import evict_kv_cache, kv_weights
from mstar_amd.mx_cache import MXKVCache

INVALID, UNSUPPORTED, WORKSPACE = -1, -2, -3


@pytest.fixture(scope="module")
def L():
    return _lib.lib()


@pytest.fixture(scope="module")
def mem():
    buf = (ctypes.c_int32 * 64)()
    base = (ctypes.addressof(buf) + 15) // 16 * 16
    return buf, ctypes.c_void_p(base), ctypes.c_void_p(base + 2)


def _kv(**kw):
    d = _lib.MiPagedKV()
    d.data, d.dtype, d.page_size, d.num_kv_heads, d.head_dim = 4096, 0, 16, 4, 128
    d.page_stride, d.kv_stride, d.token_stride, d.head_stride = 2 * 16 * 4 * 128, 16 * 4 * 128, 4 * 128, 128
    d.max_pages = 64
    for k, v in kw.items():
        setattr(d, k, v)
    return ctypes.byref(d)


def _mx(dtype=6, **kw):
    return _kv(**{"dtype": dtype, "k_scale": 8192, "v_scale": 8192 + 4 * 4 * 16, **kw})


def test_qk_norm_rope_arguments(L, mem):
    _, p, odd = mem

    def call(q=p, k=p, v=p, dt=0, d=128, qw=p, wd=0, eps=1e-6, kv=None, idx=p, stride=1, append=3, rd=128, pos=p, pdt=5, n=3, il=0, scale=1.0,
             theta=1e4, l31=(0, 1.0, 4.0), qs=512, hk=4):
        return L.mi_qk_norm_rope(q, qs, 128, 4, k, 512, 128, hk, v, 512, 128, dt, d, qw, p, wd, eps, 1, kv, idx, idx, stride, append, None,
                                 rd, pos, pdt, n, il, scale, theta, l31[0], l31[1], l31[2], 8192.0, None)

    assert call(n=0) == 0
    for bad in (dict(n=-1), dict(q=None), dict(k=None), dict(qw=None), dict(pos=None), dict(eps=-1.0), dict(eps=float("nan")), dict(scale=0.0),
                dict(theta=0.0), dict(l31=(1, 4.0, 1.0)), dict(l31=(1, 0.0, 1.0)), dict(q=odd), dict(qs=516), dict(append=-1)):
        assert call(**bad) == INVALID, bad
    for bad in (dict(dt=2), dict(wd=1), dict(pdt=0), dict(d=100, rd=96), dict(d=520), dict(rd=24), dict(rd=0), dict(rd=144), dict(rd=12, il=1)):
        assert call(**bad) == UNSUPPORTED, bad
    for bad in (dict(v=None), dict(idx=None), dict(stride=0), dict(append=4), dict(hk=2), dict(v=odd), dict(kv=_kv(data=4100)),
                dict(kv=_kv(token_stride=516)), dict(kv=_kv(dtype=3)), dict(kv=_mx(k_scale=8194)), dict(kv=_kv(page_size=0)),
                dict(kv=_kv(head_dim=64)), dict(kv=_mx(head_stride=136))):
        assert call(**{"kv": _kv(), **bad}) == INVALID, bad
    assert call(kv=_kv(dtype=9)) == UNSUPPORTED
    assert call(d=80, rd=80, kv=_mx(head_dim=80)) == UNSUPPORTED  # blocks of 32


def test_attention_weights_arguments(L, mem):
    _, p, odd = mem

    def call(q=p, dt=0, kv=None, qo=p, ip=p, batch=4, most=64, entries=32, hq=32, parts=3, w=p, ws=p, nbytes=1 << 30, qs=4096):
        return L.mi_attention_weights(q, dt, qs, 128, kv or _kv(), qo, ip, p, p, batch, most, entries, hq, 1, 0.1, parts, w, ws, nbytes, None)

    for none in (dict(batch=0), dict(most=0), dict(entries=0)):
        assert call(**none) == 0, none
    for bad in (dict(batch=-1), dict(most=-1), dict(entries=-1), dict(parts=0), dict(parts=4), dict(hq=30), dict(q=None), dict(ip=None),
                dict(w=None), dict(ws=None), dict(q=odd), dict(qs=4100), dict(w=odd), dict(ws=odd), dict(kv=_kv(dtype=3)), dict(kv=_kv(data=4104)),
                dict(kv=_kv(head_stride=132)), dict(kv=_mx(k_scale=8194)), dict(kv=_kv(page_size=0)), dict(kv=_kv(num_kv_heads=0))):
        assert call(**bad) == INVALID, bad
    for bad in (dict(hq=128), dict(kv=_kv(page_size=24)), dict(kv=_kv(head_dim=96)), dict(dt=4), dict(kv=_kv(dtype=1)), dict(dt=2),
                dict(dt=2, kv=_mx()), dict(entries=1 << 27), dict(most=1 << 28), dict(kv=_kv(page_size=1 << 25))):
        assert call(**bad) == UNSUPPORTED, bad
    need = L.mi_attention_weights_bytes(4, 64, 32, 16, 32, 4, 1, 3)
    assert call(nbytes=need - 1) == WORKSPACE


def test_attention_weights_bytes(L):
    size = L.mi_attention_weights_bytes
    # a score of every place, kv head and row at least, where they do not fit a workgroup
    assert size(4, 4, 1000, 16, 32, 4, 0, 1) >= 4 * 16000 * 32
    assert size(4, 4, 60, 16, 32, 4, 0, 1) == 0
    for entries in (60, 1000):
        assert size(4, 4, entries, 16, 32, 4, 0, 3) == size(4, 4, entries, 16, 32, 4, 0, 1)  # one query each: all are short
    assert size(4, 400, 100, 16, 32, 4, 1, 3) > size(4, 400, 100, 16, 32, 4, 1, 1)
    assert size(4, 400, 100, 16, 32, 4, 1, 2) >= 4 * 400 * 32
    assert size(0, 0, 0, 16, 32, 4, 1, 3) >= 0
    for bad in ((-1, 4, 4, 16, 32, 4, 1, 3), (4, 4, 4, 16, 30, 4, 1, 3), (4, 4, 4, 0, 32, 4, 1, 3), (4, 4, 4, 16, 32, 4, 1, 0)):
        assert size(*bad) == INVALID


def test_argument_blocks(L):
    for name, fmt in (("mi_qk_norm_rope_block", _lib.QK_NORM_ROPE_ARGS), ("mi_attention_weights_block", _lib.ATTENTION_WEIGHTS_ARGS),
                      ("mi_kv_evict_block", _lib.KV_EVICT_ARGS)):
        assert getattr(L, name)(None) == INVALID
        zeros = getattr(L, name)(bytes(fmt.size))  # no tokens to rotate; no layer for the others
        assert zeros == (0 if name == "mi_qk_norm_rope_block" else INVALID)


def test_kv_evict_arguments(L, mem):
    _, p, odd = mem

    def call(kv=None, layers=2, stride=1 << 16, w=p, out=p, wstride=4096, ip=p, batch=3, entries=32, keep=20, recent=4, sinks=2, kept=p):
        return L.mi_kv_evict(kv or _kv(), layers, stride, 0, w, out, wstride, ip, p, p, batch, entries, keep, recent, sinks, kept, None)

    assert call(batch=0) == 0 and call(layers=0) == 0
    for bad in (dict(batch=-1), dict(layers=-1), dict(entries=-1), dict(keep=0), dict(keep=-3), dict(recent=-1), dict(sinks=-1),
                dict(recent=19, sinks=2), dict(recent=2 ** 31 - 1, sinks=2 ** 31 - 1, keep=2 ** 31 - 1), dict(w=None), dict(out=None), dict(ip=None), dict(kept=None), dict(w=odd), dict(out=odd),
                dict(wstride=4098), dict(stride=(1 << 16) + 4), dict(kv=_kv(data=4104)), dict(kv=_kv(token_stride=516)), dict(kv=_kv(data=None)),
                dict(kv=_mx(k_scale=None)), dict(kv=_mx(v_scale=8192 + 64))):
        assert call(**bad) == INVALID, bad
    for bad in (dict(kv=_kv(dtype=9)), dict(kv=_kv(head_dim=96)), dict(kv=_kv(page_size=18)), dict(kv=_kv(page_size=1 << 25)),
                dict(entries=1 << 27), dict(batch=1 << 30)):
        assert call(**bad) == UNSUPPORTED, bad


def test_python_refusals_without_a_gpu():
    cache = torch.zeros(2, 4, 2, 16, 1, 64, dtype=torch.bfloat16)
    w = kv_weights(cache)
    assert w.shape == (2, 4, 1, 16) and kv_weights(cache[0]).shape == (4, 1, 16)
    mx = MXKVCache(3, 4, 16, 2, 64, bits=4, device="cpu")
    assert kv_weights(mx).shape == (3, 4, 2, 16) and kv_weights(mx[1]).shape == (4, 2, 16)
    idx = (torch.tensor([0, 1]), torch.tensor([0]), torch.tensor([3]))
    with pytest.raises(ValueError):
        evict_kv_cache(cache, w, *idx, keep=4)  # not on a GPU
    for bad in (cache[0, 0], cache.transpose(2, 3), object()):
        with pytest.raises(ValueError):
            kv_weights(bad)
