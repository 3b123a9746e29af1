"""The windowed, microscaled and read entry points without a GPU: arguments are checked before any HIP call."""

import ctypes

import pytest
import torch

from mstar_amd import _lib
from mstar_amd.kv_transfer import CPUPagePool, pool_desc
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
    return _kv(**{"dtype": dtype, "k_scale": 8192, "v_scale": 16384, **kw})


def test_decode_window_arguments(L, mem):
    _, p, odd = mem

    def call(kv=None, q=p, dt=0, left=5, sinks=0, batch=4, hq=32, ws=1 << 26, out=p):
        return L.mi_decode_run_window(q, dt, 4096, 128, kv or _kv(), None, p, p, p, batch, hq, 0, 0.1, left, sinks, p, ws, out,
                                      4096, 128, None)

    assert call(batch=0) == 0
    assert call(sinks=-1) == INVALID
    assert call(batch=-1) == INVALID
    assert call(q=odd) == INVALID
    assert call(out=None) == INVALID
    assert call(hq=30) == INVALID
    assert call(hq=128) == UNSUPPORTED                                 # 32 q-heads a kv-head
    assert call(dt=2, kv=_kv(dtype=2)) == UNSUPPORTED                  # fp32 has no windowed kernels
    assert call(kv=_kv(dtype=1)) == UNSUPPORTED                        # bf16 q over an fp16 cache
    assert call(kv=_kv(page_size=24)) == UNSUPPORTED
    assert call(kv=_kv(head_dim=96)) == UNSUPPORTED
    assert call(ws=4096) == WORKSPACE
    for dt in (3, 6, 7):
        assert call(kv=_kv(dtype=dt)) == INVALID                       # no scales
    assert call(kv=_mx(k_scale=8194)) == INVALID                       # scale words off their alignment
    assert call(kv=_mx(head_stride=72)) == INVALID                     # rows off theirs


def test_prefill_window_arguments(L, mem):
    _, p, odd = mem

    def call(kv=None, q=p, dt=0, left=5, sinks=0, parts=3, batch=4, ws=1 << 26):
        return L.mi_prefill_run_window(q, dt, 4096, 128, kv or _kv(), p, p, p, p, batch, 64, 32, 1, 0.1, left, sinks, parts, p,
                                       ws, p, 4096, 128, None)

    assert call(batch=0) == 0
    assert call(sinks=-1) == INVALID
    for parts in (0, 4, -1):
        assert call(parts=parts) == INVALID
    assert call(q=odd) == INVALID
    assert call(dt=2, kv=_kv(dtype=2)) == UNSUPPORTED
    assert call(kv=_mx(dtype=7, v_scale=None)) == INVALID
    assert call(ws=1024) == WORKSPACE


def test_append_into_a_microscaled_layer(L, mem):
    _, p, odd = mem

    def call(kv, n=3, k_stride=512, src=0):
        return L.mi_kv_append(kv, p, p, src, k_stride, 128, 512, 128, p, p, 1, n, None, None)

    assert call(_mx(), n=0) == 0
    assert call(_kv(dtype=7)) == INVALID                               # no scales
    assert call(_mx(v_scale=16386)) == INVALID
    assert call(_mx(head_dim=80)) == UNSUPPORTED                       # no whole blocks
    assert call(_mx(token_stride=520)) == INVALID
    assert call(_mx(data=4104)) == INVALID
    assert call(_mx(), k_stride=516) == INVALID
    assert call(_mx(), src=6) == UNSUPPORTED                           # codes are no source
    assert call(_kv(dtype=9)) == UNSUPPORTED


def test_rope_append_refuses_a_microscaled_layer(L, mem):
    _, p, _ = mem
    assert L.mi_rope_append(p, 512, 128, 4, p, 256, 128, p, 256, 128, 0, 1, _mx(num_kv_heads=2), p, p, 1, 3, None, 128, p, 5, 3,
                            0, 1.0, 1e4, 0, 1.0, 4.0, 8192.0, None) == UNSUPPORTED


def test_read_arguments(L, mem):
    _, p, odd = mem

    def call(kv=None, batch=2, n=4, k=p, v=p, dt=0, tokens=8, indptr=p):
        return L.mi_kv_read(kv or _mx(), indptr, p, p, batch, n, k, v, dt, tokens, None)

    assert call(batch=0) == call(n=0) == call(tokens=0) == 0           # nothing to do
    for kw in ({"batch": -1}, {"n": -1}, {"tokens": -1}, {"k": None}, {"v": None}, {"k": odd}, {"indptr": None},
               {"kv": _kv(dtype=3)}, {"kv": _mx(k_scale=None)}, {"kv": _mx(data=4104)}, {"kv": _mx(num_kv_heads=0)}):
        assert call(**kw) == INVALID, kw
    assert L.mi_kv_read(None, p, p, p, 2, 4, p, p, 0, 8, None) == INVALID
    assert call(kv=_mx(head_dim=80)) == UNSUPPORTED
    assert call(kv=_kv(page_size=1 << 20, num_kv_heads=64, head_dim=256)) == UNSUPPORTED  # a page of 2^34 elements
    assert call(kv=_kv(dtype=9)) == UNSUPPORTED
    for dt in (3, 6, 9):
        assert call(dt=dt) == UNSUPPORTED


def test_transfers_refuse_a_microscaled_pool():
    pool = MXKVCache(1, 4, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError):
        pool_desc(pool)

    class Pages:
        def try_allocate(self, n):
            raise AssertionError("pages were taken before the check")

    cpu = CPUPagePool.__new__(CPUPagePool)
    cpu.page_allocator = Pages()
    with pytest.raises(ValueError):
        cpu.offload_pages("r", "main", pool, [1, 2], 20, 20)


def test_gather_needs_a_gpu():
    from mstar_amd.mx_cache import read_kv_cache

    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError):
        read_kv_cache(MXKVCache(1, 4, 16, 1, 64, device="cpu")[0], z, z, torch.empty(0, dtype=torch.int32), 0)
