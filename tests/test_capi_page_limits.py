"""Pages whose slots' offsets pass 32 bits, without a GPU: the kernels that count them in 32 bits refuse the layer."""

import ctypes

import pytest

from mstar_amd import _lib

UNSUPPORTED, WORKSPACE = -2, -3


@pytest.fixture(scope="module")
def call():
    L = _lib.lib()
    buf = (ctypes.c_int32 * 64)()
    p = ctypes.c_void_p((ctypes.addressof(buf) + 15) // 16 * 16)

    def run(window, dtype=0, q_dtype=0, ws=64, **kw):
        d = _lib.MiPagedKV()
        d.data, d.dtype, d.page_size, d.num_kv_heads, d.head_dim, d.max_pages = 4096, dtype, 16, 4, 128, 4
        d.page_stride, d.kv_stride, d.token_stride, d.head_stride = 1 << 20, 1 << 16, 512, 128
        d.k_scale, d.v_scale = (8192, 16384) if dtype in (3, 6, 7) else (None, None)
        for k, v in kw.items():
            setattr(d, k, v)
        kv = ctypes.byref(d)
        head = (p, q_dtype, 4096, 128, kv, None, p, p, p, 4, 32, 0, 0.1)
        tail = (p, ws, p, 4096, 128, None)
        return L.mi_decode_run_window(*head, 5, 0, *tail) if window else L.mi_decode_run(*head, *tail)

    run.keep = buf
    return run


@pytest.mark.parametrize("window", [True, False])
@pytest.mark.parametrize("dtype,size", [(0, 2), (3, 1), (6, 1), (7, 1)])
def test_pages_of_4_gib(call, window, dtype, size):
    """A token-major pool's stride, say: the last slot of a page lies past 2^32 bytes behind its first."""
    most = (1 << 32) // size // 16
    assert call(window, dtype, token_stride=most) == UNSUPPORTED
    assert call(window, dtype, token_stride=most - 16) == WORKSPACE  # the next check: this layer passes
    assert call(window, dtype, page_size=128, token_stride=most // 8) == UNSUPPORTED
    for stride in (-512, 1 << 40, (1 << 62) + 16):
        assert call(window, dtype, token_stride=stride) == UNSUPPORTED


@pytest.mark.parametrize("window", [True, False])
def test_pages_of_many_tokens(call, window):
    assert call(window, 7, page_size=(1 << 24) + 16, token_stride=32) == UNSUPPORTED
    assert call(window, 7, page_size=1 << 24, token_stride=32) == WORKSPACE


def test_fp32_counts_pages_in_64_bits(call):
    assert call(False, 2, 2, page_size=128, token_stride=1 << 25) == WORKSPACE
    assert call(False, 2, 2, token_stride=1 << 26) == UNSUPPORTED  # 16 tokens of 2^28 bytes
