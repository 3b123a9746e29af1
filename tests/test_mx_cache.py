"""CPU: the microscaled layer's checks, and the oracle of its formats against torch's own e4m3 cast."""

import pytest
import torch

from mstar_amd.mx_cache import MXKVCache, MXKVLayer
from oracle import microscaled as M


def test_layer_describes_its_tensors():
    c = MXKVCache(3, 5, 32, 2, 128, bits=4, device="cpu")
    assert len(c) == 3 and c.codes.shape == (3, 5, 2, 32, 2, 64) and c.scales.shape == (3, 5, 2, 2, 4, 32)
    layer = c[1]
    assert (layer.bits, layer.head_dim, layer.shape) == (4, 128, (5, 2, 32, 2, 128))
    d = layer.desc
    assert (d.data, d.k_scale, d.v_scale) == (c.codes[1].data_ptr(), c.scales[1].data_ptr(), c.scales[1, 0, 1].data_ptr())
    assert (d.page_stride, d.kv_stride, d.token_stride, d.head_stride) == c.codes.stride()[1:5]
    assert (d.dtype, d.page_size, d.num_kv_heads, d.head_dim, d.max_pages) == (7, 32, 2, 128, 5)
    e = MXKVLayer(torch.zeros(5, 2, 32, 2, 128, dtype=torch.float8_e4m3fn),
                  torch.zeros(5, 2, 2, 4, 32, dtype=torch.uint8).view(torch.float8_e8m0fnu))
    assert (e.bits, e.desc.dtype) == (8, 6)


@pytest.mark.parametrize("codes,scales", [
    ((5, 2, 32, 2, 128), (5, 2, 2, 4, 16)),       # another page size
    ((5, 2, 32, 2, 128), (4, 2, 2, 4, 32)),       # other pages
    ((5, 2, 32, 2, 128), (5, 2, 1, 4, 32)),       # other heads
    ((5, 2, 32, 2, 128), (5, 2, 2, 3, 32)),       # blocks of neither width
    ((5, 2, 32, 2, 128), (5, 2, 2, 2, 32)),       # more than a byte an element
    ((5, 1, 32, 2, 128), (5, 1, 2, 4, 32)),       # no V half
    ((5, 2, 32, 256), (5, 2, 2, 4, 32)),
    ((5, 2, 6, 2, 128), (5, 2, 2, 4, 6)),         # scale words that end inside a page
])
def test_layer_refuses_shapes(codes, scales):
    with pytest.raises(ValueError):
        MXKVLayer(torch.zeros(codes, dtype=torch.uint8), torch.zeros(scales, dtype=torch.uint8))


def test_layer_refuses_types_and_layouts():
    c, s = torch.zeros(5, 2, 32, 2, 128, dtype=torch.uint8), torch.zeros(5, 2, 2, 4, 32, dtype=torch.uint8)
    with pytest.raises(ValueError):
        MXKVLayer(c.to(torch.bfloat16), s)
    with pytest.raises(ValueError):
        MXKVLayer(c, s.float())
    with pytest.raises(ValueError):
        MXKVLayer(c[..., :64].contiguous().view(torch.float8_e4m3fn), s)  # 4 bits are bytes
    with pytest.raises(ValueError):
        MXKVLayer(c, s.transpose(3, 4).contiguous().transpose(3, 4))
    with pytest.raises(ValueError):
        MXKVLayer(torch.zeros(5, 2, 32, 2, 136, dtype=torch.uint8)[..., :128], s)  # rows of 136 bytes
    with pytest.raises(ValueError):
        MXKVLayer(torch.zeros(c.numel() + 8, dtype=torch.uint8)[8:].view(c.shape), s)
    for bad in ({"bits": 6}, {"head_dim": 48}, {"page_size": 20}, {"page_size": 0}):
        with pytest.raises(ValueError):
            MXKVCache(**{"num_layers": 1, "max_pages": 2, "page_size": 16, "num_kv_heads": 1, "head_dim": 64, "device": "cpu",
                         **bad})


def test_oracle_rounds_as_torch_does():
    x = torch.randn(64, 128, generator=torch.Generator().manual_seed(0)) * 50
    codes, scales = M.quantize(x, 8)
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    want = (x.double() / scale).float().clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
    assert torch.equal(codes, want)
    assert (M.values(codes, scales, 8) - x).abs().max() <= (scale * 16).max()


@pytest.mark.parametrize("bits", [8, 4])
def test_oracle_is_nearest(bits):
    """Each code is as near as any, by trying all of them; the scale is the least one allowed."""
    x = torch.randn(4, 64, generator=torch.Generator().manual_seed(1), dtype=torch.float64) * 3
    codes, scales = M.quantize(x, bits)
    grid = (M.E4M3 if bits == 8 else M.E2M1).nan_to_num(nan=1e300)
    scale = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    err = (M.values(codes, scales, bits) - x).abs()
    best = (grid * scale[..., None] - x[..., None]).abs().amin(-1)
    assert torch.equal(err, best)
    peak = x.reshape(4, -1, 32).abs().amax(-1)
    s = torch.exp2(scales.double() - 127)
    assert (peak <= M.LIMIT[bits] * s).all() and (peak > M.LIMIT[bits] * s / 2).all()
