"""4-bit weights on the host: storage format, quantisation, and the projection's refusals (CPU only)."""

import ctypes

import pytest
import torch

from helios_b200 import _native, ops
from helios_b200.w4 import dequantize_w4, pack_w4, quantize_w4, unpack_w4


def test_pack_layout_and_round_trip():
    codes = torch.arange(16).repeat(3, 4)[:, :40].contiguous()
    codes[1] = codes[1].flip(0)
    packed = pack_w4(codes)
    assert packed.shape == (3, 5) and torch.equal(unpack_w4(packed), codes.int())
    # Word 0 of row 0 holds k = 0..7 with codes 0..7: even k's low half, odd k's high half.
    assert packed[0, 0].item() & 0xFFFFFFFF == 0x7531_6420
    assert torch.equal(unpack_w4(pack_w4(torch.full((2, 8), 15))), torch.full((2, 8), 15, dtype=torch.int32))
    with pytest.raises(ValueError, match="multiple of 8"):
        pack_w4(torch.zeros(2, 12))


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantisation_is_nearest(group, symmetric):
    g = torch.Generator().manual_seed(group)
    w = torch.randn(24, 256, generator=g) * 0.05
    w[3] = 0
    w[4, :group] = w[4, :group].abs()  # a group of one sign
    q = quantize_w4(w, group, symmetric=symmetric)
    assert q.scales.shape == (256 // group, 24) and (q.zeros is None) == symmetric
    assert q.in_features == 256 and q.out_features == 24
    back = dequantize_w4(q, torch.float64)
    step = q.scales.t().double().repeat_interleave(group, 1)
    # Half a step inside the codes' range. The scale's rounding to bf16 (2^-8) can leave the
    # group's extremes outside it by 15 steps x 2^-8 at most; an asymmetric zero point is rounded
    # too (half a step), which shifts the range's ends by as much.
    slack = 0.5 + 15 / 256 + (0 if symmetric else 0.5)
    assert ((back - w.double()).abs() <= slack * step + 1e-12).all()
    assert (back[3] == 0).all()


def test_quantisation_refusals():
    with pytest.raises(ValueError, match="divide"):
        quantize_w4(torch.zeros(4, 96), 64)
    with pytest.raises(ValueError, match="one of"):
        quantize_w4(torch.zeros(4, 96), 48)
    with pytest.raises(ValueError, match="finite"):
        quantize_w4(torch.full((4, 64), float("nan")), 64)


def test_projection_refusals():
    lib = _native.load()
    p = ctypes.c_void_p(4096)  # never read: every call here is refused before a launch

    def call(x_stride=256, m=2, k=256, n=8, group=128, x=p, packed=p):
        return lib.hb_linear_w4(x, x_stride, m, k, packed, p, None, n, group, p, None)

    assert call(group=48) == _native.HB_ERR_UNSUPPORTED and "32, 64 or 128" in _native.last_error()
    assert call(k=192, x_stride=192) == _native.HB_ERR_INVALID
    assert call(x_stride=128) == _native.HB_ERR_INVALID
    assert call(x_stride=257) == _native.HB_ERR_INVALID and "16-byte" in _native.last_error()
    assert call(x=None) == _native.HB_ERR_INVALID
    assert call(packed=ctypes.c_void_p(4100)) == _native.HB_ERR_INVALID
    assert call(n=0) == _native.HB_ERR_INVALID and call(m=-1) == _native.HB_ERR_INVALID
    assert call(m=0) == _native.HB_OK
    w = quantize_w4(torch.ones(8, 128))
    with pytest.raises(ValueError, match="CUDA"):
        ops.linear_w4(torch.zeros(2, 128, dtype=torch.bfloat16), *w)
