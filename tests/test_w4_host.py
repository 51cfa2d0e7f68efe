"""4-bit weights on the host: storage format, quantisation, and the projection's refusals (CPU only)."""

import ctypes

import pytest
import torch

from helios_b200 import _native, ops
from helios_b200.config import Qwen3Config
from helios_b200.model import Qwen3Model
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


def test_overlapping_output_is_refused():
    lib = _native.load()
    base = 1 << 20  # never read: every call here is refused before a launch

    def call(x, out, stride=256, m=2, n=8):
        return lib.hb_linear_w4(ctypes.c_void_p(base + x), stride, m, 256, ctypes.c_void_p(base), ctypes.c_void_p(base),
                                None, n, 128, ctypes.c_void_p(base + out), None)

    for x, out, stride in ((0, 0, 256), (0, 1022, 256), (0, 1534, 512), (30, 0, 256), (16, 0, 256)):
        assert call(x, out, stride) == _native.HB_ERR_INVALID, (x, out)
    assert call(0, 1022) == _native.HB_ERR_INVALID and "overlap" in _native.last_error()


@pytest.mark.parametrize("fault", ["size", "value"])
def test_a_refused_weight_leaves_the_model_as_it_was(fault):
    config = Qwen3Config(vocab_size=64, hidden_size=128, hidden_dim=192 if fault == "size" else 256, n_layers=2,
                         n_heads=2, n_kv_heads=1, head_dim=64, context_length=64)
    model = Qwen3Model(config)
    if fault == "value":
        with torch.no_grad():
            model.blocks[1].feed_forward.down.weight[0, 0] = float("inf")
    with pytest.raises(ValueError):
        model.quantize_weights(128)
    for block in model.blocks:
        assert block.attention.w4_qkv is None and block.feed_forward.w4_down is None
        assert block.attention.output.weight.numel() and block.feed_forward.down.weight.numel()
    if fault == "size":
        model.quantize_weights(64)
        assert all(block.feed_forward.w4_down is not None for block in model.blocks)
