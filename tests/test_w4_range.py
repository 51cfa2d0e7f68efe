"""Weights at the ends of fp32's range through quantize_w4 (CPU only)."""

import pytest
import torch

from helios_b200.w4 import dequantize_w4, quantize_w4


@pytest.mark.parametrize("symmetric", [True, False])
@pytest.mark.parametrize("low,high", [(-3e38, 3e38), (-3.3e38, 0.0), (0.0, 3e38), (-1e-38, 1e-38)])
def test_what_is_accepted_is_represented(low, high, symmetric):
    """Half a step of the scale (the scale's own rounding to bf16 added: 2^-8 of 15 steps), or a refusal."""
    w = (torch.linspace(0, 1, 32, dtype=torch.float64) * (high - low) + low).repeat(2, 1).float()  # a group each
    assert w.isfinite().all()
    try:
        q = quantize_w4(w, 32, symmetric=symmetric)
    except ValueError as refused:
        assert not symmetric and "span" in str(refused) and low < 0 < high
        return
    got = dequantize_w4(q, torch.float64)
    step = q.scales.double().t().repeat_interleave(32, 1)
    assert got.isfinite().all() and ((got - w.double()).abs() <= step * (0.5 + 15 * 2.0 ** -8) + 1e-40).all()
