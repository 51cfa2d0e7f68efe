"""4-bit projections at activations that an ordinary random draw does not have: outliers that the
formula leaves out (their codes equal the zero point), infinities, and the kernel for 9 to 16 rows at
the strides and integers of test_gpu_linear_w4, whose tolerance holds here too."""

import pytest
import torch

from helios_b200 import _native, ops
from helios_b200.w4 import W4Weight, dequantize_w4, pack_w4
from tests.test_gpu_linear_w4 import DEV, expect, make, on_gpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("m", [1, 8, 9, 16, 17, 80])
def test_outliers_at_the_zero_point_leave_no_trace(m, group, zeros):
    """x = 2^15 where every code is the zero point adds (q - z) x = 0, exactly: the error stays within
    what the other products allow."""
    k, n = 384, 272
    x, w = make(m, k, n, group, zeros, seed=3)
    codes = torch.randint(0, 16, (n, k), generator=torch.Generator().manual_seed(m))
    for at in (0, 77, 383):
        codes[:, at] = w.zeros[at // group].int() if zeros else 8
        x[:, at] = 2.0 ** 15 * (-1) ** at
    w = W4Weight(pack_w4(codes), w.scales, w.zeros)
    y, tol = expect(x, w)
    got = ops.linear_w4(x.to(DEV), *on_gpu(w)).cpu().double()
    assert ((got - y).abs() <= tol).all()
    assert _native.device_status() == 0


@pytest.mark.parametrize("m", [3, 12, 40, 200])
def test_infinities_give_what_the_formula_gives(m):
    """(q - z) x is an infinity of the product's sign, or NaN where q = z."""
    x, w = make(m, 256, 60, 64, True)
    x[0, 11], x[1, 200], x[2, 3] = float("inf"), -float("inf"), float("inf")
    x[2, 130] = -float("inf")
    want = (x.double().unsqueeze(1) * dequantize_w4(w, torch.float64)).sum(-1)
    got = ops.linear_w4(x.to(DEV), *on_gpu(w)).cpu().double()
    assert want[0].isinf().any() and want[0].isnan().any()
    assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got[want.isinf()], want[want.isinf()])


def test_ring_kernel_exact_integers():
    """12 rows: small integers, every partial sum exact in fp32, the result the exact sum rounded."""
    g = torch.Generator().manual_seed(12)
    codes = torch.randint(0, 16, (100, 1280), generator=g)
    scales = torch.exp2(torch.randint(-2, 3, (10, 100), generator=g).float()).to(torch.bfloat16)
    w = W4Weight(pack_w4(codes), scales, torch.randint(0, 16, (10, 100), generator=g).to(torch.uint8))
    x = torch.randint(-8, 9, (12, 1280), generator=g).to(torch.bfloat16)
    want = (x.double() @ dequantize_w4(w, torch.float64).t()).to(torch.bfloat16)
    assert torch.equal(ops.linear_w4(x.to(DEV), *on_gpu(w)).cpu(), want)


def test_ring_kernel_strided_rows_and_bad_values():
    x, w = make(12, 256, 90, 64, True)
    wide = torch.full((12, 520), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:264] = x.to(DEV)
    out = torch.full((14, 90), 7.0, dtype=torch.bfloat16, device=DEV)
    clean = ops.linear_w4(x.to(DEV), *on_gpu(w))
    assert torch.equal(ops.linear_w4(wide[:, 8:264], *on_gpu(w), out=out[1:13]), clean)
    assert (out[0] == 7).all() and (out[13] == 7).all()
    x[2, 11], x[4, 200] = float("inf"), float("nan")
    got = ops.linear_w4(x.to(DEV), *on_gpu(w))
    keep = [r for r in range(12) if r not in (2, 4)]
    assert torch.equal(got[keep], clean[keep])
    assert got[4].isnan().all() and not got[2].isfinite().any()
