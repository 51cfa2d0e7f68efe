"""4-bit projections (ops.linear_w4) against the formula in 64 bits.

Tolerance per output: its rounding to bf16 (2^-8 relative) plus fp32 accumulation. The products
(q - z) x are exact in fp32; k additions and one scaling per group, each off by at most 2^-23 of
the running sum (tensor-core additions may truncate), bound the accumulation error by
(k + 2 k / group) 2^-23 S with S = sum |(q - z) s x|."""

import pytest
import torch

from helios_b200 import _native, ops
from helios_b200.w4 import W4Weight, dequantize_w4, pack_w4

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def make(m, k, n, group, zeros, seed=0):
    g = torch.Generator().manual_seed(seed + 7 * m + k + n)
    codes = torch.randint(0, 16, (n, k), generator=g)
    scales = (torch.rand(k // group, n, generator=g) * 0.02 + 1e-3).to(torch.bfloat16)
    z = torch.randint(0, 16, (k // group, n), generator=g).to(torch.uint8) if zeros else None
    x = torch.randn(m, k, generator=g).to(torch.bfloat16)
    return x, W4Weight(pack_w4(codes), scales, z)


def expect(x, w):
    values = dequantize_w4(w, torch.float64)
    y = x.double() @ values.t()
    size = x.double().abs() @ values.abs().t()
    k, groups = w.in_features, w.scales.shape[0]
    return y, 2.0 ** -8 * y.abs() + (k + 2 * groups) * 2.0 ** -23 * size


def on_gpu(w):
    return W4Weight(*(None if t is None else t.to(DEV) for t in w))


SHAPES = [
    (1, 32, 1, 32), (1, 128, 16, 128), (2, 96, 17, 32), (3, 64, 15, 64), (7, 320, 33, 64), (8, 2560, 96, 128),
    (9, 384, 1000, 128), (16, 9728, 48, 128), (17, 192, 130, 64), (31, 160, 257, 32), (32, 1024, 64, 128),
    (33, 640, 129, 128), (61, 2560, 200, 64), (64, 512, 128, 32), (65, 256, 131, 128), (128, 1152, 256, 128),
    (130, 288, 385, 32), (257, 448, 140, 64), (509, 2560, 260, 128),
]


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,k,n,group", SHAPES)
def test_matches_the_formula(m, k, n, group, zeros):
    x, w = make(m, k, n, group, zeros)
    y, tol = expect(x, w)
    got = ops.linear_w4(x.to(DEV), *on_gpu(w)).cpu().double()
    assert got.shape == (m, n)
    assert ((got - y).abs() <= tol).all()
    assert _native.device_status() == 0


@pytest.mark.parametrize("m", [1, 8, 40, 200])
def test_exact_integers(m):
    """Small integers: every partial sum is exact in fp32, so the result is the exact sum rounded."""
    g = torch.Generator().manual_seed(m)
    codes = torch.randint(0, 16, (100, 512), generator=g)
    scales = torch.exp2(torch.randint(-2, 3, (4, 100), generator=g).float()).to(torch.bfloat16)
    w = W4Weight(pack_w4(codes), scales, torch.randint(0, 16, (4, 100), generator=g).to(torch.uint8))
    x = torch.randint(-8, 9, (m, 512), generator=g).to(torch.bfloat16)
    want = (x.double() @ dequantize_w4(w, torch.float64).t()).to(torch.bfloat16)
    assert torch.equal(ops.linear_w4(x.to(DEV), *on_gpu(w)).cpu(), want)


@pytest.mark.parametrize("m", [5, 70])
def test_strided_rows_and_given_output(m):
    x, w = make(m, 256, 90, 64, True)
    wide = torch.full((m, 520), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:264] = x.to(DEV)
    out = torch.full((m + 2, 90), 7.0, dtype=torch.bfloat16, device=DEV)
    got = ops.linear_w4(wide[:, 8:264], *on_gpu(w), out=out[1:m + 1])
    assert got.data_ptr() == out[1:].data_ptr()
    assert torch.equal(got, ops.linear_w4(x.to(DEV), *on_gpu(w)))
    assert (out[0] == 7).all() and (out[m + 1] == 7).all()


@pytest.mark.parametrize("m", [6, 80])
def test_bad_values_stay_in_their_row(m):
    x, w = make(m, 256, 40, 128, False)
    clean = ops.linear_w4(x.to(DEV), *on_gpu(w))
    x[2, 11], x[4, 200] = float("inf"), float("nan")
    got = ops.linear_w4(x.to(DEV), *on_gpu(w))
    keep = [r for r in range(m) if r not in (2, 4)]
    assert torch.equal(got[keep], clean[keep])
    assert got[4].isnan().all() and not got[2].isfinite().any()


def test_no_rows():
    _, w = make(1, 128, 24, 128, False)
    assert ops.linear_w4(torch.empty(0, 128, dtype=torch.bfloat16, device=DEV), *on_gpu(w)).shape == (0, 24)


@pytest.mark.parametrize("m", [3, 96])
def test_repeats_streams_and_graphs(m):
    x, w = make(m, 1280, 300, 128, True)
    x, w = x.to(DEV), on_gpu(w)
    first = ops.linear_w4(x, *w)
    for _ in range(5):
        assert torch.equal(ops.linear_w4(x, *w), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.linear_w4(x, *w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first)
    static, graph = x.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops.linear_w4(static, *w)
    static.copy_(-x)
    graph.replay()
    assert torch.equal(captured, ops.linear_w4(-x, *w)) and not torch.equal(captured, first)


def test_refusals():
    x, w = make(2, 256, 16, 128, True)
    x, w = x.to(DEV), on_gpu(w)
    for bad in (lambda: ops.linear_w4(x.float(), *w), lambda: ops.linear_w4(x[:, :128], *w),
                lambda: ops.linear_w4(x, w.packed, w.scales[:, :8], w.zeros),
                lambda: ops.linear_w4(x, w.packed, w.scales, w.zeros[:1]),
                lambda: ops.linear_w4(x, w.packed.cpu(), w.scales, w.zeros),
                lambda: ops.linear_w4(x.t().contiguous().t(), *w),
                lambda: ops.linear_w4(torch.empty(2, 264, dtype=torch.bfloat16, device=DEV)[:, 4:260], *w),
                lambda: ops.linear_w4(x, *w, out=torch.empty(2, 17, dtype=torch.bfloat16, device=DEV))):
        with pytest.raises(ValueError):
            bad()
    assert _native.device_status() == 0
