"""4-bit projections whose weight rows are shared out over two kernels or several rounds: more weight
tiles than SMs, with one token tile (the rows beyond the last whole round run elsewhere) and with
several. Tolerance as in test_gpu_linear_w4, whose formula in 64 bits runs on the device here."""

import pytest
import torch

from helios_b200 import ops
from helios_b200.w4 import W4Weight, dequantize_w4, pack_w4

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("m,k,n,group", [
    (33, 256, 19456, 128), (61, 320, 19456, 64), (64, 96, 19999, 32), (64, 128, 148 * 128, 128),
    (50, 128, 149 * 128 + 1, 128), (40, 128, 37_001, 128), (130, 128, 19457, 128), (65, 64, 19456, 64),
    (64, 9728, 2560, 128), (100, 4096, 2560, 128), (200, 1280, 700, 32),
])
def test_matches_the_formula(m, k, n, group, zeros):
    g = torch.Generator(device=DEV).manual_seed(m + n)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV)
    scales = (torch.rand(k // group, n, generator=g, device=DEV) * 0.02 + 1e-3).to(torch.bfloat16)
    z = torch.randint(0, 16, (k // group, n), generator=g, device=DEV).to(torch.uint8) if zeros else None
    w = W4Weight(pack_w4(codes), scales, z)
    x = torch.randn(m, k, generator=g, device=DEV).to(torch.bfloat16)
    values = dequantize_w4(w, torch.float64)
    y, size = x.double() @ values.t(), x.double().abs() @ values.abs().t()
    tol = 2.0 ** -8 * y.abs() + (k + 2 * k // group) * 2.0 ** -23 * size
    out = torch.full((m + 2, n), 3.0, dtype=torch.bfloat16, device=DEV)
    got = ops.linear_w4(x, *w, out=out[1:m + 1])
    assert ((got.double() - y).abs() <= tol).all()
    assert (out[0] == 3).all() and (out[m + 1] == 3).all()


@pytest.mark.parametrize("m,n", [(1, 512), (8, 512), (12, 512), (96, 512), (61, 19456)])
def test_chains_wait_for_their_inputs(m, n):
    """Twelve projections, each of the one before, into two buffers in turn: queued at once, and
    replayed from a graph, they give what they give one by one."""
    k = 256
    g = torch.Generator(device=DEV).manual_seed(m)
    codes = torch.randint(0, 16, (n, k), generator=g, device=DEV)
    scales = (torch.rand(k // 64, n, generator=g, device=DEV) * 0.02 + 1e-3).to(torch.bfloat16)
    packed = pack_w4(codes)
    start = torch.randn(m, k, generator=g, device=DEV).to(torch.bfloat16)
    buffers = [torch.zeros(m, n, dtype=torch.bfloat16, device=DEV) for _ in range(2)]

    def chain(x, between=lambda: None):
        for i in range(12):
            x = ops.linear_w4(x, packed, scales, None, buffers[i % 2])[:, n - k:]
            between()
        return x.clone()

    want = chain(start, torch.cuda.synchronize)
    assert want.isfinite().all() and want.abs().amax() > 0
    for _ in range(3):
        assert torch.equal(chain(start), want)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = chain(start)
    for _ in range(3):
        for b in buffers:
            b.zero_()
        graph.replay()
        assert torch.equal(got, want)
