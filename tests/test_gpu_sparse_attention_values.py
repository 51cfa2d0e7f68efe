"""Sparse decode attention: the weights' rounding, infinite bounds, and rows and block counts beyond
those of test_gpu_sparse_attention, whose definition, selection and attention check are used here."""

import math

import pytest
import torch

from helios_b200 import _native, ops
from tests.test_gpu_sparse_attention import BLOCK, DEV, PAGE, check, pool, table, whole_bounds

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("group", [1, 2, 4, 8])
@pytest.mark.parametrize("lengths", [[2, 3, 5, 9, 40], [65, 130], [700, 1500, 3]])
def test_weights_keep_more_than_sixteen_bits(lengths, group):
    """A weight w is held in two bf16 values, 2^-16 w apart from it at most (each rounding is off by at
    most 2^-8 of what it rounds). With the scores' error d and the exponential's as derived in
    test_gpu_sparse_attention, an output is off by (2^-16 + 2 d) sum w |v| and its own rounding,
    2^-8 |y|. Rows of few keys, whose values cancel, tell the weights' rounding from the output's."""
    keys, values, g = pool(sum(-(-n // PAGE) for n in lengths) + 1, 2, 21)
    bt = table(lengths, keys.shape[0], g)
    q = torch.randn(len(lengths), 2 * group, 128, generator=g).to(torch.bfloat16)
    scale, top = 0.02, 4
    used = torch.tensor(lengths, dtype=torch.int32)
    selected = torch.empty(len(lengths), 2, top, dtype=torch.int32, device=DEV)
    got = ops.sparse_paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), whole_bounds(keys).to(DEV), bt.to(DEV),
                                     used.to(DEV), top_blocks=top, scale=scale, selected=selected).cpu().double()
    for row, length in enumerate(lengths):
        for h in range(2):
            blocks = [b for b in selected[row, h].tolist() if b >= 0]
            at = torch.cat([torch.arange(b * BLOCK, min(length, b * BLOCK + BLOCK)) for b in blocks])
            page = bt[row].long()[at // PAGE]
            k, v = keys[page, at % PAGE, h].double(), values[page, at % PAGE, h].double()
            query = q[row, h * group:(h + 1) * group].double()
            w = torch.softmax(query @ k.t() * scale, -1)
            y = w @ v
            d = scale * 130 * 2.0 ** -23 * (query.abs() @ k.abs().t()).amax(-1, keepdim=True) + 2.0 ** -20
            tol = (2.0 ** -16 + 2 * d) * (w @ v.abs()) + 2.0 ** -8 * y.abs()
            assert ((got[row, h * group:(h + 1) * group] - y).abs() <= tol).all()
    assert _native.device_status() == 0


