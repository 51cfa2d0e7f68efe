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


def ranked(q, bounds, bt, length, top, sink=1, recent=2):
    """The definition's blocks of one (row, KV head), with max(q lo, q hi) taken as it is written."""
    count = -(-length // BLOCK)
    flat = torch.stack([bounds[int(bt[b // 4]), b % 4] for b in range(count)]).double()
    q = q.double().unsqueeze(1)
    score = torch.maximum(q * flat[:, 0], q * flat[:, 1]).sum(-1)
    worst = score.isnan().any(0)
    best = score.nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).amax(0)
    forced = set(range(sink)) | set(range(count - recent, count))
    free = sorted(set(range(count)) - forced, key=lambda b: (not bool(worst[b]), -float(best[b]), b))
    return sorted(forced | set(free[:top - len(forced)]))


@pytest.mark.parametrize("group", [1, 4])
@pytest.mark.parametrize("low,high,first", [(-math.inf, None, 0.5), (None, math.inf, -0.5), (-math.inf, math.inf, 0.5),
                                            (-math.inf, None, 0.0), (-math.inf, None, -0.5), (None, math.inf, 0.5),
                                            (-math.inf, -math.inf, 0.5)])
def test_infinite_bounds_rank_as_the_formula_says(low, high, first, group):
    """An infinite minimum beside a positive query (an infinite maximum beside a negative one) leaves
    max(q lo, q hi) finite: the block ranks by it. Beside a zero it is NaN, which ranks first."""
    keys, values, g = pool(10, 2, 12)
    bt = table([2500], 10, g)
    q = torch.randn(1, 2 * group, 128, generator=g).to(torch.bfloat16)
    q[:, :, 3] = first
    bounds = whole_bounds(keys)
    for block in (5, 9, 18, 30):
        at = bounds[int(bt[0, block // 4]), :, block % 4, :, 3]
        if low is not None:
            at[:, 0] = low
        if high is not None:
            at[:, 1] = high
    selected = torch.empty(1, 2, 9, dtype=torch.int32, device=DEV)
    ops.sparse_paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), bounds.to(DEV), bt.to(DEV),
                               torch.tensor([2500], dtype=torch.int32, device=DEV), top_blocks=9, selected=selected)
    for h in range(2):
        want = ranked(q[0, h * group:(h + 1) * group], bounds[:, h], bt[0], 2500, 9)
        assert selected[0, h].tolist() == want
    assert _native.device_status() == 0


@pytest.mark.parametrize("length,top", [(40_961, 20), (41_000, 32), (100_000, 40)])
def test_rows_beyond_the_registers_of_the_selection(length, top):
    """More than 640 blocks: the selection reads its keys from shared memory."""
    pages = -(-length // PAGE) + 1
    keys, values, g = pool(pages, 1, 31)
    bt = table([length], pages, g)
    q = torch.randn(1, 4, 128, generator=g).to(torch.bfloat16)
    bounds = whole_bounds(keys)
    check(q, keys, values, bounds, bt, [length], top)
    # Ties at the cut: every score equal, then one block ahead and one behind.
    bounds[:] = bounds[:1, :, :1]
    check(q, keys, values, bounds, bt, [length], top)
    bounds[int(bt[0, 70]), :, 2, 1] += 1
    bounds[int(bt[0, 11]), :, 1, 1] -= 1
    check(q, keys, values, bounds, bt, [length], top)
    assert _native.device_status() == 0


@pytest.mark.parametrize("length,top", [(70_000, 1024), (60_000, 1024), (20_000, 200)])
def test_many_blocks(length, top):
    pages = -(-length // PAGE) + 1
    keys, values, g = pool(pages, 1, 32)
    bt = table([length], pages, g)
    q = torch.randn(1, 2, 128, generator=g).to(torch.bfloat16)
    check(q, keys, values, whole_bounds(keys), bt, [length], top)


def test_the_widest_table():
    """1,536 pages of 256 tokens, most of them one and the same."""
    pages, length = 40, 1536 * 256
    keys, values, g = pool(pages, 1, 33)
    bt = torch.randint(0, pages, (1, 1536), generator=g).int()
    q = torch.randn(1, 1, 128, generator=g).to(torch.bfloat16)
    check(q, keys, values, whole_bounds(keys), bt, [length], 24)
    assert _native.device_status() == 0
