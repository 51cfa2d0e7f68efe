"""Key block bounds and sparse decode attention against their definitions in 64 bits.

Bounds are minima and maxima of stored values: they have to be equal. So do the selected blocks:
scores are compared exactly, whatever their magnitude. Attention tolerance per output, with
weights w (summing to 1) and A = sum w |v|: the weights are rounded to bf16 for the product with V
(2^-8 A), a score's fp32 error d = scale * 130 * 2^-23 * sum |q k| (128 exact products added in
fp32, then scaled) and 2^-20 for the exponential move every weight by a relative d + 2^-20 at
most, twice through the normalisation, and the output is rounded once (2^-8 |y|)."""

import math

import pytest
import torch

from helios_b200 import _native, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")
PAGE, BLOCK = 256, 64


def pool(pages, heads, seed, page=PAGE):
    g = torch.Generator().manual_seed(seed)
    keys = torch.randn(pages, page, heads, 128, generator=g)
    keys = keys + torch.randn(pages, page // BLOCK, 1, heads, 128, generator=g).repeat_interleave(BLOCK, 1).view(keys.shape)
    values = torch.randn(pages, page, heads, 128, generator=g)
    return keys.to(torch.bfloat16), values.to(torch.bfloat16), g


def table(lengths, pages, g, page=PAGE, width=None):
    order = torch.randperm(pages, generator=g).tolist()
    need = [-(-length // page) for length in lengths]
    out = torch.zeros(len(lengths), width or max(1, *need), dtype=torch.int32)
    for row, n in enumerate(need):
        for j in range(n):
            out[row, j] = order.pop()
    return out


def whole_bounds(keys):
    pages, page, heads, _ = keys.shape
    blocks = keys.view(pages, page // BLOCK, BLOCK, heads, 128)
    return torch.stack((blocks.amin(2), blocks.amax(2)), 3).permute(0, 2, 1, 3, 4).contiguous()


# ---------------------------------------------------------------- bounds
def tick(lengths, counts):
    cu = torch.tensor([0] + list(counts)).cumsum(0).int()
    rows = torch.repeat_interleave(torch.arange(len(counts)), torch.tensor(counts)).int()
    return cu, torch.tensor(lengths, dtype=torch.int32), rows


@pytest.mark.parametrize("heads,page", [(1, 256), (2, 64), (8, 256), (12, 512)])
@pytest.mark.parametrize("lengths,counts", [
    ([1], [1]), ([64], [1]), ([65], [1]), ([64], [64]), ([200], [200]), ([300], [100]),
    ([5, 700, 129, 64, 513], [1, 1, 65, 64, 300]), ([900, 31, 257], [900, 2, 1]),
])
def test_bounds_of_touched_blocks(lengths, counts, heads, page):
    pages = sum(-(-n // page) for n in lengths) + 2
    keys, _, g = pool(pages, heads, 5, page)
    bt = table(lengths, pages, g, page)
    start = torch.full((pages, heads, page // BLOCK, 2, 128), 99.0, dtype=torch.bfloat16)
    want = start.clone()
    for row, (length, count) in enumerate(zip(lengths, counts)):
        for block in range((length - count) // BLOCK, (length - 1) // BLOCK + 1):
            first = block * BLOCK
            p, at = int(bt[row, first // page]), first % page
            part = keys[p, at:at + min(BLOCK, length - first)]
            want[p, :, at // BLOCK, 0], want[p, :, at // BLOCK, 1] = part.amin(0), part.amax(0)
    cu, used, token_row = tick(lengths, counts)
    got = start.to(DEV)
    assert ops.key_block_bounds(keys.to(DEV), got, bt.to(DEV), cu.to(DEV), used.to(DEV), token_row.to(DEV)) is got
    assert torch.equal(got.cpu(), want)
    assert _native.device_status() == 0


def test_bounds_carry_nan_and_ignore_keys_past_the_row():
    keys, _, _ = pool(2, 2, 1)
    keys[1, 70, 0, 3] = float("nan")
    keys[1, 71, 1, 4] = float("inf")
    keys[1, 80:] = float("nan")  # left by an earlier owner of the page
    cu, used, token_row = tick([80], [1])
    bt = torch.tensor([[1]], dtype=torch.int32)
    got = torch.zeros(2, 2, 4, 2, 128, dtype=torch.bfloat16, device=DEV)
    ops.key_block_bounds(keys.to(DEV), got, bt.to(DEV), cu.to(DEV), used.to(DEV), token_row.to(DEV))
    got = got.cpu()
    assert got[1, 0, 1, :, 3].isnan().all() and got[1].isnan().sum() == 2
    assert got[1, 1, 1, 1, 4] == float("inf") and (got[1, :, 0] == 0).all() and (got[0] == 0).all()


def test_bounds_flag_pages_outside_the_pool():
    keys, _, _ = pool(2, 2, 1)
    cu, used, token_row = tick([10, 20], [1, 1])
    bt = torch.tensor([[7], [1]], dtype=torch.int32)
    got = torch.zeros(2, 2, 4, 2, 128, dtype=torch.bfloat16, device=DEV)
    ops.key_block_bounds(keys.to(DEV), got, bt.to(DEV), cu.to(DEV), used.to(DEV), token_row.to(DEV))
    assert _native.device_status() == 1 << 3
    assert (got[0] == 0).all() and (got[1, :, 0] != 0).any()


# ---------------------------------------------------------------- selection and attention
def select(q, bounds, bt, length, top, sink, recent, page=PAGE):
    """Blocks of one (row, KV head): q [group, 128] and bounds [pages, blocks per page, 2, 128]."""
    count = max(0, -(-length // BLOCK))
    if count <= top:
        return list(range(count))
    per_page = page // BLOCK
    flat = torch.stack([bounds[int(bt[b // per_page]), b % per_page] for b in range(count)]).double()
    q = q.double()
    score = (q.clamp(max=0) @ flat[:, 0].t() + q.clamp(min=0) @ flat[:, 1].t())
    score = torch.where(score.isnan().any(0), math.inf, score.nan_to_num(nan=0.0, posinf=1e300, neginf=-1e300).amax(0))
    forced = set(range(sink)) | set(range(count - recent, count))
    free = sorted(set(range(count)) - forced, key=lambda b: (-float(score[b]), b))
    return sorted(forced | set(free[:top - len(forced)]))


def check(q, keys, values, bounds, bt, lengths, top, sink=1, recent=2, page=PAGE, scale=None, finite=True):
    rows, heads = q.shape[0], keys.shape[2]
    group = q.shape[1] // heads
    selected = torch.full((rows, heads, top), -7, dtype=torch.int32, device=DEV)
    used = torch.tensor(lengths, dtype=torch.int32)
    got = ops.sparse_paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), bounds.to(DEV), bt.to(DEV), used.to(DEV),
                                     top_blocks=top, sink_blocks=sink, recent_blocks=recent, scale=scale,
                                     selected=selected).cpu().double()
    selected = selected.cpu()
    scale = 128 ** -0.5 if scale is None else scale
    for row, length in enumerate(lengths):
        for h in range(heads):
            query = q[row, h * group:(h + 1) * group].double()
            blocks = select(query, bounds[:, h], bt[row], length, top, sink, recent, page)
            assert selected[row, h].tolist() == blocks + [-1] * (top - len(blocks))
            out = got[row, h * group:(h + 1) * group]
            if not blocks:
                assert (out == 0).all()
                continue
            at = torch.cat([torch.arange(b * BLOCK, min(length, b * BLOCK + BLOCK)) for b in blocks])
            page_of = bt[row].long()[at // page]
            k, v = keys[page_of, at % page, h].double(), values[page_of, at % page, h].double()
            w = torch.softmax(query @ k.t() * scale, -1)
            y = w @ v
            if not finite:
                assert torch.equal(out.isfinite(), y.isfinite())
                continue
            d = abs(scale) * 130 * 2.0 ** -23 * (query.abs() @ k.abs().t()).amax(-1, keepdim=True) + 2.0 ** -20
            tol = (2.0 ** -8 + 2 * d) * (w @ v.abs()) + 2.0 ** -8 * y.abs()
            assert ((out - y).abs() <= tol).all()
    return got


@pytest.mark.parametrize("group", [1, 2, 4, 8])
@pytest.mark.parametrize("lengths,top", [
    ([1], 4), ([64, 65, 63], 4), ([0, 300, -3], 4), ([640], 4), ([641, 2000, 77, 1279], 8), ([5000], 17),
    ([1500] * 9, 5), ([700] * 80, 3),
])
def test_matches_the_definition(lengths, top, group):
    heads = 2
    pages = sum(-(-max(0, n) // PAGE) for n in lengths) + 1
    keys, values, g = pool(pages, heads, 11)
    bt = table([max(0, n) for n in lengths], pages, g)
    q = torch.randn(len(lengths), heads * group, 128, generator=g).to(torch.bfloat16)
    check(q, keys, values, whole_bounds(keys), bt, lengths, top)
    assert _native.device_status() == 0


@pytest.mark.parametrize("top,sink,recent", [(1, 0, 1), (3, 1, 2), (5, 5 - 1, 1), (6, 0, 6), (8, 0, 1), (40, 2, 3)])
def test_forced_blocks(top, sink, recent):
    keys, values, g = pool(9, 2, 3)
    bt = table([2100], 9, g)
    q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16)
    check(q, keys, values, whole_bounds(keys), bt, [2100], top, sink, recent)


def test_page_sizes_wide_tables_and_scale():
    for page in (64, 512):
        keys, values, g = pool(3000 // page + 4, 4, 8, page)
        bt = table([2900], keys.shape[0], g, page, width=3000 // page + 3)
        bt[:, -(-2900 // page):] = 999_999  # entries past the row's pages are not read
        q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16)
        check(q, keys, values, whole_bounds(keys), bt, [2900], 6, page=page, scale=0.03)
    assert _native.device_status() == 0


def test_ties_go_to_the_lower_block():
    keys, values, g = pool(12, 2, 4)
    bt = table([3000], 12, g)
    q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16)
    bounds = whole_bounds(keys)
    check(torch.zeros_like(q), keys, values, bounds, bt, [3000], 9)       # every score 0
    bounds[:] = bounds[:1, :, :1]
    check(q, keys, values, bounds, bt, [3000], 9)                         # every score equal
    bounds[int(bt[0, 5]), :, 2, 1] += 1                                   # one block ahead, one behind
    bounds[int(bt[0, 6]), :, 1, 1] -= 1
    check(q, keys, values, bounds, bt, [3000], 9)


def test_scores_that_fp32_cannot_tell_apart():
    """Two large terms that cancel, and blocks that differ by far less than fp32 resolves beside them."""
    keys, values, g = pool(10, 2, 6)
    bt = table([2500], 10, g)
    q = torch.ones(1, 8, 128).to(torch.bfloat16)
    bounds = torch.zeros(10, 2, 4, 2, 128)
    bounds[..., 1, 0], bounds[..., 1, 127] = 2.0 ** 14, -(2.0 ** 14)
    bounds[..., 1, 5] = torch.randint(0, 200, (10, 2, 4), generator=g) * 2.0 ** -16
    check(q, keys, values, bounds.to(torch.bfloat16), bt, [2500], 11)


def test_large_outlier_channels():
    keys, values, g = pool(40, 2, 9)
    keys[..., 7] *= 64
    keys[..., 100] *= -48
    bt = table([10_000], 40, g)
    q = torch.randn(1, 16, 128, generator=g).to(torch.bfloat16)
    check(q, keys, values, whole_bounds(keys), bt, [10_000], 20)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_bad_keys_are_selected_not_hidden(bad):
    keys, values, g = pool(10, 2, 12)
    bt = table([2500], 10, g)
    q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16)
    q[:, :, 3] = 0.5 if bad > 0 else -0.5
    keys[int(bt[0, 4]), 70, 1, 3] = bad
    blocks = keys.view(10, 4, BLOCK, 2, 128)
    bounds = whole_bounds(keys)
    got = check(q, keys, values, bounds, bt, [2500], 6, finite=False)
    assert got[0, :4].isfinite().all() and blocks.shape[0] == 10


def test_values_past_the_row_are_not_read():
    keys, values, g = pool(4, 2, 13)
    bt = table([900], 4, g)
    q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16)
    bounds = whole_bounds(keys)
    last = int(bt[0, 3])
    keys[last, 900 - 768:] = float("nan")
    values[last, 900 - 768:] = float("nan")
    check(q, keys, values, bounds, bt, [900], 5)


def test_bad_pages_are_flagged_and_skipped():
    keys, values, g = pool(10, 2, 14)
    bt = table([2300, 2300], 20, g) % 10
    bt[0, 0] = -1   # a forced block's page
    bt[1, 3] = 10   # scored blocks' page
    q = torch.randn(2, 8, 128, generator=g).to(torch.bfloat16)
    out = ops.sparse_paged_attention(q.to(DEV), keys.to(DEV), values.to(DEV), whole_bounds(keys).to(DEV), bt.to(DEV),
                                     torch.tensor([2300, 99_999], dtype=torch.int32, device=DEV), top_blocks=6)
    assert _native.device_status() == 1 << 3
    assert out.isfinite().all()


def test_repeats_streams_and_graphs():
    keys, values, g = pool(60, 8, 15)
    lengths = [3000, 100, 5000]
    bt = table(lengths, 60, g)
    q = torch.randn(3, 32, 128, generator=g).to(torch.bfloat16).to(DEV)
    args = [t.to(DEV) for t in (keys, values, whole_bounds(keys), bt, torch.tensor(lengths, dtype=torch.int32))]

    def run(query):
        return ops.sparse_paged_attention(query, *args, top_blocks=12)

    first = run(q)
    for _ in range(5):
        assert torch.equal(run(q), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = [run(q), run(-q)]
        again = run(q)
    main = run(q)  # at the same time, on another stream
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(outs[0], first) and torch.equal(again, first) and torch.equal(main, first)
    static, graph = q.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = run(static)
    static.copy_(-q)
    args[4][1] = 900  # lengths are read on the device
    args[3][1] = args[3][0]
    graph.replay()
    assert torch.equal(captured, run(-q)) and torch.equal(captured[[0, 2]], outs[1][[0, 2]])


def test_refusals():
    keys, values, g = pool(4, 2, 16)
    bt = table([900], 4, g).to(DEV)
    q = torch.randn(1, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    keys, values = keys.to(DEV), values.to(DEV)
    bounds, used = whole_bounds(keys), torch.tensor([900], dtype=torch.int32, device=DEV)

    def run(q=q, keys=keys, values=values, bounds=bounds, bt=bt, used=used, **kw):
        return ops.sparse_paged_attention(q, keys, values, bounds, bt, used, **{"top_blocks": 4, **kw})

    run()
    for bad in (dict(top_blocks=2), dict(recent_blocks=0), dict(sink_blocks=-1), dict(top_blocks=2000),
                dict(q=q[:, :6]), dict(q=q.float()), dict(q=q.cpu()), dict(bounds=bounds[:3]), dict(values=values[:3]),
                dict(bt=bt.long()), dict(used=used.repeat(2)), dict(selected=torch.empty(1, 2, 4, device=DEV)),
                dict(selected=torch.empty(1, 2, 5, dtype=torch.int32, device=DEV)), dict(out=q[:, :4]),
                dict(bt=torch.zeros(1, 1537, dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            run(**bad)
    with pytest.raises(ValueError):
        ops.key_block_bounds(keys, bounds, bt, used, used, used)
    assert _native.device_status() == 0


@pytest.mark.parametrize("rows", [1, 20])
def test_output_in_place_of_the_queries(rows):
    keys, values, g = pool(4, 2, 16)
    keys, values = keys.to(DEV), values.to(DEV)
    bt = table([900], 4, g).to(DEV).repeat(rows, 1)
    q = torch.randn(rows, 8, 128, generator=g).to(torch.bfloat16).to(DEV)
    used = torch.full((rows,), 900, dtype=torch.int32, device=DEV)
    want = ops.sparse_paged_attention(q, keys, values, whole_bounds(keys), bt, used, top_blocks=6)
    assert torch.equal(ops.sparse_paged_attention(q, keys, values, whole_bounds(keys), bt, used, q, top_blocks=6), want)
