"""Logit controls (ops.control_logits) against the formula in 64 bits.

Tolerance per logit: at most five fp32 operations, each off by 2^-24 of its operands' size, and one
rounding to bf16 (2^-8 of the result)."""

import math

import pytest
import torch

from helios_b200 import _native, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda")


def formula(logits, r, f, p, told, prompts, biases, allowed):
    """Rows of float64 results and the size of what was added up."""
    x = logits.double().clone()
    size = x.abs()
    for row in range(x.shape[0]):
        tokens = told[row]
        seen = sorted(set(tokens))
        for t in seen:
            x[row, t] = x[row, t] / r[row] if x[row, t] > 0 else x[row, t] * r[row]
            size[row, t] = max(size[row, t], x[row, t].abs())
        produced = tokens[prompts[row]:]
        for t in set(produced):
            x[row, t] -= f[row] * produced.count(t) + p[row]
            size[row, t] += abs(f[row]) * produced.count(t) + abs(p[row])
        for t, b in biases[row].items():
            x[row, t] += b
            size[row, t] += abs(b)
        if allowed[row] is not None:
            x[row, ~allowed[row]] = -math.inf
    return x, size


def problem(rows, vocab, history, seed, spread=None):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(rows, vocab, generator=g) * 4).to(torch.bfloat16)
    told = [torch.randint(0, min(vocab, spread or vocab), (int(n),), generator=g).tolist()
            for n in torch.randint(0, history + 1, (rows,), generator=g)]
    prompts = [int(len(t) * float(torch.rand(1, generator=g))) for t in told]
    r = (1 + torch.rand(rows, generator=g) * 0.5).tolist()
    f = (torch.rand(rows, generator=g) * 2 - 0.5).tolist()
    p = (torch.rand(rows, generator=g) * 2 - 0.5).tolist()
    biases = [{int(t): float(torch.randn(1, generator=g) * 5)
               for t in torch.randint(0, vocab, (int(torch.randint(0, 9, (1,), generator=g)),), generator=g)}
              for _ in range(rows)]
    allowed = [torch.rand(vocab, generator=g) < 0.3 if row % 3 else None for row in range(rows)]
    return logits, r, f, p, told, prompts, biases, allowed


def words(allowed, vocab):
    masks = [a for a in allowed if a is not None]
    out = torch.zeros(max(1, len(masks)), (vocab + 31) // 32, dtype=torch.int64)
    for i, a in enumerate(masks):
        at = torch.nonzero(a).flatten()
        out[i].scatter_add_(0, at // 32, 1 << (at % 32))
    which = iter(range(len(masks)))
    rows = torch.tensor([-1 if a is None else next(which) for a in allowed], dtype=torch.int32)
    return torch.where(out >= 2 ** 31, out - 2 ** 32, out).int().to(DEV), rows.to(DEV)


def arguments(logits, r, f, p, told, prompts, biases, allowed, g=None):
    rows, vocab = logits.shape
    slots = torch.randperm(rows + 2, generator=torch.Generator().manual_seed(rows))[:rows]
    width = max(1, max(map(len, told)))
    history = torch.full((rows + 2, width), -5, dtype=torch.int32)  # entries past a length are not read
    lengths, plens = torch.zeros(rows + 2, dtype=torch.int32), torch.zeros(rows + 2, dtype=torch.int32)
    for row, tokens in enumerate(told):
        s = int(slots[row])
        history[s, :len(tokens)] = torch.tensor(tokens, dtype=torch.int32)
        lengths[s], plens[s] = len(tokens), prompts[row]
    offsets = torch.tensor([0] + [len(b) for b in biases]).cumsum(0).int()
    tokens = torch.tensor([t for b in biases for t in sorted(b)], dtype=torch.int32)
    values = torch.tensor([b[t] for b in biases for t in sorted(b)], dtype=torch.float32)
    mask, mask_rows = words(allowed, vocab)
    return dict(repetition=torch.tensor(r, device=DEV), frequency=torch.tensor(f, device=DEV),
                presence=torch.tensor(p, device=DEV), history=history.to(DEV), slots=slots.int().to(DEV),
                lengths=lengths.to(DEV), prompt_lengths=plens.to(DEV),
                bias=(offsets.to(DEV), tokens.to(DEV), values.to(DEV)), mask=mask, mask_rows=mask_rows)


def close(got, want, size):
    got = got.cpu().double()
    banned = want == -math.inf
    assert torch.equal(got == -math.inf, banned)
    tol = 2.0 ** -8 * want.abs() + 6 * 2.0 ** -24 * size
    assert ((got - want).abs() <= tol)[~banned].all()


@pytest.mark.parametrize("rows,vocab,history,spread", [
    (1, 1, 3, None), (3, 31, 50, None), (2, 1000, 0, None), (4, 1025, 700, 40), (7, 8200, 2000, None),
    (5, 20_001, 300, 11), (2, 151_936, 3000, 500), (2, 311_391, 900, None),
])
def test_matches_the_formula(rows, vocab, history, spread):
    case = problem(rows, vocab, history, vocab, spread)
    args = arguments(*case)
    got = ops.control_logits(case[0].to(DEV), **args)
    close(got, *formula(*case))
    # In place, and on rows inside a wider tensor (another alignment): the same values.
    wide = torch.full((rows, vocab + 5), 3.0, dtype=torch.bfloat16, device=DEV)
    view = wide[:, 2:vocab + 2]
    view.copy_(case[0])
    assert ops.control_logits(view, **args, out=view) is view
    assert torch.equal(view, got)
    assert (wide[:, :2] == 3).all() and (wide[:, vocab + 2:] == 3).all()
    assert _native.device_status() == 0


@pytest.mark.parametrize("drop", ["repetition", "frequency", "presence", "history", "bias", "mask"])
def test_each_control_may_be_absent(drop):
    case = list(problem(4, 3000, 400, 21, 60))
    args = arguments(*case)
    args[drop] = None
    if drop == "history":
        case[4], case[5] = [[]] * 4, [0] * 4
    elif drop == "bias":
        case[6] = [{}] * 4
    elif drop == "mask":
        case[7] = [None] * 4
    else:
        case[{"repetition": 1, "frequency": 2, "presence": 3}[drop]] = [1.0 if drop == "repetition" else 0.0] * 4
    close(ops.control_logits(case[0].to(DEV), **args), *formula(*case))


def test_no_controls_copies():
    x = torch.randn(3, 777).to(torch.bfloat16).to(DEV)
    assert torch.equal(ops.control_logits(x), x)
    assert ops.control_logits(x[:0]).shape == (0, 777)


def test_rows_without_history_and_shared_slots():
    x = torch.randn(3, 500).to(torch.bfloat16)
    told = [4, 4, 9]
    args = dict(frequency=torch.tensor([1.0, 1.0, 2.0], device=DEV),
                history=torch.tensor([[4, 4, 9, 0]], dtype=torch.int32, device=DEV),
                slots=torch.tensor([0, -1, 0], dtype=torch.int32, device=DEV),
                lengths=torch.tensor([3], dtype=torch.int32, device=DEV),
                prompt_lengths=torch.tensor([1], dtype=torch.int32, device=DEV))
    case = (x, [1.0] * 3, [1.0, 1.0, 2.0], [0.0] * 3, [told, [], told], [1] * 3, [{}] * 3, [None] * 3)
    close(ops.control_logits(x.to(DEV), **args), *formula(*case))


def test_values_that_are_not_finite():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    x[:, 0], x[:, 1], x[:, 2], x[:, 3] = math.inf, -math.inf, math.nan, torch.finfo(torch.bfloat16).min
    allowed = torch.ones(64, dtype=torch.bool)
    allowed[[0, 2]] = False
    mask, mask_rows = words([None, allowed], 64)
    bias = (torch.tensor([0, 2, 2], dtype=torch.int32, device=DEV), torch.tensor([5, 6], dtype=torch.int32, device=DEV),
            torch.tensor([-math.inf, math.nan], device=DEV))
    got = ops.control_logits(x.to(DEV), repetition=torch.tensor([2.0, 2.0], device=DEV),
                             history=torch.tensor([[0, 1, 2, 3]], dtype=torch.int32, device=DEV),
                             slots=torch.zeros(2, dtype=torch.int32, device=DEV),
                             lengths=torch.tensor([4], dtype=torch.int32, device=DEV),
                             prompt_lengths=torch.tensor([4], dtype=torch.int32, device=DEV), bias=bias, mask=mask,
                             mask_rows=mask_rows).cpu()
    assert got[0, 0] == math.inf and got[0, 1] == -math.inf and got[0, 2].isnan() and got[0, 3] == -math.inf
    assert got[0, 5] == -math.inf and got[0, 6].isnan() and (got[0, 7:] == 0).all()
    assert got[1, 0] == -math.inf and got[1, 1] == -math.inf and got[1, 2] == -math.inf and (got[1, 4:] == 0).all()


def test_a_mask_may_leave_nothing():
    x = torch.randn(2, 4100).to(torch.bfloat16).to(DEV)
    mask = torch.zeros(1, 129, dtype=torch.int32, device=DEV)
    got = ops.control_logits(x, mask=mask, mask_rows=torch.tensor([0, -1], dtype=torch.int32, device=DEV))
    assert (got[0] == -math.inf).all() and torch.equal(got[1], x[1])


def test_bias_lists_out_of_order():
    x = torch.zeros(1, 400, dtype=torch.bfloat16, device=DEV)

    def run(tokens, values):
        n = torch.tensor([0, len(tokens)], dtype=torch.int32, device=DEV)
        return ops.control_logits(x, bias=(n, torch.tensor(tokens, dtype=torch.int32, device=DEV),
                                           torch.tensor(values, device=DEV)))[0].cpu()

    got = run([7, 7, 7, 300], [1.0, 2.0, 4.0, 8.0])  # of equal neighbours the last counts
    assert got[7] == 4 and got[300] == 8 and got.count_nonzero() == 2 and _native.device_status() == 0
    got = run([9, 5, 6], [1.0, 2.0, 4.0])
    assert got[9] == 0 and got[5] == 2 and got[6] == 4 and _native.device_status() == 1 << 4
    got = run([-1, 5, 400], [1.0, 2.0, 4.0])
    assert got[5] == 2 and got.count_nonzero() == 1 and _native.device_status() == 1 << 4


def test_indices_outside_are_flagged_and_skipped():
    x = torch.randn(2, 400).to(torch.bfloat16).to(DEV)
    base = dict(presence=torch.ones(2, device=DEV), history=torch.tensor([[3, 400, -1]], dtype=torch.int32, device=DEV),
                lengths=torch.tensor([9], dtype=torch.int32, device=DEV),  # more than the arena holds
                prompt_lengths=torch.tensor([0], dtype=torch.int32, device=DEV))
    got = ops.control_logits(x, **base, slots=torch.tensor([0, -1], dtype=torch.int32, device=DEV))
    assert _native.device_status() == 1 << 4
    assert torch.equal(got[1], x[1]) and (got[0] != x[0]).sum() == 1 and got[0, 3] != x[0, 3]
    got = ops.control_logits(x, **base, slots=torch.tensor([1, -2], dtype=torch.int32, device=DEV))
    assert _native.device_status() == 1 << 5 and torch.equal(got, x)
    mask = torch.zeros(1, 13, dtype=torch.int32, device=DEV)
    got = ops.control_logits(x, mask=mask, mask_rows=torch.tensor([1, -2], dtype=torch.int32, device=DEV))
    assert _native.device_status() == 1 << 5 and torch.equal(got, x)
    bad = (torch.tensor([0, 5, 1], dtype=torch.int32, device=DEV), torch.tensor([2], dtype=torch.int32, device=DEV),
           torch.ones(1, device=DEV))
    got = ops.control_logits(x, bias=bad)
    assert _native.device_status() == 1 << 5 and torch.equal(got, x)


def test_streams_and_graphs():
    case = problem(9, 5000, 900, 33, 100)
    args, x = arguments(*case), case[0].to(DEV)
    first = ops.control_logits(x, **args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.control_logits(x, **args)
    here = ops.control_logits(x, **args)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, first) and torch.equal(here, first)
    graph, static = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(graph):
        captured = ops.control_logits(static, **args)
    static.copy_(x.flip(0))
    args["lengths"].zero_()
    graph.replay()
    assert torch.equal(captured, ops.control_logits(x.flip(0).contiguous(), **args))
    assert not torch.equal(captured, first)


def test_refusals():
    x = torch.zeros(2, 100, dtype=torch.bfloat16, device=DEV)
    two, one = torch.zeros(2, dtype=torch.int32, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    history = torch.zeros(1, 4, dtype=torch.int32, device=DEV)
    for bad in (dict(repetition=torch.ones(3, device=DEV)), dict(frequency=torch.ones(2)), dict(history=history),
                dict(history=history, slots=one, lengths=one, prompt_lengths=one),
                dict(history=history, slots=two, lengths=two, prompt_lengths=one),
                dict(history=history.long(), slots=two, lengths=one, prompt_lengths=one),
                dict(mask=torch.zeros(1, 4, dtype=torch.int32, device=DEV)),
                dict(mask=torch.zeros(1, 3, dtype=torch.int32, device=DEV), mask_rows=two),
                dict(bias=(two, one, torch.zeros(1, device=DEV))), dict(out=torch.zeros(2, 99, device=DEV))):
        with pytest.raises(ValueError):
            ops.control_logits(x, **bad)
    with pytest.raises(ValueError):
        ops.control_logits(x.cpu())
    with pytest.raises(ValueError):
        ops.control_logits(x.t())
    assert _native.device_status() == 0


def test_outputs_over_part_of_the_logits_are_refused():
    memory = torch.zeros(4 * 100 + 8, dtype=torch.bfloat16, device=DEV)
    x = memory[:400].view(4, 100)
    for out in (memory[8:].view(4, 100), memory[:300].view(3, 100)):
        with pytest.raises(ValueError):
            ops.control_logits(x if out.shape[0] == 4 else memory[100:400].view(3, 100), out=out)
    assert torch.equal(ops.control_logits(x[:2], out=x[2:]), x[:2])
    assert _native.device_status() == 0
