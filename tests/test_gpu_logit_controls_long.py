"""Logit controls on histories and bias lists that take a CTA more than one pass, against the formula
in 64 bits (tolerance as in test_gpu_logit_controls)."""

import pytest
import torch

from helios_b200 import _native, ops
from tests.test_gpu_logit_controls import DEV, arguments, close, formula

pytestmark = pytest.mark.gpu


def case(told, prompts, vocab, biases=None, seed=5):
    g = torch.Generator().manual_seed(seed)
    rows = len(told)
    logits = (torch.randn(rows, vocab, generator=g) * 4).to(torch.bfloat16)
    return (logits, [1.2] * rows, [0.01] * rows, [0.3] * rows, told, prompts, biases or [{}] * rows,
            [None if row % 2 else torch.rand(vocab, generator=g) < 0.5 for row in range(rows)])


@pytest.mark.parametrize("vocab", [700, 40_000])
def test_histories_past_the_first_pass(vocab):
    g = torch.Generator().manual_seed(vocab)
    told = [(torch.rand(n, generator=g) ** 3 * vocab).int().clamp(max=vocab - 1).tolist() for n in (8193, 20_001, 65_535)]
    c = case(told, [4000, 20_001, 1], vocab)
    close(ops.control_logits(c[0].to(DEV), **arguments(*c)), *formula(*c))
    assert _native.device_status() == 0


@pytest.mark.parametrize("prompt", [0, 1, 65_535])
def test_one_token_fills_a_history(prompt):
    c = case([[9] * 65_535, [3]], [prompt, 0], 1000)
    close(ops.control_logits(c[0].to(DEV), **arguments(*c)), *formula(*c))


def test_bias_lists_past_the_first_pass():
    g = torch.Generator().manual_seed(8)
    biases = [{int(t): float(torch.randn(1, generator=g)) for t in torch.randperm(30_000, generator=g)[:n]}
              for n in (513, 4000, 0)]
    c = case([[5] * 40, [7, 7, 2], []], [10, 0, 0], 30_000, biases)
    close(ops.control_logits(c[0].to(DEV), **arguments(*c)), *formula(*c))
    assert _native.device_status() == 0
