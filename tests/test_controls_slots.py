"""Token history slots when a call is refused (CPU only)."""

import pytest
import torch

from helios_b200.controls import TokenHistory


@pytest.mark.parametrize("prompt", [[2 ** 40], ["a"], [1, None], [0] * 9])
def test_a_refused_prompt_takes_no_slot(prompt):
    history = TokenHistory(1, 8, "cpu")
    for _ in range(3):
        with pytest.raises((RuntimeError, TypeError, ValueError)) as refused:
            history.open(prompt)
        assert "in use" not in str(refused.value)
    slot = history.open([1, 2])
    assert history.tokens[slot, :2].tolist() == [1, 2] and history.length(slot) == 2
    with pytest.raises(RuntimeError, match="in use"):
        history.open([3])


def test_a_refused_append_changes_nothing():
    history = TokenHistory(2, 4, "cpu")
    a, b = history.open([1]), history.open([2, 3])
    before = [t.clone() for t in (history.tokens, history.lengths, history.prompt_lengths)]
    for bad in ([a, b], [2 ** 40, 1]), ([a, 7], [1, 2]), ([a, b], torch.tensor([1])):
        with pytest.raises((RuntimeError, ValueError)):
            history.append(*bad)
    assert history.length(a) == 1 and history.length(b) == 2
    for now, then in zip((history.tokens, history.lengths, history.prompt_lengths), before):
        assert torch.equal(now, then)
