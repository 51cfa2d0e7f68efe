"""Logit controls and token histories on the host (CPU only): settings, masks, slots, refusals."""

import math

import pytest
import torch

from helios_b200.controls import LogitControls, TokenHistory, control_rows, pack_mask
from helios_b200.config import Qwen3Config
from helios_b200.paged_cache import KVPagePool, SparseAttention


def test_controls_settings():
    assert not LogitControls().penalised and LogitControls(frequency_penalty=0.1, slot=3).penalised
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=math.nan), dict(repetition_penalty=math.inf),
                dict(frequency_penalty=math.inf, slot=0), dict(presence_penalty=0.5), dict(logit_bias={-1: 1.0}),
                dict(logit_bias={3: math.nan})):
        with pytest.raises(ValueError):
            LogitControls(**bad)


@pytest.mark.parametrize("vocab", [1, 31, 32, 33, 1000])
def test_pack_mask(vocab):
    allowed = torch.rand(3, vocab, generator=torch.Generator().manual_seed(vocab)) < 0.5
    words = pack_mask(allowed)
    assert words.dtype == torch.int32 and words.shape == (3, (vocab + 31) // 32)
    token = torch.arange(vocab)
    assert torch.equal(((words[:, token // 32] >> (token % 32)) & 1).bool(), allowed)
    with pytest.raises(ValueError):
        pack_mask(allowed.int())


def test_history_slots():
    history = TokenHistory(2, 5, "cpu")
    a, b = history.open([7, 8]), history.open([])
    with pytest.raises(RuntimeError, match="in use"):
        history.open([1])
    history.append([b, a], torch.tensor([3, 4]))
    history.append([a], [5])
    assert history.tokens[a].tolist()[:4] == [7, 8, 4, 5] and history.tokens[b].tolist()[:1] == [3]
    assert history.lengths[[a, b]].tolist() == [4, 1] and history.prompt_lengths[[a, b]].tolist() == [2, 0]
    history.append([a], [6])
    for bad in (lambda: history.append([a], [9]), lambda: history.append([b, b], [1, 2]),
                lambda: history.append([b], torch.tensor([1, 2])), lambda: history.open([0] * 6)):
        with pytest.raises(ValueError):
            bad()
    history.close(a)
    for bad in (lambda: history.close(a), lambda: history.append([a], [1]), lambda: history.length(9)):
        with pytest.raises(ValueError, match="not open"):
            bad()
    c = history.open([1])  # the slot again, without its old tokens
    assert c == a and history.length(c) == 1 and history.lengths[c] == 1 and history.prompt_lengths[c] == 1
    with pytest.raises(ValueError):
        TokenHistory(1, 65_536, "cpu")


def test_control_rows_refusals():
    x = torch.zeros(2, 40, dtype=torch.bfloat16)
    history = TokenHistory(1, 4, "cpu")
    with pytest.raises(ValueError, match="Each logit row"):
        control_rows(x, [None])
    with pytest.raises(ValueError, match="TokenHistory"):
        control_rows(x, [None, LogitControls(presence_penalty=1.0, slot=0)])
    with pytest.raises(ValueError, match="not open"):
        control_rows(x, [None, LogitControls(presence_penalty=1.0, slot=0)], history)
    with pytest.raises(ValueError, match="outside the vocabulary"):
        control_rows(x, [None, LogitControls(logit_bias={40: 1.0})])
    with pytest.raises(ValueError, match="allowed"):
        control_rows(x, [LogitControls(allowed=torch.ones(41, dtype=torch.bool)), None])
    assert torch.equal(control_rows(x, [None, None]), x)
    assert control_rows(x, [None, None], out=x) is x


def test_sparse_attention_settings():
    assert SparseAttention() == SparseAttention(32, 1, 2)
    for bad in ((2, 1, 2), (8, -1, 2), (8, 1, 0), (1025, 1, 2)):
        with pytest.raises(ValueError):
            SparseAttention(*bad)


def test_pool_bounds_cover_keys_appended_before():
    config = Qwen3Config(vocab_size=64, context_length=2048, hidden_size=64, n_heads=4, n_layers=2, hidden_dim=64,
                         head_dim=128, n_kv_heads=2, dtype=torch.bfloat16)
    pool = KVPagePool(config, 3, device=torch.device("cpu"))
    pool.storage.normal_()
    assert pool.bounds is None
    pool.enable_key_bounds()
    assert pool.bounds.shape == (2, 3, 2, 4, 2, 128)
    block = pool.keys[1][2, 64:128, 1]
    assert torch.equal(pool.bounds[1, 2, 1, 1, 0], block.amin(0)) and torch.equal(pool.bounds[1, 2, 1, 1, 1], block.amax(0))
    first = pool.bounds
    pool.enable_key_bounds()
    assert pool.bounds is first


@pytest.mark.parametrize("bad", [dict(repetition_penalty=1e39, slot=0), dict(repetition_penalty=1e-50, slot=0),
                                 dict(frequency_penalty=-1e39, slot=0), dict(presence_penalty=math.nan, slot=0),
                                 dict(logit_bias={3: math.inf}), dict(logit_bias={3: 1e39})])
def test_settings_that_fp32_does_not_hold(bad):
    with pytest.raises(ValueError):
        LogitControls(**bad)
    assert LogitControls(logit_bias={3: -math.inf}).logit_bias[3] == -math.inf
