"""Sparse attention switched off and on again between ticks, eager and captured."""

import pytest
import torch

from helios_b200 import _native, ops
from helios_b200.paged_cache import PagedKVCache, SparseAttention
from tests.test_gpu_decode_step import DEV, _close, _decode, _decoder, _model, _prompts

pytestmark = pytest.mark.gpu


def _counting(monkeypatch):
    calls = []
    real = ops.key_block_bounds
    monkeypatch.setattr(ops, "key_block_bounds", lambda *args: calls.append(1) or real(*args))
    return calls


def test_switched_off_no_tick_keeps_bounds(monkeypatch):
    calls = _counting(monkeypatch)
    model = _model()
    prompts = _prompts((5, 700, 1500))
    dense = _decode(_decoder(model), prompts, 3)
    assert not calls
    decoder = _decoder(model, sparse_attention=SparseAttention(5))
    _decode(decoder, prompts, 3)
    assert calls and decoder.page_pool.bounds is not None
    calls.clear()
    decoder.sparse_attention = None
    for a, b in zip(_decode(decoder, prompts, 3), dense):
        assert torch.equal(a, b)
    assert not calls and decoder.page_pool.bounds is None


def test_switching_between_captured_ticks():
    """Off and on again with graphs: each tick is that of a decoder which never switched."""
    prompts = _prompts((900, 1500), seed=4)
    steps = (True, True, True, False, False, False, True, True, True)

    def run(graphs):
        model = _model(2)
        if graphs:
            model.enable_cuda_graphs(8)
        decoder = _decoder(model)
        caches = [PagedKVCache(decoder.page_pool, len(p) + 20) for p in prompts]
        logits = [decoder.packed_caches(caches, prompts).clone()]
        junk = []
        for on in steps:
            if not on:
                junk.append(torch.full((8 << 20,), 0x7F, dtype=torch.uint8, device=DEV))  # where freed bounds were
            decoder.sparse_attention = SparseAttention(6) if on else None
            logits.append(decoder.decode_caches(caches, logits[-1].argmax(-1)).clone())
        if graphs:
            assert model._graphs.replays > 0
        return logits

    for a, b in zip(run(True), run(False)):
        _close(a, b)
    assert _native.device_status() == 0


def test_bounds_of_the_pools_owner_stay():
    model = _model()
    prompts = _prompts((300, 20))
    decoder = _decoder(model)
    decoder.page_pool.enable_key_bounds()
    bounds = decoder.page_pool.bounds
    for setting in (None, SparseAttention(5), None):
        decoder.sparse_attention = setting
        _decode(decoder, prompts, 2)
        assert decoder.page_pool.bounds is bounds
    decoder.page_pool.disable_key_bounds()
    assert decoder.page_pool.bounds is None


def test_two_decoders_of_one_pool():
    """One of them switches off: the other's next tick takes the bounds anew from the pool."""
    model = _model(1)
    prompts = _prompts((900, 1500), seed=6)

    def run(switch):
        a, b = _decoder(model, sparse_attention=SparseAttention(6)), _decoder(model, sparse_attention=SparseAttention(6))
        b.page_pool = a.page_pool
        caches = [PagedKVCache(a.page_pool, len(p) + 20) for p in prompts]
        logits = [a.packed_caches(caches, prompts).clone()]
        for i in range(4):
            if switch and i % 2:
                a.sparse_attention = None
                other = PagedKVCache(a.page_pool, 40)
                a.packed_caches([other], [[1, 2, 3]])
                assert (a.page_pool.bounds is None) == (i == 1)  # after that they are b's
                other.close()
            logits.append(b.decode_caches(caches, logits[-1].argmax(-1)).clone())
            a.sparse_attention = SparseAttention(6)
        return logits

    for x, y in zip(run(True), run(False)):
        assert torch.equal(x, y)
