"""Key bounds of a pool, switched on and off by its owner or by a decoder's setting, and sparse ticks that
are refused (CPU only)."""

import dataclasses
from types import SimpleNamespace

import pytest
import torch

from helios_b200.config import Qwen3Config
from helios_b200.decode import Decoder
from helios_b200.paged_cache import KVPagePool, PagedBatchCache, PagedKVCache, SparseAttention

CONFIG = Qwen3Config(vocab_size=64, context_length=2048, hidden_size=64, n_heads=4, n_layers=2, hidden_dim=64,
                     head_dim=128, n_kv_heads=2, dtype=torch.bfloat16)


def test_bounds_go_with_the_setting_that_brought_them():
    pool = KVPagePool(CONFIG, 3, device=torch.device("cpu"))
    batch = PagedBatchCache([PagedKVCache(pool, 100)])
    decoder = Decoder(None)
    decoder._set_sparse(batch)
    assert pool.bounds is None and batch.sparse is None
    decoder.sparse_attention = SparseAttention()
    decoder._set_sparse(batch)
    assert pool.bounds is not None and batch.sparse == SparseAttention()
    pool.storage.normal_()
    decoder.sparse_attention = None
    decoder._set_sparse(batch)
    assert pool.bounds is None and batch.sparse is None
    pool.enable_key_bounds()  # the owner's: taken from the keys there are now, and kept
    assert torch.equal(pool.bounds[1, 2, 1, 1, 0], pool.keys[1][2, 64:128, 1].amin(0))
    for setting in (SparseAttention(), None):
        decoder.sparse_attention = setting
        decoder._set_sparse(batch)
        assert pool.bounds is not None
    pool.disable_key_bounds()
    assert pool.bounds is None


@pytest.mark.parametrize("call", ["decode", "packed"])
def test_a_refused_tick_leaves_its_caches_alone(call, monkeypatch):
    """Bounds that find no memory, and rows longer than the sparse kernel covers: refused before the
    tick takes pages or marks its caches, and the decoder holds on to none of them."""
    pool = KVPagePool(dataclasses.replace(CONFIG, context_length=400_000), 1, device=torch.device("cpu"))
    decoder = Decoder(SimpleNamespace(training=False))
    decoder.sparse_attention = SparseAttention()

    def run(cache, error, match):
        with pytest.raises(error, match=match):
            decoder.decode_caches([cache], [1]) if call == "decode" else decoder.packed_caches([cache], [[1, 2]])
        batch = decoder._paged_decode_batch if call == "decode" else decoder._packed_batch
        assert batch.caches == () and cache._pending_tokens is None and not cache.pages
        assert pool.free_pages == 1

    run(PagedKVCache(pool, 393_217), ValueError, "393,216")

    def full():
        raise torch.OutOfMemoryError("no memory for the bounds")

    monkeypatch.setattr(pool, "enable_key_bounds", full)
    run(PagedKVCache(pool, 100), torch.OutOfMemoryError, "bounds")
