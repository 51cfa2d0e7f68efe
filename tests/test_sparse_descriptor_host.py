"""The host half of a tick with sparse attention: rows with one token get no dense work (CPU only)."""

import numpy as np
import pytest
import torch

from helios_b200.config import Qwen3Config
from helios_b200.paged_cache import KVPagePool, PackedBatchCache, PagedKVCache, SparseAttention

CONFIG = Qwen3Config(vocab_size=64, context_length=4096, hidden_size=64, n_heads=8, n_layers=1, hidden_dim=64,
                     head_dim=128, n_kv_heads=2, dtype=torch.bfloat16)


def _batch(lengths, shared=0):
    pool = KVPagePool(CONFIG, 80, device=torch.device("cpu"))
    lead = pool.acquire(shared)
    caches = []
    for length in lengths:
        cache = PagedKVCache(pool, 4096)
        cache.pages = lead + pool.acquire(-(-(length + 300) // 256) - shared)
        cache.length = length
        caches.append(cache)
    return PackedBatchCache(caches)


@pytest.mark.parametrize("shared", [0, 5])
@pytest.mark.parametrize("counts", [[1, 1, 1], [1, 300, 1], [1, 4, 1], [4, 300, 1], [5, 2, 16]])
def test_single_token_rows_get_no_dense_work(counts, shared):
    lengths = [2000, 1500, 1700]
    want = _batch(lengths, shared)._host_descriptor(counts, [1] * 3)
    batch = _batch(lengths, shared)
    batch.sparse = SparseAttention()
    got = batch._host_descriptor(counts, [1] * 3)
    single = np.array(counts) == 1
    assert (got["rows"][single, 5] == -1).all() and (got["rows"][~single, 5] == 0).all()
    assert (got["rows"][:, 6] == 0).all() and got["num_prefix_items"] == 0
    assert np.array_equal(got["rows"][:, :5], want["rows"][:, :5])
    assert got["num_prefill_items"] == want["num_prefill_items"]
    # What is left is the work of the other rows alone.
    others = [i for i in range(3) if not single[i]]
    if others:
        alone = _batch([lengths[i] for i in others])._host_descriptor([counts[i] for i in others], [1] * len(others))
        for name in ("num_decode_items", "partial_records", "num_prefill_items", "split_keys"):
            assert got[name] == alone[name], name
    else:
        assert got["num_decode_items"] == got["partial_records"] == 0
