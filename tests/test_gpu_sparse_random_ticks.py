"""Key bounds through random ticks: chunks, drafts that are cut back, aliased pages, closed and reused
pages. After every tick the bounds of each block of its rows are those of the row's keys, and with
blocks enough for every key the logits are those of dense attention."""

import random

import pytest
import torch

from helios_b200 import _native
from helios_b200.paged_cache import PagedKVCache, SparseAttention
from tests.test_gpu_decode_step import _close, _decoder, _model

pytestmark = pytest.mark.gpu


def _check_bounds(pool, cache):
    length = cache.length
    for layer in range(pool.config.n_layers):
        table = torch.tensor([page.index for page in cache.pages], device=pool.keys[layer].device)
        keys = pool.keys[layer][table].flatten(0, 1)[:length]      # [length, heads, d]
        got = pool.bounds[layer][table].transpose(1, 2).flatten(0, 1)  # [blocks, heads, 2, d]
        for block in range(-(-length // 64)):
            part = keys[64 * block:64 * block + 64]
            assert torch.equal(got[block, :, 0], part.amin(0)) and torch.equal(got[block, :, 1], part.amax(0))


@pytest.mark.parametrize("seed", [1, 2, 3])
def test_bounds_follow_the_keys(seed):
    rng = random.Random(seed)
    model = _model(seed)
    sparse, dense = _decoder(model, pages=40, sparse_attention=SparseAttention(64)), _decoder(model, pages=40)
    decoders = (sparse, dense)
    rows = []  # a request's cache in either pool
    for step in range(24):
        if len(rows) < 4 and (not rows or rng.random() < 0.5):
            pair = [PagedKVCache(d.page_pool, 1900) for d in decoders]
            whole = [r for r in rows if r[0].length >= 256]
            if whole and rng.random() < 0.6:  # restored from another request's pages
                source = rng.choice(whole)
                end = rng.randint(1, source[0].length // 256) * 256
                for cache, other in zip(pair, source):
                    cache.restore_blocks([other.snapshot_block(0, end)])
            rows.append(pair)
        counts = [rng.choice((1, 1, 1, rng.randint(2, 16), rng.randint(17, 400))) if r[0].length else
                  rng.randint(1, 700) for r in rows]
        counts = [min(c, 1899 - r[0].length) or 1 for c, r in zip(counts, rows)]
        chunks = [[rng.randrange(4096) for _ in range(c)] for c in counts]
        before = [r[0].length for r in rows]
        a, b = (d.packed_caches([r[i] for r in rows], chunks) for i, d in enumerate(decoders))
        _close(a, b)
        for pair in rows:
            _check_bounds(sparse.page_pool, pair[0])
        for pair, count, start in zip(rows, counts, before):
            if 1 < count <= 16:  # a draft of which a part is kept
                for cache in pair:
                    cache.truncate(start + 1 + (count - 1) // 2)
        for pair in [r for r in rows if r[0].length > 1400 or rng.random() < 0.08]:
            for cache in pair:
                cache.close()
            rows.remove(pair)
    assert _native.device_status() == 0
