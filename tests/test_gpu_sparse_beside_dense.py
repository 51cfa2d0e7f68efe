"""Rows beside the sparse attention's: which work the dense kernels get, and what it computes."""

import pytest
import torch

from helios_b200 import _native
from helios_b200.config import Qwen3Config
from helios_b200.paged_cache import KVPagePool, PackedBatchCache, PagedKVCache, SparseAttention
from tests.test_gpu_decode_step import DEV, SHAPE, _close, _decoder, _model, _prompts, _reference_rows

pytestmark = pytest.mark.gpu


def _tick(caches, counts, q, k, v, sparse):
    batch = PackedBatchCache(caches)
    batch.sparse = sparse
    batch.prepare_packed(counts)
    out = batch.attend(0, q, k, v)[0].transpose(0, 1)  # [tokens, heads, d]
    items = (batch.num_decode_items, batch.num_prefill_items, batch.num_prefix_items)
    return batch, out, items


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("counts", [[1, 300, 1], [1, 1, 4], [1, 1, 1], [1, 90, 3], [200, 5, 1]])
def test_rows_beside_sparse_ones(counts, shared):
    """Single-token rows go to the sparse kernel alone; the others' attention is that of a dense tick."""
    pool = KVPagePool(Qwen3Config(**{**SHAPE, "n_layers": 1}), 60, device=DEV)
    pool.enable_key_bounds()
    setting = SparseAttention(top_blocks=6)
    g = torch.Generator().manual_seed(7)
    first = PagedKVCache(pool, 3000)
    draw = lambda total: [torch.randn(1, n, total, 128, generator=g).to(torch.bfloat16).to(DEV) for n in (8, 2, 2)]
    batch, _, _ = _tick([first], [1536], *draw(1536), None)
    batch.advance_packed()
    caches = []
    for _ in range(3):
        cache = PagedKVCache(pool, 3000)
        if shared:  # pages restored by aliasing, which dense ticks read once for all rows
            cache.restore_blocks([first.snapshot_block(0, 1280)])
        else:
            batch, _, _ = _tick([cache], [1100], *draw(1100), None)
            batch.advance_packed()
        caches.append(cache)
    q, k, v = draw(sum(counts))
    results = []
    for sparse in (None, setting):
        batch, out, items = _tick(caches, counts, q, k, v, sparse)
        if sparse is not None:
            assert items[2] == 0 and (items[0] > 0) == any(1 < c <= 16 for c in counts)
        results.append(out.clone())
        for cache in caches:
            cache._pending_tokens = None  # the same tick again: it writes the same keys and values
    at = 0
    for cache, count in zip(caches, counts):
        dense, got = (r[at:at + count].float() for r in results)
        if count == 1:
            want = _reference_rows(pool, 0, q[0, :, at].cpu(), cache, setting)
            assert (got[0].cpu().double() - want).abs().max() < 0.02 and want.abs().max() > 0.05
        elif count > 16:
            assert torch.equal(got, dense)  # the same tiles
        else:
            # Other splits: each output is within its bf16 rounding and that of the weights (2^-8 of
            # at most 5, the largest value) of the exact one.
            assert (got - dense).abs().max() <= 2 * (2.0 ** -8 * dense.abs().max() + 2.0 ** -8 * 5)
        at += count
    assert _native.device_status() == 0


def test_a_tick_packed_for_sparse_rows_needs_the_setting():
    pool = KVPagePool(Qwen3Config(**{**SHAPE, "n_layers": 1}), 4, device=DEV)
    pool.enable_key_bounds()
    batch = PackedBatchCache([PagedKVCache(pool, 100)])
    batch.sparse = SparseAttention()
    batch.prepare_packed([1])
    batch.sparse = None
    x = torch.zeros(1, 8, 1, 128, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(RuntimeError, match="prepared for sparse"):
        batch.attend(0, x, x[:, :2], x[:, :2])


def test_captured_ticks_with_shared_prefixes():
    """Rows that share restored pages, beside a drafted row: dense ticks (prefix items) and sparse ones
    (none) in turn, from graphs as eagerly."""
    prompt, draft = _prompts((1280, 4), seed=12)

    def run(graphs):
        model = _model(5)
        if graphs:
            model.enable_cuda_graphs(8)
        decoder = _decoder(model, pages=60)
        first = PagedKVCache(decoder.page_pool, 1400)
        decoder.packed_caches([first], [prompt])
        caches = [first]
        for token in (7, 9, 11):
            cache = PagedKVCache(decoder.page_pool, 1400)
            cache.restore_blocks([first.snapshot_block(0, 1280)])
            caches.append(cache)
        out = []
        for step in range(10):
            decoder.sparse_attention = SparseAttention(6) if step % 4 < 2 else None
            chunks = [[step + 1], [20 + step], draft, [40 + step]]
            out.append(decoder.packed_caches(caches, chunks).clone())
        if graphs:
            assert model._graphs.replays > 0
        return out

    for a, b in zip(run(True), run(False)):
        _close(a, b)
    assert _native.device_status() == 0
