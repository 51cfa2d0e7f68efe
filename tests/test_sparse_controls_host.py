"""Refusals of the sparse attention and the logit controls that need no device (CPU only)."""

import ctypes

import pytest
import torch

from helios_b200 import _native, ops

P = ctypes.c_void_p(4096)  # never read: every call here is refused, or has no work, before a launch


@pytest.fixture(scope="module")
def lib():
    from helios_b200 import build

    build.build()
    return _native.load()


def sparse(lib, rows=1, heads=8, kv_heads=2, dim=128, page=256, width=4, top=8, sink=1, recent=2, q=P, pages=10):
    return lib.hb_sparse_paged_attention(q, P, P, P, pages, page, P, width, P, None, rows, heads, kv_heads, dim, top, sink,
                                         recent, ctypes.c_float(0.1), None, P, None)


def test_sparse_attention_refusals(lib):
    unsupported, invalid = _native.HB_ERR_UNSUPPORTED, _native.HB_ERR_INVALID
    assert sparse(lib, dim=64) == unsupported and "head_dim 128" in _native.last_error()
    assert sparse(lib, heads=6) == unsupported
    assert sparse(lib, heads=7) == invalid
    assert sparse(lib, page=96) == invalid
    assert sparse(lib, width=1537) == unsupported and "393216 tokens" in _native.last_error()
    assert sparse(lib, top=2) == invalid and sparse(lib, top=1025) == invalid
    assert sparse(lib, recent=0) == invalid and sparse(lib, sink=-1) == invalid
    assert sparse(lib, recent=2 ** 31 - 1) == invalid and sparse(lib, sink=2 ** 31 - 1) == invalid
    assert sparse(lib, q=None) == invalid and sparse(lib, q=ctypes.c_void_p(4104)) == invalid
    assert sparse(lib, pages=2 ** 24) == unsupported
    assert sparse(lib, rows=0) == 0


def test_key_block_bounds_refusals(lib):
    def call(dim=128, page=256, rows=1, tokens=1, keys=P, width=4):
        return lib.hb_key_block_bounds(keys, P, 10, page, P, width, P, P, P, rows, tokens, 2, dim, None)

    assert call(dim=64) == _native.HB_ERR_UNSUPPORTED
    assert call(page=32) == _native.HB_ERR_INVALID and call(width=0) == _native.HB_ERR_INVALID
    assert call(keys=None) == _native.HB_ERR_INVALID
    assert call(tokens=0) == 0 and call(rows=0) == 0


def test_logit_control_refusals(lib):
    def call(stride=100, rows=2, vocab=100, history=None, width=4, slots=None, entries=0, offsets=None, mask=None,
             masks=0, out=ctypes.c_void_p(8192), out_stride=100, logits=P):
        return lib.hb_control_logits(logits, stride, rows, vocab, None, None, None, history, 1, width, slots, slots,
                                     slots, offsets, None, None, entries, mask, masks, None, out, out_stride, None)

    invalid = _native.HB_ERR_INVALID
    assert call(stride=99) == invalid and call(out_stride=99) == invalid and call(vocab=0) == invalid
    assert call(rows=70_000) == invalid and call(logits=None) == invalid
    assert call(history=P) == invalid and "history" in _native.last_error()
    assert call(history=P, slots=P, width=65_536) == _native.HB_ERR_UNSUPPORTED
    assert call(offsets=P, entries=3) == invalid and call(offsets=P, entries=-1) == invalid
    assert call(mask=P, masks=1) == invalid
    assert call(out=P, stride=100, out_stride=104) == invalid and "in place" in _native.last_error()
    assert call(rows=0) == 0


def test_host_tensors_are_refused():
    x = torch.zeros(2, 8, 128, dtype=torch.bfloat16)
    pool = torch.zeros(2, 256, 2, 128, dtype=torch.bfloat16)
    bounds = torch.zeros(2, 2, 4, 2, 128, dtype=torch.bfloat16)
    table, rows = torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        ops.sparse_paged_attention(x, pool, pool, bounds, table, rows, top_blocks=4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.key_block_bounds(pool, bounds, table, rows, rows, rows)
    with pytest.raises(ValueError, match="CUDA"):
        ops.control_logits(torch.zeros(2, 100, dtype=torch.bfloat16))
