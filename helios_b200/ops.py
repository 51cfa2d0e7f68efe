"""Torch-facing wrappers over the C ABI: tensors in, raw pointers to the library.

Every op runs on the caller's current CUDA stream, checks dtypes, devices and
contiguity on the host, and raises ``ValueError`` (bad arguments, as the
reference does) or ``RuntimeError`` (CUDA failure). Outputs are written into
caller-provided tensors; nothing here allocates device memory except where an
op's docstring says it returns a new tensor.
"""

from __future__ import annotations

import torch

from helios_b200 import _native

BF16 = torch.bfloat16
TICK_ROW_FIELDS = 7  # slot, length, count, logit count, pages, shared prefix keys, group rows
DECODE_ITEM_INTS = 6  # row, first key, end key, record base, splits of the row, 0
PREFIX_ITEM_INTS = 5  # first row, rows, first key, end key, prefix split index


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


# The handle of a device's current stream: what torch.cuda.current_stream(device).cuda_stream
# gives, without the Stream object (2.2 us of host time per call against 0.06).
_raw_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def _stream(device: torch.device) -> int:
    if _raw_stream is not None and device.index is not None:
        return _raw_stream(device.index)
    return torch.cuda.current_stream(device).cuda_stream


def _need(t: torch.Tensor, dtype: torch.dtype, name: str, *, contiguous: bool = True) -> None:
    if not t.is_cuda:
        raise ValueError(f"{name} must be a CUDA tensor (there is no CPU path)")
    if t.dtype != dtype:
        raise ValueError(f"{name} must be {dtype}, got {t.dtype}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


def lib():
    return _native.load()


def tick_pack(rows_dev: torch.Tensor, num_rows: int, updates_dev: torch.Tensor | None, num_updates: int,
              arena: torch.Tensor, page_size: int, width: int, num_pages: int, decode_max_tokens: int,
              split_keys: int, prefill_tile_tokens: int, total_tokens: int, out: dict, *,
              prefix_split_keys: int | None = None) -> None:
    """Kernel (a): expand row descriptors into the tick's metadata (``out`` holds the buffers)."""
    _need(rows_dev, torch.int32, "rows")
    _need(arena, torch.int32, "arena")
    rc = lib().hb_tick_pack(
        rows_dev.data_ptr(), num_rows, _ptr(updates_dev) if num_updates else None, num_updates, arena.data_ptr(),
        arena.shape[0], arena.shape[1], page_size, width, num_pages, decode_max_tokens, split_keys,
        prefill_tile_tokens, split_keys if prefix_split_keys is None else prefix_split_keys, total_tokens,
        out["block_table"].data_ptr(), out["cu_seq_q"].data_ptr(), out["cu_seq_k"].data_ptr(),
        out["seqused_k"].data_ptr(), out["positions"].data_ptr(), out["write_slots"].data_ptr(),
        out["token_row"].data_ptr(), out["logit_store"].data_ptr(), out["logit_store"].numel(),
        out["decode_items"].data_ptr(), out["decode_items"].numel() // DECODE_ITEM_INTS,
        out["prefill_items"].data_ptr(), out["prefill_items"].numel() // 3,
        _ptr(out.get("prefix_items")), out["prefix_items"].numel() // PREFIX_ITEM_INTS if "prefix_items" in out else 0,
        _ptr(out.get("counts")),
        _ptr(out.get("row_records")), _stream(rows_dev.device))
    _native.check(rc, "hb_tick_pack")


def qk_norm_rope_append(q: torch.Tensor | None, k: torch.Tensor, v: torch.Tensor, *, q_scale, k_scale, eps: float,
                        cos, sin, positions, write_slots: torch.Tensor, q_out: torch.Tensor | None,
                        key_pool: torch.Tensor, value_pool: torch.Tensor) -> None:
    """Kernel (b). q/k/v are ``[T, heads, d]`` views (any token/head strides, unit
    element stride); pools are one layer ``[P, page, Hkv, d]``."""
    tokens, kv_heads, dim = k.shape
    heads = q.shape[1] if q is not None else kv_heads
    for name, t in (("k", k), ("v", v)) + ((("q", q),) if q is not None else ()):
        _need(t, BF16, name, contiguous=False)
        if t.stride(-1) != 1:
            raise ValueError(f"{name} rows must be contiguous along head_dim")
    _need(key_pool, BF16, "key_pool")
    _need(value_pool, BF16, "value_pool")
    if q_out is not None:
        _need(q_out, BF16, "q_out")
    if write_slots.dtype != torch.long:
        raise ValueError("write_slots must be int64")
    pool_slots = key_pool.shape[0] * key_pool.shape[1]
    rc = lib().hb_qk_norm_rope_append(
        _ptr(q), q.stride(0) if q is not None else 0, q.stride(1) if q is not None else 0,
        k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
        _ptr(q_scale), _ptr(k_scale), float(eps), _ptr(cos), _ptr(sin), cos.shape[0] if cos is not None else 0,
        _ptr(positions), write_slots.data_ptr(), _ptr(q_out), key_pool.data_ptr(), value_pool.data_ptr(),
        pool_slots, tokens, heads, kv_heads, dim, _stream(k.device))
    _native.check(rc, "hb_qk_norm_rope_append")


def workspace_bytes(partial_records: int, heads: int, head_dim: int) -> int:
    return int(lib().hb_attention_workspace_bytes(partial_records, heads, head_dim))


def paged_attention(q: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, meta, out: torch.Tensor,
                    *, scale: float | None = None) -> torch.Tensor:
    """Kernel (c): ``q [T, H, d]`` against the paged pool described by ``meta``
    (a prepared paged batch cache); writes ``out [T, H, d]``. A cache in capacity mode
    passes its device work counts and launches grids sized to its capacities."""
    _need(q, BF16, "q")
    _need(out, BF16, "out")
    _need(key_pool, BF16, "key_pool")
    _need(value_pool, BF16, "value_pool")
    tokens, heads, dim = q.shape
    kv_heads = key_pool.shape[2]
    scale = dim ** -0.5 if scale is None else scale
    ws = meta.workspace
    rc = lib().hb_paged_attention(
        q.data_ptr(), key_pool.data_ptr(), value_pool.data_ptr(), key_pool.shape[0], key_pool.shape[1],
        meta.block_table.data_ptr(), meta.block_table.shape[1], meta.cu_seq_q.data_ptr(), meta.seqused_k.data_ptr(),
        meta.batch_size, meta.row_records.data_ptr(),
        meta.decode_items.data_ptr(), meta.launch_decode_items, meta.prefill_items.data_ptr(),
        meta.launch_prefill_items, meta.prefix_items.data_ptr(), meta.launch_prefix_items,
        _ptr(meta.attention_counts), meta.launch_partial_records, meta.split_keys, tokens,
        heads, kv_heads, dim, float(scale),
        _ptr(ws), ws.numel() if ws is not None else 0, out.data_ptr(), _stream(q.device))
    _native.check(rc, "hb_paged_attention")
    return out


def rmsnorm(x: torch.Tensor, scale: torch.Tensor, eps: float, *, out: torch.Tensor | None = None,
            row_index: torch.Tensor | None = None) -> torch.Tensor:
    """Row RMSNorm of ``x [rows, hidden]`` (rows gathered by ``row_index`` first)."""
    _need(x, BF16, "x")
    _need(scale, torch.float32, "scale")
    rows = x.shape[0] if row_index is None else row_index.shape[0]
    if out is None:
        out = torch.empty(rows, x.shape[1], dtype=BF16, device=x.device)
    if row_index is not None and row_index.dtype != torch.long:
        raise ValueError("row_index must be int64")
    rc = lib().hb_rmsnorm(x.data_ptr(), x.shape[0], _ptr(row_index), scale.data_ptr(), float(eps), out.data_ptr(),
                          rows, x.shape[1], _stream(x.device))
    _native.check(rc, "hb_rmsnorm")
    return out


def add_rmsnorm(x: torch.Tensor, y: torch.Tensor, scale: torch.Tensor, eps: float, sum_out: torch.Tensor,
                norm_out: torch.Tensor) -> None:
    """``sum_out = bf16(x + y)``; ``norm_out = rmsnorm(sum_out)``."""
    for name, t in (("x", x), ("y", y), ("sum_out", sum_out), ("norm_out", norm_out)):
        _need(t, BF16, name)
    _need(scale, torch.float32, "scale")
    rc = lib().hb_add_rmsnorm(x.data_ptr(), y.data_ptr(), scale.data_ptr(), float(eps), sum_out.data_ptr(),
                              norm_out.data_ptr(), x.shape[0], x.shape[1], _stream(x.device))
    _native.check(rc, "hb_add_rmsnorm")


def swiglu(gate_up: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    _need(gate_up, BF16, "gate_up")
    _need(out, BF16, "out")
    if gate_up.shape[1] != 2 * out.shape[1] or gate_up.shape[0] != out.shape[0]:
        raise ValueError("gate_up must be [rows, 2 * inter] for out [rows, inter]")
    rc = lib().hb_swiglu(gate_up.data_ptr(), out.data_ptr(), gate_up.shape[0], out.shape[1], _stream(out.device))
    _native.check(rc, "hb_swiglu")
    return out


def gemm_swiglu(x: torch.Tensor, w_gate_up: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """``silu(x Wg^T) * (x Wu^T)`` with the reference's bf16 rounding points, for ``x [m, k]``
    and the fused ``w_gate_up [2 * inter, k]`` (gate rows then up rows), on tcgen05."""
    _need(x, BF16, "x")
    _need(w_gate_up, BF16, "w_gate_up")
    m, k = x.shape
    inter = w_gate_up.shape[0] // 2
    if w_gate_up.shape[1] != k or w_gate_up.shape[0] != 2 * inter:
        raise ValueError("w_gate_up must be [2 * intermediate, hidden] matching x")
    if out is None:
        out = torch.empty((m, inter), dtype=BF16, device=x.device)
    rc = lib().hb_gemm_swiglu(x.data_ptr(), m, k, w_gate_up.data_ptr(), inter, out.data_ptr(), _stream(x.device))
    _native.check(rc, "hb_gemm_swiglu")
    return out


# Buffers a larger call replaced: kept alive, since a CUDA graph captured earlier still
# launches kernels on their addresses.
_RETIRED: list[torch.Tensor] = []


_ARGMAX_KEYS: dict[torch.device, torch.Tensor] = {}


def lm_head_argmax(x: torch.Tensor, weight: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """Greedy token ids ``argmax_j bf16(x[r] . weight[j])`` (int64 ``[m]``; ties to the lowest id)
    for the final-normed logit rows ``x [m, k]`` against the tied ``weight [vocab, k]``, with the
    argmax in the tcgen05 GEMM's epilogue: the logits are never written (hb_lm_head_argmax)."""
    _need(x, BF16, "x")
    _need(weight, BF16, "weight")
    m, k = x.shape
    if weight.shape[1] != k:
        raise ValueError("weight must be [vocab, hidden] matching x")
    dev = x.device
    keys = _ARGMAX_KEYS.get(dev)
    if keys is None or keys.numel() < m:
        if torch.cuda.is_current_stream_capturing():
            # Memory allocated under capture belongs to the graph's pool; the keys outlive graphs.
            raise RuntimeError("lm_head_argmax: run one call of this size before capturing it")
        # Zeroed once; every call leaves the keys it used at zero.
        if keys is not None:
            _RETIRED.append(keys)
        keys = _ARGMAX_KEYS[dev] = torch.zeros(max(m, 256), dtype=torch.int64, device=dev)
    if out is None:
        out = torch.empty(m, dtype=torch.long, device=dev)
    rc = lib().hb_lm_head_argmax(x.data_ptr(), m, k, weight.data_ptr(), weight.shape[0], keys.data_ptr(),
                                 out.data_ptr(), _stream(dev))
    _native.check(rc, "hb_lm_head_argmax")
    return out


def _together(device: torch.device, **tensors: torch.Tensor | None) -> None:
    """Every given tensor on ``device``, contiguous."""
    for name, t in tensors.items():
        if t is not None:
            if t.device != device:
                raise ValueError(f"{name} must be on {device}, got {t.device}")
            if not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous")


_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _call(fn, name: str, device: int, *args) -> None:
    """Run an entry point on the current stream of CUDA device ``device``, with that device current."""
    stream = _raw_stream(device) if _raw_stream is not None else torch.cuda.current_stream(device).cuda_stream
    if _get_device() == device:
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc:
        _native.check(rc, name)


# The operators below test their arguments in one expression, which is all that a call in order
# pays for (each _need costs 0.3 us of host time, more than a decode step's smallest kernels can
# hide; get_device(), -1 for host tensors, costs half of comparing devices); only when it fails, a
# second pass finds out which argument to name.
I32, F32 = torch.int32, torch.float32


def _refuse_linear_w4(x, packed, scales, zeros, out) -> None:
    _need(x, BF16, "x", contiguous=False)
    _need(packed, I32, "packed")
    _need(scales, BF16, "scales")
    if x.dim() != 2 or packed.dim() != 2 or scales.dim() != 2:
        raise ValueError("x, packed and scales must be 2-D")
    m, k = x.shape
    n, groups = packed.shape[0], scales.shape[0]
    if packed.shape[1] * 8 != k or scales.shape[1] != n or groups == 0 or k % groups:
        raise ValueError("packed must be [n, k / 8] and scales [k / group, n] for x [m, k]")
    if x.stride(1) != 1:
        raise ValueError("x rows must be contiguous")
    if zeros is not None:
        _need(zeros, torch.uint8, "zeros")
        if zeros.shape != scales.shape:
            raise ValueError("zeros must have the shape of scales")
    if out is not None:
        _need(out, BF16, "out")
        if out.shape != (m, n):
            raise ValueError("out must be [m, n]")
    _together(x.device, packed=packed, scales=scales, zeros=zeros, out=out)
    raise ValueError("linear_w4 arguments do not fit together")


def linear_w4(x: torch.Tensor, packed: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """``x [m, k] @ W^T`` (bf16 ``[m, n]``) for a weight held in 4 bits: ``W[j, i] = (q[j, i] -
    z[g, j]) * scales[g, j]``, ``g = i // group``. ``packed`` int32 ``[n, k / 8]`` (word c: even i's
    in the low half, odd i's in the high half, see hb_linear_w4), ``scales`` bf16 ``[k / group, n]``,
    ``zeros`` uint8 ``[k / group, n]`` (None: 8); groups of 32, 64 or 128. ``x`` may have any row
    stride that keeps its rows 16-byte aligned. ``helios_b200.w4.quantize_w4`` makes the three
    tensors from a weight. Returns ``out`` (apart from ``x``), or a new tensor."""
    dev = x.get_device()
    if not (x.is_cuda and x.dtype is BF16 and packed.dtype is I32 and scales.dtype is BF16
            and packed.get_device() == dev and scales.get_device() == dev and packed.is_contiguous()
            and scales.is_contiguous() and x.dim() == 2 and packed.dim() == 2 and scales.dim() == 2):
        _refuse_linear_w4(x, packed, scales, zeros, out)
    m, k = x.shape
    n, words = packed.shape
    groups, scale_n = scales.shape
    if not (words * 8 == k and scale_n == n and groups and k % groups == 0 and x.stride(1) == 1
            and (zeros is None or (zeros.dtype is torch.uint8 and zeros.get_device() == dev and zeros.is_contiguous()
                                   and zeros.shape == scales.shape))
            and (out is None or (out.dtype is BF16 and out.get_device() == dev and out.is_contiguous()
                                 and out.shape == (m, n)))):
        _refuse_linear_w4(x, packed, scales, zeros, out)
    if out is None:
        out = x.new_empty((m, n))
    _call(lib().hb_linear_w4, "hb_linear_w4", dev, x.data_ptr(), x.stride(0) if m > 1 else k, m, k, packed.data_ptr(),
          scales.data_ptr(), None if zeros is None else zeros.data_ptr(), n, k // groups, out.data_ptr())
    return out


BLOCK_KEYS = 64        # keys per block of the sparse attention
MAX_TOP_BLOCKS = 1024  # blocks it attends to at most
MAX_SPARSE_TOKENS = 393_216  # keys that a row's block table covers at most


def _check_bounds(key_pool: torch.Tensor, bounds: torch.Tensor) -> None:
    _need(key_pool, BF16, "key_pool")
    _need(bounds, BF16, "bounds")
    if key_pool.dim() != 4:
        raise ValueError("key_pool must be [pages, page, kv_heads, head_dim]")
    pages, page, heads, dim = key_pool.shape
    if bounds.shape != (pages, heads, page // BLOCK_KEYS, 2, dim):
        raise ValueError("bounds must be [pages, kv_heads, page / 64, 2, head_dim] for the key pool")


def _refuse_bounds(key_pool, bounds, block_table, cu_seq_q, seqused_k, token_row) -> None:
    _check_bounds(key_pool, bounds)
    for name, t in (("block_table", block_table), ("cu_seq_q", cu_seq_q), ("seqused_k", seqused_k),
                    ("token_row", token_row)):
        _need(t, I32, name)
    _together(key_pool.device, bounds=bounds, block_table=block_table, cu_seq_q=cu_seq_q, seqused_k=seqused_k,
              token_row=token_row)
    raise ValueError("block_table must be [rows, width], with rows + 1 entries in cu_seq_q and rows in seqused_k")


def key_block_bounds(key_pool: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor,
                     cu_seq_q: torch.Tensor, seqused_k: torch.Tensor, token_row: torch.Tensor) -> torch.Tensor:
    """Bring ``bounds`` up to date with the keys a tick appended (hb_key_block_bounds): one layer's
    ``key_pool [pages, page, Hkv, d]`` and ``bounds [pages, Hkv, page / 64, 2, d]``, with the tick's
    ``block_table [rows, width]``, ``cu_seq_q [rows + 1]``, ``seqused_k [rows]`` and ``token_row
    [tokens]`` (all int32). Only blocks holding new positions are written. Returns ``bounds``."""
    dev = key_pool.get_device()
    if not (key_pool.is_cuda and key_pool.dtype is BF16 and bounds.dtype is BF16 and block_table.dtype is I32
            and cu_seq_q.dtype is I32 and seqused_k.dtype is I32 and token_row.dtype is I32
            and bounds.get_device() == dev and block_table.get_device() == dev and cu_seq_q.get_device() == dev
            and seqused_k.get_device() == dev
            and token_row.get_device() == dev and key_pool.is_contiguous() and bounds.is_contiguous()
            and block_table.is_contiguous() and cu_seq_q.is_contiguous() and seqused_k.is_contiguous()
            and token_row.is_contiguous() and key_pool.dim() == 4 and block_table.dim() == 2):
        _refuse_bounds(key_pool, bounds, block_table, cu_seq_q, seqused_k, token_row)
    pages, page, heads, dim = key_pool.shape
    rows, width = block_table.shape
    if not (bounds.shape == (pages, heads, page // BLOCK_KEYS, 2, dim) and cu_seq_q.numel() == rows + 1
            and seqused_k.numel() == rows):
        _refuse_bounds(key_pool, bounds, block_table, cu_seq_q, seqused_k, token_row)
    _call(lib().hb_key_block_bounds, "hb_key_block_bounds", dev, key_pool.data_ptr(), bounds.data_ptr(), pages, page,
          block_table.data_ptr(), width, cu_seq_q.data_ptr(), seqused_k.data_ptr(), token_row.data_ptr(), rows,
          token_row.numel(), heads, dim)
    return bounds


def _refuse_sparse(q, key_pool, value_pool, bounds, block_table, seqused_k, cu_seq_q, out, selected,
                   top_blocks) -> None:
    _need(q, BF16, "q")
    _need(value_pool, BF16, "value_pool")
    _check_bounds(key_pool, bounds)
    _need(block_table, I32, "block_table")
    _need(seqused_k, I32, "seqused_k")
    if q.dim() != 3 or value_pool.shape != key_pool.shape or q.shape[2] != key_pool.shape[3]:
        raise ValueError("q must be [rows, heads, head_dim], and both pools must match each other and its head_dim")
    if block_table.dim() != 2 or seqused_k.numel() != block_table.shape[0]:
        raise ValueError("block_table and seqused_k need one row per sequence")
    if cu_seq_q is not None:
        _need(cu_seq_q, I32, "cu_seq_q")
        if cu_seq_q.numel() != block_table.shape[0] + 1:
            raise ValueError("cu_seq_q needs rows + 1 entries")
    elif block_table.shape[0] != q.shape[0]:
        raise ValueError("without cu_seq_q, q needs one token per row")
    if out is not None:
        _need(out, BF16, "out")
        if out.shape != q.shape:
            raise ValueError("out must have the shape of q")
    if selected is not None:
        _need(selected, I32, "selected")
        if selected.shape != (block_table.shape[0], key_pool.shape[2], top_blocks):
            raise ValueError("selected must be [rows, kv_heads, top_blocks]")
    _together(q.device, key_pool=key_pool, value_pool=value_pool, bounds=bounds, block_table=block_table,
              seqused_k=seqused_k, cu_seq_q=cu_seq_q, out=out, selected=selected)
    raise ValueError("sparse_paged_attention with cu_seq_q needs out")


def sparse_paged_attention(q: torch.Tensor, key_pool: torch.Tensor, value_pool: torch.Tensor, bounds: torch.Tensor,
                           block_table: torch.Tensor, seqused_k: torch.Tensor, out: torch.Tensor | None = None, *,
                           top_blocks: int, sink_blocks: int = 1, recent_blocks: int = 2,
                           scale: float | None = None, selected: torch.Tensor | None = None,
                           cu_seq_q: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of one query token per row, ``q [rows, H, d]``, over the ``top_blocks`` 64-key blocks
    that the ``bounds`` of key_block_bounds select for it and each KV head, the row's first
    ``sink_blocks`` and last ``recent_blocks`` blocks always among them (hb_sparse_paged_attention).
    ``selected`` (int32 ``[rows, Hkv, top_blocks]``) gets the blocks in ascending order, then -1.
    Returns ``out [rows, H, d]``, or a new tensor; a row without keys gives zeros. With ``cu_seq_q``
    (int32 ``[rows + 1]``, as tick_pack writes it) ``q`` and ``out`` are ``[tokens, H, d]``, row r's token is
    ``cu_seq_q[r]``, and rows with other than one token are left as ``out`` has them (it has to be given then)."""
    dev = q.get_device()
    refuse = (q, key_pool, value_pool, bounds, block_table, seqused_k, cu_seq_q, out, selected, top_blocks)
    if not (q.is_cuda and q.dtype is BF16 and key_pool.dtype is BF16 and value_pool.dtype is BF16
            and bounds.dtype is BF16 and block_table.dtype is I32 and seqused_k.dtype is I32
            and key_pool.get_device() == dev and value_pool.get_device() == dev and bounds.get_device() == dev
            and block_table.get_device() == dev and seqused_k.get_device() == dev and q.is_contiguous()
            and key_pool.is_contiguous() and value_pool.is_contiguous() and bounds.is_contiguous()
            and block_table.is_contiguous() and seqused_k.is_contiguous() and q.dim() == 3 and key_pool.dim() == 4
            and block_table.dim() == 2):
        _refuse_sparse(*refuse)
    tokens, heads, dim = q.shape
    pool_shape = key_pool.shape
    pages, page, kv_heads, pool_dim = pool_shape
    rows, width = block_table.shape
    if not (value_pool.shape == pool_shape and dim == pool_dim and seqused_k.numel() == rows
            and (tokens == rows if cu_seq_q is None else
                 cu_seq_q.dtype is I32 and cu_seq_q.get_device() == dev and cu_seq_q.is_contiguous()
                 and cu_seq_q.numel() == rows + 1 and out is not None)
            and bounds.shape == (pages, kv_heads, page // BLOCK_KEYS, 2, dim)
            and (out is None or (out.dtype is BF16 and out.get_device() == dev and out.is_contiguous()
                                 and out.shape == q.shape))
            and (selected is None or (selected.dtype is I32 and selected.get_device() == dev
                                      and selected.is_contiguous()
                                      and selected.shape == (rows, kv_heads, top_blocks)))):
        _refuse_sparse(*refuse)
    if out is None:
        out = torch.empty_like(q)
    _call(lib().hb_sparse_paged_attention, "hb_sparse_paged_attention", dev, q.data_ptr(), key_pool.data_ptr(),
          value_pool.data_ptr(), bounds.data_ptr(), pages, page, block_table.data_ptr(), width, seqused_k.data_ptr(),
          None if cu_seq_q is None else cu_seq_q.data_ptr(), rows, heads, kv_heads, dim, top_blocks, sink_blocks,
          recent_blocks, dim ** -0.5 if scale is None else scale,
          None if selected is None else selected.data_ptr(), out.data_ptr())
    return out


def _refuse_controls(logits, repetition, frequency, presence, history, slots, lengths, prompt_lengths, bias, mask,
                     mask_rows, out) -> None:
    _need(logits, BF16, "logits", contiguous=False)
    if logits.dim() != 2 or logits.stride(1) != 1:
        raise ValueError("logits must be [rows, V] with contiguous rows")
    rows, vocab = logits.shape
    for name, t in (("repetition", repetition), ("frequency", frequency), ("presence", presence)):
        if t is not None:
            _need(t, F32, name)
            if t.numel() != rows:
                raise ValueError(f"{name} needs one value per row")
    if history is not None:
        if slots is None or lengths is None or prompt_lengths is None:
            raise ValueError("a history needs slots, lengths and prompt_lengths")
        for name, t in (("history", history), ("slots", slots), ("lengths", lengths),
                        ("prompt_lengths", prompt_lengths)):
            _need(t, I32, name)
        if (history.dim() != 2 or slots.numel() != rows or lengths.numel() != history.shape[0]
                or prompt_lengths.numel() != history.shape[0]):
            raise ValueError("history must be [slots, width], with one entry of slots per row and of lengths and "
                             "prompt_lengths per history row")
    offsets = tokens = values = None
    if bias is not None:
        offsets, tokens, values = bias
        _need(offsets, I32, "bias offsets")
        _need(tokens, I32, "bias tokens")
        _need(values, F32, "bias values")
        if offsets.numel() != rows + 1 or tokens.numel() != values.numel():
            raise ValueError("bias needs rows + 1 offsets and as many values as tokens")
    if mask is not None:
        _need(mask, I32, "mask")
        if mask_rows is None:
            raise ValueError("a mask needs mask_rows")
        _need(mask_rows, I32, "mask_rows")
        if mask.dim() != 2 or mask.shape[1] != (vocab + 31) // 32 or mask_rows.numel() != rows:
            raise ValueError("mask must be [masks, ceil(V / 32)] and mask_rows [rows]")
    if out is not None and out is not logits:
        _need(out, BF16, "out")
        if out.shape != logits.shape:
            raise ValueError("out must have the shape of logits")
        _together(logits.device, out=out)
    _together(logits.device, repetition=repetition, frequency=frequency, presence=presence, history=history,
              slots=slots, lengths=lengths, prompt_lengths=prompt_lengths, bias_offsets=offsets, bias_tokens=tokens,
              bias_values=values, mask=mask, mask_rows=mask_rows)
    raise ValueError("control_logits arguments do not fit together")


def control_logits(logits: torch.Tensor, *, repetition: torch.Tensor | None = None,
                   frequency: torch.Tensor | None = None, presence: torch.Tensor | None = None,
                   history: torch.Tensor | None = None, slots: torch.Tensor | None = None,
                   lengths: torch.Tensor | None = None, prompt_lengths: torch.Tensor | None = None,
                   bias: tuple[torch.Tensor, torch.Tensor, torch.Tensor] | None = None,
                   mask: torch.Tensor | None = None, mask_rows: torch.Tensor | None = None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Penalties, biases and grammar masks on ``logits [rows, V]`` (bf16, rows may be strided), as
    hb_control_logits defines them. ``repetition`` / ``frequency`` / ``presence``: fp32 ``[rows]``
    (None: 1, 0, 0), applied to the tokens of ``history`` (int32 ``[slots, width]``; row r's is
    ``history[slots[r], :lengths[slots[r]]]``, its first ``prompt_lengths[slots[r]]`` the prompt;
    slot -1: none). ``bias``: int32 offsets ``[rows + 1]``, int32 tokens (ascending within a row) and
    fp32 values. ``mask`` int32 ``[masks, ceil(V / 32)]`` with ``mask_rows`` int32 ``[rows]`` (-1: none).
    Returns ``out`` (``logits`` itself works in place), or a new tensor."""
    dev = logits.get_device()
    args = (repetition, frequency, presence, history, slots, lengths, prompt_lengths, bias, mask, mask_rows, out)
    if not (logits.is_cuda and logits.dtype is BF16 and logits.dim() == 2 and logits.stride(1) == 1):
        _refuse_controls(logits, *args)
    rows, vocab = logits.shape
    for t in (repetition, frequency, presence):
        if t is not None and not (t.dtype is F32 and t.get_device() == dev and t.numel() == rows and t.is_contiguous()):
            _refuse_controls(logits, *args)
    history_rows = history_width = entries = masks = 0
    history_ptrs = bias_ptrs = (None, None, None, None)
    mask_ptr = mask_rows_ptr = None
    if history is not None:
        if slots is None or lengths is None or prompt_lengths is None or history.dim() != 2:
            _refuse_controls(logits, *args)
        history_rows, history_width = history.shape
        if not (history.dtype is I32 and slots.dtype is I32 and lengths.dtype is I32 and prompt_lengths.dtype is I32
                and history.get_device() == dev and slots.get_device() == dev and lengths.get_device() == dev
                and prompt_lengths.get_device() == dev and history.is_contiguous() and slots.is_contiguous()
                and lengths.is_contiguous() and prompt_lengths.is_contiguous() and slots.numel() == rows
                and lengths.numel() == history_rows and prompt_lengths.numel() == history_rows):
            _refuse_controls(logits, *args)
        history_ptrs = (history.data_ptr(), slots.data_ptr(), lengths.data_ptr(), prompt_lengths.data_ptr())
    if bias is not None:
        offsets, tokens, values = bias
        entries = tokens.numel()
        if not (offsets.dtype is I32 and tokens.dtype is I32 and values.dtype is F32 and offsets.get_device() == dev
                and tokens.get_device() == dev and values.get_device() == dev and offsets.is_contiguous()
                and tokens.is_contiguous() and values.is_contiguous() and offsets.numel() == rows + 1
                and values.numel() == entries):
            _refuse_controls(logits, *args)
        bias_ptrs = (offsets.data_ptr(), tokens.data_ptr(), values.data_ptr())
    if mask is not None:
        if not (mask_rows is not None and mask.dtype is I32 and mask_rows.dtype is I32 and mask.get_device() == dev
                and mask_rows.get_device() == dev and mask.is_contiguous() and mask_rows.is_contiguous()
                and mask.dim() == 2 and mask.shape[1] == (vocab + 31) // 32 and mask_rows.numel() == rows):
            _refuse_controls(logits, *args)
        masks, mask_ptr, mask_rows_ptr = mask.shape[0], mask.data_ptr(), mask_rows.data_ptr()
    if out is None:
        out = torch.empty_like(logits) if logits.is_contiguous() else logits.new_empty((rows, vocab))
    elif out is not logits and not (out.dtype is BF16 and out.get_device() == dev and out.shape == logits.shape
                                    and out.is_contiguous()):
        _refuse_controls(logits, *args)
    _call(lib().hb_control_logits, "hb_control_logits", dev, logits.data_ptr(), logits.stride(0) if rows > 1 else vocab,
          rows, vocab, _ptr(repetition), _ptr(frequency), _ptr(presence), history_ptrs[0], history_rows,
          history_width, history_ptrs[1], history_ptrs[2], history_ptrs[3], bias_ptrs[0], bias_ptrs[1], bias_ptrs[2],
          entries, mask_ptr, masks, mask_rows_ptr, out.data_ptr(), out.stride(0) if rows > 1 else vocab)
    return out


def embedding(ids: torch.Tensor, table: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    if ids.dtype != torch.long or not ids.is_cuda or not ids.is_contiguous():
        raise ValueError("token ids must be a contiguous CUDA int64 tensor")
    _need(table, BF16, "table")
    _need(out, BF16, "out")
    rc = lib().hb_embedding(ids.data_ptr(), table.data_ptr(), table.shape[0], out.data_ptr(), ids.numel(),
                            table.shape[1], _stream(out.device))
    _native.check(rc, "hb_embedding")
    return out


def page_copy(storage: torch.Tensor, src_pages: torch.Tensor, dst_pages: torch.Tensor) -> None:
    """Copy pages ``src -> dst`` in every pool tensor of ``storage [tensors, P, ...]``."""
    if src_pages.dtype != torch.int32 or dst_pages.dtype != torch.int32:
        raise ValueError("page lists must be int32")
    tensors, num_pages = storage.shape[0], storage.shape[1]
    page_bytes = storage[0, 0].numel() * storage.element_size()
    rc = lib().hb_page_copy(storage.data_ptr(), storage.stride(0) * storage.element_size(), tensors, page_bytes,
                            num_pages, src_pages.data_ptr(), dst_pages.data_ptr(), src_pages.numel(),
                            _stream(storage.device))
    _native.check(rc, "hb_page_copy")


def sample(logits: torch.Tensor, temperature: torch.Tensor, top_p: torch.Tensor, uniforms: torch.Tensor,
           out: torch.Tensor | None = None) -> torch.Tensor:
    """Kernel (d): one token id per row of bf16 ``logits [rows, V]`` (row stride may exceed V)."""
    _need(logits, BF16, "logits", contiguous=False)
    if logits.stride(1) != 1:
        raise ValueError("logit rows must be contiguous")
    for name, t in (("temperature", temperature), ("top_p", top_p), ("uniforms", uniforms)):
        _need(t, torch.float32, name)
    rows, vocab = logits.shape
    if out is None:
        out = torch.empty(rows, dtype=torch.long, device=logits.device)
    rc = lib().hb_sample(logits.data_ptr(), logits.stride(0), rows, vocab, temperature.data_ptr(), top_p.data_ptr(),
                         uniforms.data_ptr(), out.data_ptr(), _stream(logits.device))
    _native.check(rc, "hb_sample")
    return out


def verify_drafts(tokens: torch.Tensor, cu_seq_q: torch.Tensor, logit_offsets: torch.Tensor,
                  predictions: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Speculative verification on the device: ``(accepted [B] int32, emitted [logit rows]
    int64)``; row r's emitted tokens are ``emitted[logit_offsets[r] : logit_offsets[r] +
    accepted[r] + 1]`` (engine.py:507-520)."""
    _need(tokens, torch.long, "tokens")
    _need(cu_seq_q, torch.int32, "cu_seq_q")
    _need(logit_offsets, torch.int32, "logit_offsets")
    _need(predictions, torch.long, "predictions")
    rows = cu_seq_q.numel() - 1
    if logit_offsets.numel() != rows + 1:
        raise ValueError("logit_offsets needs one entry per row plus one")
    accepted = torch.empty(rows, dtype=torch.int32, device=tokens.device)
    emitted = torch.zeros(predictions.numel(), dtype=torch.long, device=tokens.device)
    rc = lib().hb_verify_drafts(tokens.data_ptr(), cu_seq_q.data_ptr(), logit_offsets.data_ptr(),
                                predictions.data_ptr(), rows, accepted.data_ptr(), emitted.data_ptr(),
                                _stream(tokens.device))
    _native.check(rc, "hb_verify_drafts")
    return accepted, emitted
