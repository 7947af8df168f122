"""The paged KV cache held in 8 bits: store, load and decode attention.

The counterparts of ``store_kvcache`` (worker/kernels/kvcache_mgmt.py:298-478) and ``paged_attention``
(worker/kernels/paged_attn.py:700-1015) for a pool in half the bytes; the reference's pools are fp16 only.  A pool is

    k_cache, v_cache    int8 or float8_e4m3fn  [num_blocks, num_layers, num_kv_heads, block_size, head_dim]
    k_scale, v_scale    float32                [num_blocks, num_layers, num_kv_heads]

and elastic chunks are lists of such tensors (``*_new``), addressed as in the fp16 functions.  A code q stands for
``q * scale`` of its block, layer and head: int8 ``scale = amax / 127``, e4m3 the smallest power of two with
``amax <= 448 * scale``, with amax over the block's tokens.  Scales below the smallest normal fp32 number are 0, and a
block with a value that is not finite has the scale NaN, so that what is read back from it is NaN.

Rows (``k``, ``v``, ``q``) may be fp16, bf16 or fp32 and may be views of a fused projection: elements and heads
contiguous, tokens any distance apart.  Index tensors are contiguous int32 on the same device.  Nothing here
synchronises or allocates in the steady state; everything can be captured in a CUDA graph, where an attention call
brings its own scratch, so graphs share none.
"""
from __future__ import annotations

import struct

import torch

from ..._lib import MKV_MAX_SEGMENTS, MkvPoolQ8, check, lib
from ._common import raw_stream, require_cuda, workspace_q8

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}       # mkv_dtype
_CODES = {torch.int8: 1, torch.float8_e4m3fn: 2}                        # mkv_q8_code


def alloc_kvcache_q8(num_blocks: int, model_config, engine_config, dtype: torch.dtype = torch.int8, device="cuda"):
    """Zero-filled ``(k_cache, v_cache, k_scale, v_scale)`` of ``num_blocks`` blocks (a pool or an elastic chunk)."""
    if dtype not in _CODES:
        raise RuntimeError(f"unsupported 8-bit KV dtype {dtype}")
    shape = (num_blocks, model_config.num_layers, model_config.num_kv_heads, engine_config.block_size, model_config.head_dim)
    codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
    return (*codes, *[torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)])


# mkv_pool_q8, packed rather than assigned field by field: the header and the first segment's four pointers at once (each
# stands in front of an array), further segments' pointers one by one.
_FIELDS = (MkvPoolQ8.k_base.offset, MkvPoolQ8.v_base.offset, MkvPoolQ8.k_scale.offset, MkvPoolQ8.v_scale.offset)
_PACK = struct.Struct("6i2qQ%dxQ%dxQ%dxQ" % tuple(y - x - 8 for x, y in zip(_FIELDS, _FIELDS[1:]))).pack_into
_POINTER = struct.Struct("Q").pack_into


def _check_segment(k, v, ks, vs, dtype, shape, entries, dev):
    assert k.shape == shape and v.shape == shape and ks.numel() == entries and vs.numel() == entries, \
        "k_cache and v_cache have one shape, the scales one entry for each block, layer and head"
    assert k.dtype is dtype and v.dtype is dtype and ks.dtype is torch.float32 and vs.dtype is torch.float32
    assert k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
    assert k.get_device() == dev and v.get_device() == dev and ks.get_device() == dev and vs.get_device() == dev


def _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new, model_config,
          engine_config, num_blocks_org, chunk_blocks):
    """(descriptor, shape of the original pool, device index)"""
    dev = k_cache.get_device()
    if dev < 0:
        require_cuda(k_cache, "k_cache")
    dtype, shape = k_cache.dtype, k_cache.shape
    code = _CODES.get(dtype)
    if code is None:
        raise RuntimeError(f"unsupported 8-bit KV dtype {dtype}")
    blocks, layers, heads, bs, d = shape
    assert heads == model_config.num_kv_heads and d == model_config.head_dim and bs == engine_config.block_size
    _check_segment(k_cache, v_cache, k_scale, v_scale, dtype, shape, blocks * layers * heads, dev)
    n_new = len(k_cache_new)
    assert len(v_cache_new) == n_new and len(k_scale_new) == n_new and len(v_scale_new) == n_new
    pool = MkvPoolQ8()
    _PACK(pool, 0, 1 + n_new, code, layers, heads, bs, d, blocks, int(chunk_blocks) if n_new else 0, k_cache.data_ptr(),
          v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr())
    if n_new:
        if n_new + 1 > MKV_MAX_SEGMENTS:
            raise RuntimeError(f"too many elastic KV chunks ({n_new}); the library supports {MKV_MAX_SEGMENTS - 1}")
        if int(num_blocks_org) != blocks:
            raise RuntimeError("num_blocks_org is not the number of blocks of the original pool")
        chunk = torch.Size((int(chunk_blocks), layers, heads, bs, d))
        for j, parts in enumerate(zip(k_cache_new, v_cache_new, k_scale_new, v_scale_new)):
            if parts[0].shape != chunk:
                raise RuntimeError("elastic KV chunks must all hold kv_cache_new_block_size blocks of the pool's shape")
            _check_segment(*parts, dtype, chunk, chunk[0] * layers * heads, dev)
            for field, t in zip(_FIELDS, parts):
                _POINTER(pool, field + 8 * (1 + j), t.data_ptr())
    return pool, shape, dev


def _rows(x, heads, d, dev):
    """Distance of two tokens, in elements, of rows [tokens, heads, head_dim] whose elements and heads are contiguous."""
    shape, stride = x.shape, x.stride()
    assert len(shape) == 3 and shape[1] == heads and shape[2] == d, f"rows are [tokens, {heads}, {d}]"
    assert x.get_device() == dev, "rows are on another device than the cache"
    assert (stride[2] == 1 or d == 1) and (stride[1] == d or heads == 1), "elements and heads of a row are contiguous"
    return stride[0] if shape[0] > 1 else heads * d


def _ints(x, dev, n, name):
    assert x.dtype is torch.int32 and x.is_contiguous() and x.get_device() == dev and x.shape[0] >= n, \
        f"{name}: contiguous int32 on the cache's device, one for each sequence"
    return x.data_ptr()


def _table(x, dev):
    assert x.dtype is torch.int32 and x.is_contiguous() and x.get_device() == dev, "block_table: contiguous int32 on the cache's device"
    rows, cols = x.shape
    return x.data_ptr(), cols, rows


def _dtype(x):
    code = _DTYPES.get(x.dtype)
    if code is None:
        raise RuntimeError(f"unsupported dtype {x.dtype}")
    return code


def store_kvcache_q8(
    k: torch.Tensor,            # [num_tokens, num_kv_heads, head_dim]
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    k_cache_new: list,
    v_cache_new: list,
    k_scale_new: list,
    v_scale_new: list,
    block_table: torch.Tensor,  # [max_seqs_in_block_table, max_blocks_per_seq] int32
    model_config,
    engine_config,
    infer_state,
    cur_layer: int,
):
    """New K/V rows into the 8-bit pool, like ``store_kvcache``: the prefill tokens come first in ``k`` and ``v``, one
    row for each decoding sequence after them.

    A prompt's blocks take their scales from the prompt alone (slots behind its end keep their bytes).  A decoding
    sequence's newest token is appended: in the first slot of a block the scale starts from it, later the larger of the
    block's scale and the token's holds, and where that is the token's the older codes are rounded again.  A block that
    a call writes belongs to one sequence: a scale has one writer.  A sequence given more than once in one of the two
    parts: its last entry counts.  Sequences of length 0, ids outside the table and blocks outside the pool are skipped."""
    pool, shape, dev = _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new,
                             model_config, engine_config, infer_state.num_blocks_org, infer_state.kv_cache_new_block_size)
    heads, d = shape[2], shape[4]
    assert k.dtype is v.dtype and k.shape[0] == v.shape[0]
    dtype = _dtype(k)
    ks, vs = _rows(k, heads, d, dev), _rows(v, heads, d, dev)
    n_pre, n_dec = infer_state.num_prefill_seqs, infer_state.num_decoding_seqs
    n_tok = infer_state.num_prefill_tokens if n_pre > 0 else 0
    assert k.shape[0] >= n_tok + n_dec
    table, cols, rows = _table(block_table, dev)
    seq_ids = _ints(infer_state.seq_ids, dev, n_pre + n_dec, "seq_ids")
    stream = raw_stream(dev)
    if n_pre > 0:
        status = lib.mkv_store_kv_q8_prefill(
            dev, stream, k.data_ptr(), v.data_ptr(), ks, vs, dtype, n_tok, pool, table, cols, rows, seq_ids,
            _ints(infer_state.prefill_seq_start_locs, dev, n_pre, "prefill_seq_start_locs"),
            _ints(infer_state.prefill_seq_lens, dev, n_pre, "prefill_seq_lens"), n_pre,
            int(infer_state.max_prefill_len) or 1, cur_layer)     # (sizes the launch; 0 would be none)
        check(status, "mkv_store_kv_q8_prefill")
    if n_dec > 0:
        skip = n_tok * k.element_size()
        status = lib.mkv_store_kv_q8_decode(
            dev, stream, k.data_ptr() + skip * ks, v.data_ptr() + skip * vs, ks, vs, dtype, pool, table, cols, rows,
            seq_ids + 4 * n_pre, _ints(infer_state.decoding_seq_lens, dev, n_dec, "decoding_seq_lens"), n_dec, cur_layer)
        check(status, "mkv_store_kv_q8_decode")


def load_kvcache_q8(
    k: torch.Tensor,            # [rows, num_kv_heads, head_dim], written
    v: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    k_cache_new: list,
    v_cache_new: list,
    k_scale_new: list,
    v_scale_new: list,
    block_table: torch.Tensor,
    model_config,
    engine_config,
    seq_ids: torch.Tensor,      # [n] int32
    begins: torch.Tensor,       # [n] int32, first token of each range
    ends: torch.Tensor,         # [n] int32, behind its last token
    start_locs: torch.Tensor,   # [n] int32, row of its first token in k and v
    max_len: int,               # the longest range; sizes the launch only
    cur_layer: int,
):
    """Cached tokens back as rows: token t of ``seq_ids[i]``, ``begins[i] <= t < ends[i]``, becomes row
    ``start_locs[i] + t - begins[i]`` of ``k`` and ``v`` - a cached prefix for a prefill attention that wants contiguous
    rows, or a sequence on its way into another pool.  Values are the fp32 product of code and scale, rounded to the
    rows' type.  Rows that no range reaches, and rows of tokens whose page is not
    in the table or the pool, are left as they were."""
    pool, shape, dev = _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new,
                             model_config, engine_config, k_cache.shape[0], k_cache_new[0].shape[0] if len(k_cache_new) else 0)
    heads, d = shape[2], shape[4]
    assert k.dtype is v.dtype and k.shape[0] == v.shape[0]
    dtype = _dtype(k)
    ks, vs = _rows(k, heads, d, dev), _rows(v, heads, d, dev)
    n = seq_ids.shape[0]
    table, cols, rows = _table(block_table, dev)
    check(lib.mkv_load_kv_q8(
        dev, raw_stream(dev), k.data_ptr(), v.data_ptr(), ks, vs, dtype, k.shape[0], pool, table, cols, rows,
        _ints(seq_ids, dev, n, "seq_ids"), _ints(begins, dev, n, "begins"), _ints(ends, dev, n, "ends"),
        _ints(start_locs, dev, n, "start_locs"), n, int(max_len) or 1, cur_layer), "mkv_load_kv_q8")


def paged_attention_q8(
    q: torch.Tensor,            # [num_decoding_seqs, num_q_heads, head_dim]
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    k_scale: torch.Tensor,
    v_scale: torch.Tensor,
    k_cache_new: list,
    v_cache_new: list,
    k_scale_new: list,
    v_scale_new: list,
    block_table: torch.Tensor,
    model_config,
    engine_config,
    infer_state,
    cur_layer: int,
    o: torch.Tensor,            # [num_decoding_seqs, num_q_heads(*)head_dim], written
):
    """Decode attention over the 8-bit pool, like ``paged_attention``: softmax(scale * q K^T) V of every decoding
    sequence's one query token over its ``decoding_seq_lens`` cached tokens, with scores and sums in fp32, rounded once.

    Rows of sequences of length 0 are left as they were.  A page that is not in the table or the pool takes no part
    (and is reported by ``read_attn_error_flags``); a row that is left without any token is NaN.
    ``infer_state.max_decoding_len`` sizes the launch: lengths above it (a captured step whose sequences grew) are
    attended in full."""
    batch = infer_state.num_decoding_seqs
    if batch == 0:
        return
    pool, shape, dev = _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new,
                             model_config, engine_config, infer_state.num_blocks_org, infer_state.kv_cache_new_block_size)
    hq, hkv, bs, d = model_config.num_q_heads, shape[2], shape[3], shape[4]
    dtype = _dtype(q)
    q_stride = _rows(q, hq, d, dev)
    assert q.shape[0] >= batch
    assert o.dtype is q.dtype and o.is_contiguous() and o.get_device() == dev and o.numel() >= batch * hq * d
    n_pre = infer_state.num_prefill_seqs
    table, cols, rows = _table(block_table, dev)
    seq_ids = _ints(infer_state.seq_ids, dev, n_pre + batch, "seq_ids") + 4 * n_pre
    lens = _ints(infer_state.decoding_seq_lens, dev, batch, "decoding_seq_lens")
    max_len = infer_state.max_decoding_len or engine_config.max_blocks_per_seq * bs
    stream = raw_stream(dev)
    ws, ws_bytes = workspace_q8(dev, stream, batch, hq, hkv, d)
    check(lib.mkv_paged_attention_q8(
        dev, stream, q.data_ptr(), q_stride, o.data_ptr(), dtype, pool, table, cols, rows, seq_ids, lens, batch, hq,
        cur_layer, infer_state.softmax_scale, max_len, ws.data_ptr(), ws_bytes), "mkv_paged_attention_q8")
