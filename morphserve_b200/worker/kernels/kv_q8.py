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

import ctypes as C

import torch

from ..._lib import MKV_MAX_SEGMENTS, MkvPoolQ8, check, lib
from ._common import device_and_stream, require_cuda, workspace_q8

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}       # mkv_dtype
_CODES = {torch.int8: 1, torch.float8_e4m3fn: 2}                        # mkv_q8_code


def alloc_kvcache_q8(num_blocks: int, model_config, engine_config, dtype: torch.dtype = torch.int8, device="cuda"):
    """Zero-filled ``(k_cache, v_cache, k_scale, v_scale)`` of ``num_blocks`` blocks (a pool or an elastic chunk)."""
    if dtype not in _CODES:
        raise RuntimeError(f"unsupported 8-bit KV dtype {dtype}")
    shape = (num_blocks, model_config.num_layers, model_config.num_kv_heads, engine_config.block_size, model_config.head_dim)
    codes = [torch.zeros(shape, dtype=torch.int8, device=device).view(dtype) for _ in range(2)]
    return (*codes, *[torch.zeros(shape[:3], dtype=torch.float32, device=device) for _ in range(2)])


def _segment(pool, i, k, v, ks, vs, dtype, device):
    assert k.dtype == v.dtype == dtype and ks.dtype == vs.dtype == torch.float32
    assert k.shape == v.shape and ks.shape == vs.shape and k.shape[:3] == ks.shape
    assert k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous()
    assert k.device == device and v.device == device and ks.device == device and vs.device == device
    pool.k_base[i] = k.data_ptr()
    pool.v_base[i] = v.data_ptr()
    pool.k_scale[i] = ks.data_ptr()
    pool.v_scale[i] = vs.data_ptr()


def _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new, model_config,
          engine_config, num_blocks_org, chunk_blocks) -> MkvPoolQ8:
    require_cuda(k_cache, "k_cache")
    dtype = k_cache.dtype
    code = _CODES.get(dtype)
    if code is None:
        raise RuntimeError(f"unsupported 8-bit KV dtype {dtype}")
    n_new = len(k_cache_new)
    if n_new + 1 > MKV_MAX_SEGMENTS:
        raise RuntimeError(f"too many elastic KV chunks ({n_new}); the library supports {MKV_MAX_SEGMENTS - 1}")
    assert len(v_cache_new) == n_new and len(k_scale_new) == n_new and len(v_scale_new) == n_new
    blocks, layers, heads, bs, d = k_cache.shape
    assert heads == model_config.num_kv_heads and d == model_config.head_dim and bs == engine_config.block_size
    pool = MkvPoolQ8()
    pool.num_segments = 1 + n_new
    pool.code = code
    pool.num_layers = layers
    pool.num_kv_heads = heads
    pool.block_size = bs
    pool.head_dim = d
    pool.num_blocks_org = blocks
    _segment(pool, 0, k_cache, v_cache, k_scale, v_scale, dtype, k_cache.device)
    if n_new:
        if int(num_blocks_org) != blocks:
            raise RuntimeError("num_blocks_org is not the number of blocks of the original pool")
        pool.chunk_blocks = int(chunk_blocks)
        for j in range(n_new):
            if tuple(k_cache_new[j].shape) != (pool.chunk_blocks, layers, heads, bs, d):
                raise RuntimeError("elastic KV chunks must all hold kv_cache_new_block_size blocks of the pool's shape")
            _segment(pool, 1 + j, k_cache_new[j], v_cache_new[j], k_scale_new[j], v_scale_new[j], dtype, k_cache.device)
    return pool


def _rows(x, heads, d, device, name):
    """Distance of two tokens, in elements, of rows [tokens, heads, head_dim] whose elements and heads are contiguous."""
    assert x.dim() == 3 and x.shape[1] == heads and x.shape[2] == d, f"{name} is [tokens, {heads}, {d}]"
    assert x.device == device, f"{name} is on another device than the cache"
    assert (x.stride(2) == 1 or d == 1) and (x.stride(1) == d or heads == 1), f"{name}: elements and heads are contiguous"
    return x.stride(0) if x.shape[0] > 1 else heads * d


def _ints(device, **tensors):
    for name, t in tensors.items():
        assert t.dtype == torch.int32 and t.is_contiguous() and t.device == device, \
            f"{name}: contiguous int32 on the cache's device"


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
    block's scale and the token's holds, and where that is the token's the older codes are rounded again.  A sequence
    given more than once in one of the two parts: its last entry counts.  Sequences of length 0, ids outside the table
    and blocks outside the pool are skipped."""
    pool = _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new, model_config,
                 engine_config, infer_state.num_blocks_org, infer_state.kv_cache_new_block_size)
    device = k_cache.device
    heads, d = pool.num_kv_heads, pool.head_dim
    assert k.dtype == v.dtype and k.shape[0] == v.shape[0]
    dtype = _dtype(k)
    ks, vs = _rows(k, heads, d, device, "k"), _rows(v, heads, d, device, "v")
    seq_ids = infer_state.seq_ids
    _ints(device, block_table=block_table, seq_ids=seq_ids)
    n_pre, n_dec = infer_state.num_prefill_seqs, infer_state.num_decoding_seqs
    n_tok = infer_state.num_prefill_tokens if n_pre > 0 else 0
    assert seq_ids.shape[0] >= n_pre + n_dec and k.shape[0] >= n_tok + n_dec
    dev, stream = device_and_stream(k_cache)
    if n_pre > 0:
        starts, lens = infer_state.prefill_seq_start_locs, infer_state.prefill_seq_lens
        _ints(device, prefill_seq_start_locs=starts, prefill_seq_lens=lens)
        assert starts.shape[0] >= n_pre and lens.shape[0] >= n_pre
        check(lib.mkv_store_kv_q8_prefill(
            dev, stream, k.data_ptr(), v.data_ptr(), ks, vs, dtype, n_tok, pool, block_table.data_ptr(),
            block_table.shape[1], block_table.shape[0], seq_ids.data_ptr(), starts.data_ptr(), lens.data_ptr(), n_pre,
            int(infer_state.max_prefill_len), cur_layer), "mkv_store_kv_q8_prefill")
    if n_dec > 0:
        lens = infer_state.decoding_seq_lens
        _ints(device, decoding_seq_lens=lens)
        assert lens.shape[0] >= n_dec
        skip = n_tok * k.element_size()
        check(lib.mkv_store_kv_q8_decode(
            dev, stream, k.data_ptr() + skip * ks, v.data_ptr() + skip * vs, ks, vs, dtype, pool, block_table.data_ptr(),
            block_table.shape[1], block_table.shape[0], seq_ids.data_ptr() + 4 * n_pre, lens.data_ptr(), n_dec,
            cur_layer), "mkv_store_kv_q8_decode")


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
    rows, or a sequence on its way into another pool.  Rows that no range reaches, and rows of tokens whose page is not
    in the table or the pool, are left as they were."""
    pool = _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new, model_config,
                 engine_config, k_cache.shape[0], k_cache_new[0].shape[0] if len(k_cache_new) else 0)
    device = k_cache.device
    heads, d = pool.num_kv_heads, pool.head_dim
    assert k.dtype == v.dtype and k.shape[0] == v.shape[0]
    dtype = _dtype(k)
    ks, vs = _rows(k, heads, d, device, "k"), _rows(v, heads, d, device, "v")
    n = seq_ids.shape[0]
    _ints(device, block_table=block_table, seq_ids=seq_ids, begins=begins, ends=ends, start_locs=start_locs)
    assert begins.shape[0] == n and ends.shape[0] == n and start_locs.shape[0] == n
    dev, stream = device_and_stream(k_cache)
    check(lib.mkv_load_kv_q8(
        dev, stream, k.data_ptr(), v.data_ptr(), ks, vs, dtype, k.shape[0], pool, block_table.data_ptr(),
        block_table.shape[1], block_table.shape[0], seq_ids.data_ptr(), begins.data_ptr(), ends.data_ptr(),
        start_locs.data_ptr(), n, int(max_len), cur_layer), "mkv_load_kv_q8")


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
    sequence's one query token over its ``decoding_seq_lens`` cached tokens, in fp32, rounded once.

    Rows of sequences of length 0 are left as they were.  A page that is not in the table or the pool takes no part
    (and is reported by ``read_attn_error_flags``); a row that is left without any token is NaN.
    ``infer_state.max_decoding_len`` sizes the launch: lengths above it (a captured step whose sequences grew) are
    attended in full."""
    batch = infer_state.num_decoding_seqs
    if batch == 0:
        return
    pool = _pool(k_cache, v_cache, k_scale, v_scale, k_cache_new, v_cache_new, k_scale_new, v_scale_new, model_config,
                 engine_config, infer_state.num_blocks_org, infer_state.kv_cache_new_block_size)
    device = k_cache.device
    hq, hkv, d = model_config.num_q_heads, pool.num_kv_heads, pool.head_dim
    dtype = _dtype(q)
    q_stride = _rows(q, hq, d, device, "q")
    assert q.shape[0] >= batch
    assert o.dtype == q.dtype and o.is_contiguous() and o.device == device and o.numel() >= batch * hq * d
    seq_ids, lens = infer_state.seq_ids, infer_state.decoding_seq_lens
    n_pre = infer_state.num_prefill_seqs
    _ints(device, block_table=block_table, seq_ids=seq_ids, decoding_seq_lens=lens)
    assert seq_ids.shape[0] >= n_pre + batch and lens.shape[0] >= batch
    max_len = getattr(infer_state, "max_decoding_len", None) or engine_config.max_blocks_per_seq * pool.block_size
    dev, stream = device_and_stream(k_cache)
    ws, ws_bytes = workspace_q8(dev, stream, batch, hq, hkv, d)
    check(lib.mkv_paged_attention_q8(
        dev, stream, q.data_ptr(), q_stride, o.data_ptr(), dtype, pool, block_table.data_ptr(), block_table.shape[1],
        block_table.shape[0], seq_ids.data_ptr() + 4 * n_pre, lens.data_ptr(), batch, hq, cur_layer,
        float(infer_state.softmax_scale), int(max_len), ws.data_ptr(), ws_bytes), "mkv_paged_attention_q8")
