"""Rotary embedding by position, without tables: both pair layouts, part of the head, frequencies scaled for long
contexts.

``rotary_embedding_inplace`` (worker/kernels/rotary_emb.py:43-58) takes gathered fp16 cos/sin rows, rotates whole heads
in the half layout and knows linear scaling only (worker/model.py:229-241).  Here the kernel forms the angles itself, in
64 bits, from the tokens' positions and one frequency for each pair.
"""
from __future__ import annotations

import ctypes as C
import math

import torch

from ..._lib import check, lib
from ._common import raw_stream, require_cuda

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}       # mkv_dtype


def rotary_inv_freq(model_config, device="cuda"):
    """``(inv_freq, attention_scale)`` of a model: radians a position for each pair (float64 on ``device``) and the
    factor on sines and cosines.

    Read from ``model_config``: ``head_dim``, ``rope_theta`` (default 10000), ``partial_rotary_factor`` (default 1: the
    part of the head that is rotated), ``max_position_embeddings`` and ``rope_scaling``: nothing, a number (linear, as in
    worker/model.py:232-238), or a mapping with ``rope_type`` (or ``type``) and ``factor``:

      default          no scaling
      linear           positions divided by ``factor``
      ntk              base * factor^(d / (d - 2))
      llama3           by bands of turns over ``original_max_position_embeddings``: above ``high_freq_factor`` kept, below
                       ``low_freq_factor`` divided by ``factor``, blended between
      yarn             by pair index: kept above ``beta_fast`` (32) turns, divided below ``beta_slow`` (1), a ramp between;
                       attention_scale = ``attention_factor``, else 0.1 ln(factor) + 1; its further variants (``mscale``,
                       ``mscale_all_dim``, ``truncate`` switched off) are refused
    """
    dim = int(model_config.head_dim * (getattr(model_config, "partial_rotary_factor", 1.0) or 1.0))
    dim -= dim % 2
    if dim < 2:
        raise ValueError("the rotated part of a head has at least two elements")
    base = float(getattr(model_config, "rope_theta", 10000.0) or 10000.0)
    scaling = getattr(model_config, "rope_scaling", None)
    if scaling is None:
        scaling = {}
    elif isinstance(scaling, (int, float)):
        scaling = {"rope_type": "linear", "factor": float(scaling)}
    kind = scaling.get("rope_type", scaling.get("type", "default"))
    factor = float(scaling.get("factor", 1.0))
    if kind not in ("default", "linear", "ntk", "llama3", "yarn"):
        raise ValueError(f"unknown rope_type {kind!r}")
    if kind != "default" and not factor > 0:
        raise ValueError("the scaling factor is positive")
    if kind == "ntk" and dim > 2:
        base *= factor ** (dim / (dim - 2))
    inv = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    attention_scale = 1.0
    if kind == "linear":
        inv = inv / factor
    elif kind in ("llama3", "yarn"):
        original = scaling.get("original_max_position_embeddings") or getattr(model_config, "max_position_embeddings", None)
        if not original:
            raise ValueError(f"{kind} scaling needs original_max_position_embeddings")
        if kind == "llama3":
            low, high = float(scaling.get("low_freq_factor", 1.0)), float(scaling.get("high_freq_factor", 4.0))
            if not high > low:
                raise ValueError("high_freq_factor is above low_freq_factor")
            keep = ((original * inv / (2 * math.pi) - low) / (high - low)).clamp(0, 1)
            inv = inv * keep + inv / factor * (1 - keep)
        else:
            if scaling.get("mscale") or scaling.get("mscale_all_dim") or scaling.get("truncate", True) is False:
                raise ValueError("yarn scaling with mscale, mscale_all_dim or truncate=False")
            at = [dim * math.log(original / (float(scaling.get(name, turns)) * 2 * math.pi)) / (2 * math.log(base))
                  for name, turns in (("beta_fast", 32.0), ("beta_slow", 1.0))]
            low, high = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
            ramp = ((torch.arange(dim // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
            inv = inv / factor * ramp + inv * (1 - ramp)
            attention_scale = scaling.get("attention_factor")
            if attention_scale is None:
                attention_scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    return inv.to(device), float(attention_scale)


_INTS = {torch.int32: 4, torch.int64: 8}
_Strides = C.c_int64 * 8


def _strides(x, n, heads, d):
    """Distances of two tokens and of two heads; elements are contiguous, nothing overlaps."""
    s = x.stride()
    assert s[2] == 1, "elements are contiguous"
    if n > 1 and heads > 1:     # the heads of a token lie in front of the next token, or the other way round
        near, far, inner = (s[1], s[0], heads) if s[0] >= s[1] else (s[0], s[1], n)
        assert near >= d and far >= (inner - 1) * near + d, "tokens and heads do not overlap"
    else:
        assert (n <= 1 or s[0] >= d) and (heads <= 1 or s[1] >= d), "tokens and heads do not overlap"
    return s


def rotary_embedding_positions(
    q: torch.Tensor,                # [num_tokens, num_q_heads, head_dim]
    k: torch.Tensor,                # [num_tokens, num_kv_heads, head_dim]
    positions: torch.Tensor,        # [num_tokens] int32 or int64
    inv_freq: torch.Tensor,         # [rotary_dim / 2] float64, radians a position (see rotary_inv_freq)
    *,
    interleaved: bool = False,      # pairs are neighbours (2j, 2j + 1) instead of (j, j + rotary_dim / 2)
    attention_scale: float = 1.0,
    q_out: torch.Tensor = None,     # where the result goes; default: in place
    k_out: torch.Tensor = None,
):
    """Rotate pair j of every head of token t by ``positions[t] * inv_freq[j]`` and scale it by ``attention_scale``;
    elements behind the rotated part pass through unchanged.  In place, or into ``q_out`` / ``k_out`` (memory that does
    not overlap q and k).  fp16, bf16 or fp32, computed in fp32 and rounded once.  Elements are contiguous; tokens and
    heads may lie any distance apart, so q and k may be views of one fused projection.  Positions of up
    to 2^53 (what a 64-bit float counts) and frequencies of up to 1 give the angle to about 2^-24 of half a turn."""
    dev = q.get_device()
    if dev < 0:
        require_cuda(q, "q")
    shape, k_shape, dtype = q.shape, k.shape, q.dtype
    code = _DTYPES.get(dtype)
    if code is None:
        raise RuntimeError(f"unsupported dtype {dtype}")
    n, hq, d = shape
    hkv = k_shape[1]
    assert len(k_shape) == 3 and k_shape[0] == n and k_shape[2] == d and k.dtype is dtype and k.get_device() == dev
    qs, ks = _strides(q, n, hq, d), _strides(k, n, hkv, d)
    qos, kos = qs, ks
    if q_out is None:
        q_out = q
    else:
        assert q_out.shape == shape and q_out.dtype is dtype and q_out.get_device() == dev
        qos = _strides(q_out, n, hq, d)
    if k_out is None:
        k_out = k
    else:
        assert k_out.shape == k_shape and k_out.dtype is dtype and k_out.get_device() == dev
        kos = _strides(k_out, n, hkv, d)
    assert positions.dtype in _INTS and positions.is_contiguous() and positions.shape == shape[:1]
    assert inv_freq.dtype is torch.float64 and inv_freq.is_contiguous() and inv_freq.dim() == 1
    assert positions.get_device() == dev and inv_freq.get_device() == dev
    pairs = inv_freq.shape[0]
    assert 2 * pairs <= d, "inv_freq has at most head_dim / 2 entries"
    check(lib.mkv_rotary_positions(
        dev, raw_stream(dev), q.data_ptr(), k.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
        _Strides(qs[0], qs[1], ks[0], ks[1], qos[0], qos[1], kos[0], kos[1]), positions.data_ptr(), _INTS[positions.dtype],
        inv_freq.data_ptr(), pairs, bool(interleaved), attention_scale, n, hq, hkv, d, code), "mkv_rotary_positions")
