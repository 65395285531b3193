"""Per-head norms of Q and K, the position rotation and the cache store in
one pass (C ABI ``akv_qk_norm_rope``).

A layer of a model with normalised queries and keys runs, per token and head,
an RMS norm over the head, the rotation at the token's position, and the
store of K and V at the token's slot: four native modules around
akv/system/sglang.patch:2437-2445 in the reference's runtime.
``qk_norm_rope`` reads each projected element once and writes each result
once.  Positions and slots are those of ``context_slots.SlotMapper``; the
cos / sin table is the one ``reposition_kv_layers`` reads
(``akv_b200.rope``), so a key stored here is the key a later Reposition
re-rotates.
"""

from __future__ import annotations

import torch

from . import _native

_NONE = (0, 0, 0)


def _heads(name, t, dtype, index, shape):
    """(address, stride of the first dimension, of the second)."""
    s = t.stride()
    if t.dtype != dtype or t.get_device() != index or len(s) != 3 or s[2] != 1 or \
            (shape is not None and t.shape != shape):
        raise ValueError(f"{name} must be [tokens, heads, head_dim] of the type and device of q, "
                         "with unit last stride")
    return t.data_ptr(), s[0], s[1]


def qk_norm_rope(q, k, positions, cos_sin_cache, *, q_weight=None, k_weight=None, eps=1e-6,
                 rotary_dim=None, is_neox_style=True, q_out=None, k_out=None, v=None, k_pool=None,
                 v_pool=None, slots=None, error_flag=None):
    """Returns ``(q_out, k_out)``.

    ``q`` [tokens, Hq, D], ``k`` (and ``v``) [tokens, Hkv, D]: fp16, bf16 or fp32, the
    last stride 1, the others multiples of 16 bytes (views of a fused
    projection).  D and ``rotary_dim`` (default: the table's width) are
    multiples of 16, D at most 512; dimensions from ``rotary_dim`` on are
    normed and not rotated.  ``positions``: int32 or int64 [tokens];
    ``cos_sin_cache`` [max_position, rotary_dim] as ``reposition_kv_layers``.

    ``q_weight`` / ``k_weight``: [D], of q's type or both fp32; without one
    that side is rotated and not normed.  Arithmetic is fp32, rounded once.

    With ``k_pool`` / ``v_pool`` [slots, Hkv, D], ``v`` and ``slots`` (int32 or
    int64 [tokens]), K and V are stored at the tokens' slots; a token with a
    negative slot is padding and is not stored.  ``k_out`` then is written
    only if given; without pools it is allocated.  ``q_out`` may be ``q`` and
    ``k_out`` ``k``; other overlaps are not supported, and two tokens of one
    call must not have the same slot.

    A slot past the pools, or a position outside the table (rotated as
    position 0), is not stored and sets ``error_flag`` (int32 [1]) if given.
    """
    index = q.get_device()
    if index < 0:
        raise ValueError("qk_norm_rope runs on CUDA tensors")
    dtype = q.dtype
    code = _native.DTYPE_CODE.get(dtype)
    if code is None:
        raise ValueError("qk_norm_rope runs on fp16, bf16 or fp32")
    qa = _heads("q", q, dtype, index, None)
    tokens, hq, d = q.shape
    ka = _heads("k", k, dtype, index, None)
    k_tokens, hkv, k_dim = k.shape
    if k_tokens != tokens or k_dim != d:
        raise ValueError("k must have q's tokens and head_dim")
    if cos_sin_cache.ndim != 2 or cos_sin_cache.get_device() != index:
        raise ValueError("cos_sin_cache must be [max_position, rotary_dim] on the device of q")
    max_position, width = cos_sin_cache.shape
    cache_stride, unit = cos_sin_cache.stride()
    rotary = width if rotary_dim is None else rotary_dim
    cache_code = _native.DTYPE_CODE.get(cos_sin_cache.dtype)
    if cache_code is None or rotary != width or unit != 1:
        raise ValueError("cos_sin_cache must be floating point and rotary_dim wide")
    if d % 16 or d > 512 or rotary % 16 or not 0 < rotary <= d:
        raise ValueError("head_dim and rotary_dim must be multiples of 16, at most 512")
    if positions.shape != (tokens,) or positions.get_device() != index or \
            not positions.is_contiguous():
        raise ValueError("positions must be a contiguous vector of one entry per token")
    weight_code = code
    for w in (q_weight, k_weight):
        if w is None:
            continue
        if w.shape != (d,) or w.stride(0) != 1 or w.get_device() != index or \
                w.dtype not in (dtype, torch.float32):
            raise ValueError("norm weights must be [head_dim] of q's type or fp32")
        weight_code = _native.DTYPE_CODE[w.dtype]
    if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
        raise ValueError("norm weights must have one type")
    if q_out is None:
        q_out = torch.empty_like(q)
    qo = _heads("q_out", q_out, dtype, index, q.shape)
    va = kp = vp = _NONE
    num_slots = slots_ptr = slots64 = 0
    if k_pool is not None:
        if v is None or v_pool is None or slots is None:
            raise ValueError("a store needs v, k_pool, v_pool and slots")
        va = _heads("v", v, dtype, index, k.shape)
        kp = _heads("k_pool", k_pool, dtype, index, None)
        vp = _heads("v_pool", v_pool, dtype, index, None)
        k_shape, v_shape = k_pool.shape, v_pool.shape
        if k_shape[1:] != (hkv, d) or v_shape[1:] != (hkv, d):
            raise ValueError("KV pools must be [slots, num_kv_heads, head_dim]")
        num_slots = min(k_shape[0], v_shape[0])
        if slots.shape != (tokens,) or slots.get_device() != index or not slots.is_contiguous():
            raise ValueError("slots must be a contiguous vector of one entry per token")
        slots_ptr, slots64 = slots.data_ptr(), _native.is64(slots)
    elif v is not None or v_pool is not None or slots is not None:
        raise ValueError("a store needs v, k_pool, v_pool and slots")
    elif k_out is None:
        k_out = torch.empty_like(k)
    ko = _NONE if k_out is None else _heads("k_out", k_out, dtype, index, k.shape)
    flag = 0
    if error_flag is not None:
        if error_flag.get_device() != index or error_flag.dtype != torch.int32:
            raise ValueError("error_flag must be an int32 tensor on the device of q")
        flag = error_flag.data_ptr()
    positions64 = _native.is64(positions)
    if tokens == 0:
        return q_out, k_out
    status = _native.launch(index, _native.lib.akv_qk_norm_rope, _native.QK_NORM_ROPE.pack(
        *qa, *ka, *va, code, tokens, hq, hkv, d, rotary, 1 if is_neox_style else 0,
        0 if q_weight is None else q_weight.data_ptr(),
        0 if k_weight is None else k_weight.data_ptr(), weight_code, eps, positions.data_ptr(),
        positions64, cos_sin_cache.data_ptr(), cache_code, cache_stride, max_position, *qo, *ko,
        *kp, *vp, num_slots, slots_ptr, slots64, flag))
    _native.check(status, "qk_norm_rope")
    return q_out, k_out
