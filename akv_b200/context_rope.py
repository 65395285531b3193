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

_fields, _INT32, _INT64, _CODE = _native.fields, _native.INT32, _native.INT64, _native.FIELD_CODE
_WHAT = ("must be [tokens, heads, head_dim] of the type and device of q, with unit last stride "
         "(k, v and the outputs with its tokens and head_dim)")


def _vector(name, t, n, index):
    """(address, 1 if int64) of a contiguous index vector of at least n entries."""
    ptr, dev, dt, size, step = _fields(1, t)
    if size < n or dev != index or (step != 1 and n > 1) or (dt != _INT32 and dt != _INT64):
        raise ValueError(f"{name} must be a contiguous int32 or int64 vector of an entry for each "
                         "token on the device of q")
    return ptr, 1 if dt == _INT64 else 0


def qk_norm_rope(q, k, positions, cos_sin_cache, *, q_weight=None, k_weight=None, eps=1e-6,
                 rotary_dim=None, is_neox_style=True, q_out=None, k_out=None, v=None, k_pool=None,
                 v_pool=None, slots=None, error_flag=None):
    """Returns ``(q_out, k_out)``.

    ``q`` [tokens, Hq, D], ``k`` (and ``v``) [tokens, Hkv, D]: fp16, bf16 or fp32, the
    last stride 1, the others multiples of 16 bytes (views of a fused
    projection).  D and ``rotary_dim`` (default: the table's width) are
    multiples of 16, D at most 512; dimensions from ``rotary_dim`` on are
    normed and not rotated.  ``positions``: int32 or int64 [>= tokens], as
    ``slots`` below (a ``SlotMap``'s whole vectors fit); ``cos_sin_cache``
    [max_position, rotary_dim] as ``reposition_kv_layers``.

    ``q_weight`` / ``k_weight``: [D], of q's type or both fp32; without one
    that side is rotated and not normed.  Arithmetic is fp32, rounded once.

    With ``k_pool`` / ``v_pool`` [slots, Hkv, D], ``v`` and ``slots`` (int32 or
    int64 [>= tokens]), K and V are stored at the tokens' slots; a token with a
    negative slot is padding and is not stored.  ``k_out`` then is written
    only if given; without pools it is allocated.  ``q_out`` may be ``q`` and
    ``k_out`` ``k``; other overlaps are not supported, and two tokens of one
    call must not have the same slot.

    A slot past the pools, or a position outside the table (rotated as
    position 0), is not stored and sets ``error_flag`` (int32 [1]) if given.
    """
    (q_ptr, index, dt, tokens, hq, d, q0, q1, unit, k_ptr, dev, k_dt, n, hkv, k_dim, k0, k1,
     k_unit) = _fields(3, q, k)
    if index < 0:
        raise ValueError("qk_norm_rope runs on CUDA tensors")
    code = _CODE.get(dt)
    if code is None:
        raise ValueError("qk_norm_rope runs on fp16, bf16 or fp32")
    if unit != 1 or k_unit != 1 or dev != index or k_dt != dt or n != tokens or k_dim != d:
        raise ValueError("q and k " + _WHAT)
    table, dev, table_dt, max_position, width, cache_stride, unit = _fields(2, cos_sin_cache)
    rotary = width if rotary_dim is None else rotary_dim
    cache_code = _CODE.get(table_dt)
    if cache_code is None or rotary != width or unit != 1 or dev != index:
        raise ValueError("cos_sin_cache must be floating point [max_position, rotary_dim] on the "
                         "device of q")
    if d % 16 or d > 512 or rotary % 16 or not 0 < rotary <= d:
        raise ValueError("head_dim and rotary_dim must be multiples of 16, at most 512")
    pos_ptr, pos64 = _vector("positions", positions, tokens, index)
    weight_dt, weights = -1, [0, 0]
    for side, w in enumerate((q_weight, k_weight)):
        if w is None:
            continue
        weights[side], dev, w_dt, n, unit = _fields(1, w)
        if n != d or unit != 1 or dev != index or (w_dt != dt and _CODE.get(w_dt) != _native.AKV_F32):
            raise ValueError("norm weights must be [head_dim] of q's type or fp32")
        if weight_dt not in (-1, w_dt):
            raise ValueError("norm weights must have one type")
        weight_dt = w_dt
    if q_out is None:
        q_out = torch.empty_like(q)
    num_slots = slots_ptr = slots64 = v_ptr = v0 = v1 = 0
    kp_ptr = kp0 = kp1 = vp_ptr = vp0 = vp1 = ko_ptr = ko0 = ko1 = 0
    if k_pool is not None:
        if v is None or v_pool is None or slots is None:
            raise ValueError("a store needs v, k_pool, v_pool and slots")
        (v_ptr, dev, v_dt, n, heads, dim, v0, v1, unit, kp_ptr, kp_dev, kp_dt, k_slots, kp_heads,
         kp_dim, kp0, kp1, kp_unit, vp_ptr, vp_dev, vp_dt, v_slots, vp_heads, vp_dim, vp0, vp1,
         vp_unit) = _fields(3, v, k_pool, v_pool)
        if n != tokens or heads != hkv or dim != d or unit != 1 or dev != index or v_dt != dt:
            raise ValueError("v " + _WHAT)
        if kp_heads != hkv or vp_heads != hkv or kp_dim != d or vp_dim != d or kp_unit != 1 or \
                vp_unit != 1 or kp_dev != index or vp_dev != index or kp_dt != dt or vp_dt != dt:
            raise ValueError("KV pools must be [slots, num_kv_heads, head_dim] of the type and "
                             "device of q, with unit last stride")
        num_slots = k_slots if k_slots < v_slots else v_slots
        slots_ptr, slots64 = _vector("slots", slots, tokens, index)
    elif v is not None or v_pool is not None or slots is not None:
        raise ValueError("a store needs v, k_pool, v_pool and slots")
    elif k_out is None:
        k_out = torch.empty_like(k)
    qo_ptr, dev, out_dt, n, heads, dim, qo0, qo1, unit = _fields(3, q_out)
    if n != tokens or heads != hq or dim != d or unit != 1 or dev != index or out_dt != dt:
        raise ValueError("q_out " + _WHAT)
    if k_out is not None:
        ko_ptr, dev, out_dt, n, heads, dim, ko0, ko1, unit = _fields(3, k_out)
        if n != tokens or heads != hkv or dim != d or unit != 1 or dev != index or out_dt != dt:
            raise ValueError("k_out " + _WHAT)
    flag = 0
    if error_flag is not None:
        if error_flag.get_device() != index or error_flag.dtype != torch.int32:
            raise ValueError("error_flag must be an int32 tensor on the device of q")
        flag = error_flag.data_ptr()
    if tokens == 0:
        return q_out, k_out
    status = _native.launch(index, _native.lib.akv_qk_norm_rope, _native.QK_NORM_ROPE.pack(
        q_ptr, q0, q1, k_ptr, k0, k1, v_ptr, v0, v1, code, tokens, hq, hkv, d, rotary,
        1 if is_neox_style else 0, weights[0], weights[1], _CODE.get(weight_dt, code), eps, pos_ptr,
        pos64, table, cache_code, cache_stride, max_position, qo_ptr, qo0, qo1, ko_ptr, ko0, ko1,
        kp_ptr, kp0, kp1, vp_ptr, vp0, vp1, num_slots, slots_ptr, slots64, flag))
    _native.check(status, "qk_norm_rope")
    return q_out, k_out
