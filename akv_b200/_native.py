"""ctypes binding of ``libakv_b200.so`` (declared in include/akv_b200.h).

The library is built in-tree by ``python -m akv_b200.build``.  There is no
fallback: importing the ops without the built library raises ImportError,
and a failed launch raises RuntimeError.
"""

from __future__ import annotations

import ctypes
import os
import struct

import torch

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libakv_b200.so")

AKV_OK, AKV_ERR_INVALID, AKV_ERR_CUDA, AKV_ERR_UNSUPPORTED = 0, 1, 2, 3
AKV_ERR_OCC_MISSING_SOURCE, AKV_ERR_OCC_MISSING_COPY_SOURCE = 4, 5
AKV_F16, AKV_BF16, AKV_F32 = 0, 1, 2
GATHER_OUT64, GATHER_LITERAL, GATHER_SEG64 = 1, 2, 4
DROP_RING_UNDERFLOW, DROP_RING_OVERFLOW, DROP_BAD_RANGE, DROP_NO_ACTIVE = 1, 2, 4, 8
DROP_BAD_PAGE = 16
REPOSITION_BULK_V = 1
SLOTS_RING_UNDERFLOW, SLOTS_CAPACITY, SLOTS_BAD_REQUEST = 1, 2, 4
SLOTS_BAD_PAGE, SLOTS_BAD_PARENT = 8, 16
SLOTS_KEEP_OFFSETS = 1 << 32

DTYPE_CODE = {torch.float16: AKV_F16, torch.bfloat16: AKV_BF16, torch.float32: AKV_F32}

_P = ctypes.c_void_p
_I32 = ctypes.c_int32
_I64 = ctypes.c_int64

LAYOUT_CAPACITY, LAYOUT_ERROR, LAYOUT_TOO_MANY = 1, 2, 4


class LayoutBatch(ctypes.Structure):
    """struct akv_layout_batch of include/akv_b200.h, field for field."""

    _fields_ = [
        ("n_requests", _I32), ("n_tiles", _I32), ("n_tokens", _I64), ("n_repositions", _I64),
        ("n_count_cells", _I64), ("token_offsets", _P), ("token_ids", _P),
        ("token_ids_is64", _I32), ("tile_offsets", _P), ("count_offsets", _P),
        ("drop_event_offsets", _P), ("drop_insert_offsets", _P), ("drop_range_offsets", _P),
        ("drop_ranges", _P), ("reposition_offsets", _P), ("reposition_raw_boundaries", _P),
        ("positions", _P), ("keep_mask", _P), ("materialized_stage", _P),
        ("birth_positions", _P), ("birth_stages", _P), ("token_to_key", _P), ("records", _P),
        ("virtual_mask", _P), ("key_to_token", _P), ("transition_offsets", _P),
        ("transition_request_offsets", _P), ("transition_raw_tokens", _P),
        ("transition_old_positions", _P), ("transition_new_positions", _P),
        ("transition_capacity", _I64), ("effective_reposition_stages", _P),
        ("effective_repositions", _P), ("ignored_repositions", _P), ("drop_event_to_key", _P),
        ("status", _P), ("active_offsets", _P), ("raw_indices", _P), ("active_positions", _P),
        ("totals", _P), ("workspace", _P),
    ]


class PackedArgs:
    """An argument struct of 8-byte members (``/d``: a double), in the header's
    order.  Packing one and passing its address costs a tenth of a ctypes
    call with as many arguments (13 us for 42)."""

    def __init__(self, members):
        members = members.split()
        self.names = [m.split("/")[0] for m in members]
        self.struct = struct.Struct("".join("d" if m.endswith("/d") else "q" for m in members))
        self.pack = self.struct.pack


MAP_SLOTS = PackedArgs(
    "req_to_token row_stride rows columns row_ids row_ids_is64 raw_lens raw_lens_is64 new_lens "
    "new_lens_is64 batch page_size ring ring_state ring_capacity next_positions next_is64 parents "
    "capacity new_offsets slots positions tree_mask block_table table_stride table_columns totals "
    "status workspace commit")
QK_NORM_ROPE = PackedArgs(
    "q q_stride_token q_stride_head k k_stride_token k_stride_head v v_stride_token v_stride_head "
    "dtype tokens num_q_heads num_kv_heads head_dim rotary_dim is_neox_style q_weight k_weight "
    "weight_dtype eps/d positions positions_is64 cos_sin_cache cache_dtype cache_stride "
    "max_position q_out q_out_stride_token q_out_stride_head k_out k_out_stride_token "
    "k_out_stride_head k_pool k_pool_stride_slot k_pool_stride_head v_pool v_pool_stride_slot "
    "v_pool_stride_head num_slots slots slots_is64 error_flag")
TREE_ATTENTION = PackedArgs(
    "q q_stride_token q_stride_head k_pool v_pool k_stride_slot k_stride_head v_stride_slot "
    "v_stride_head num_slots dtype tokens keys kv_indices draft_slots tree_mask q_positions "
    "kv_positions window sinks sm_scale/d num_q_heads num_kv_heads head_dim items cta_items "
    "n_ctas merges n_merges partial_acc partial_ml out out_stride_token out_stride_head lse "
    "error_flag")

# name -> argument types, in the order of include/akv_b200.h
SIGNATURES = {
    "akv_version": [],
    "akv_reposition_kv_layers": [
        _P, _P, _I32, _I32, _I32, _I32, _I32, _I64, _I64, _I64, _I64, _P, _P, _P, _I64, _I64,
        _P, _P, _I32, _I64, _I32, _I32, _I64, _I64, _P, _P,
    ],
    "akv_reposition_kv_layers_ex": [
        _P, _P, _I32, _I32, _I32, _I32, _I32, _I64, _I64, _I64, _I64, _P, _P, _P, _I64, _I64,
        _P, _P, _I32, _I64, _I32, _I32, _I64, _I64, _P, _I32, _P,
    ],
    "akv_reposition_divide": [_P, _P, _P, _I64, _I32, _P],
    "akv_drop_compact_tile_tokens": [],
    "akv_drop_compact_workspace_bytes": [_I32, _I32],
    "akv_drop_compact": [
        _I32, _P, _P, _I32, _P, _P, _P, _P, _P, _I64, _I32, _P, _I64, _P, _P, _P, _P, _P, _P,
        _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P,
    ],
    "akv_drop_compact_paged": [
        _I32, _P, _P, _I32, _P, _P, _P, _P, _P, _I64, _I32, _I32, _P, _I64, _P, _P, _P, _P, _P,
        _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P,
    ],
    "akv_occurrence_advance_indices": [_P, _P],
    "akv_drop_read_view": [_P, _P, _P, _I64, _P, _P, _I32, _P, _P],
    "akv_drop_compact_static_max_requests": [],
    "akv_drop_compact_static_max_tiles": [],
    "akv_drop_compact_static": [
        _I32, _P, _P, _I32, _P, _P, _P, _P, _P, _I64, _I32, _P, _I64, _P, _P, _P, _P, _P, _P,
        _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P,
    ],
    "akv_context_decode_indices": [
        _P, _P, _I64, _P, _I32, _P, _I32, _P, _I32, _P, _I32, _P, _I32, _P, _I32, _I64, _I32,
        _P,
    ],
    "akv_context_window_lengths": [_P, _P, _I32, _P, _I32, _P, _I32, _I64, _I32, _P],
    "akv_build_decode_metadata": [
        _P, _P, _I64, _P, _P, _I64, _P, _I64, _I32, _P, _P, _P, _P, _P,
    ],
    "akv_write_row_slots": [_P, _P, _I32, _P, _I32, _P, _I32, _I64, _P],
    "akv_active_slots": [_P, _I64, _P, _I64, _I64, _I64, _I64, _P, _P, _P],
    "akv_active_slots_batch": [_P, _P, _P, _I32, _P, _P, _P],
    "akv_active_slots_chunk": [],
    "akv_gather_slots_chunk": [],
    "akv_gather_slots": [_P, _P, _I32, _P, _P, _P],
    "akv_compile_layouts_max_repositions": [],
    "akv_compile_layouts_workspace_bytes": [_I32, _I64, _I64, _I64],
    "akv_compile_layouts_batch_bytes": [],
    "akv_compile_layouts": [ctypes.POINTER(LayoutBatch), _P],
    "akv_decode_attention": [
        _P, _I64, _I64, _P, _P, _I64, _I64, _I64, _I64, _I64, _P, _P, ctypes.c_float, _I32,
        _I32, _I32, _I32, _P, _I32, _P, _I32, _P, _P, _P, _P, _I64, _I64, _P, _P, _P,
    ],
    "akv_decode_attention_ctas_per_sm": [_I32, _I32],
    "akv_map_slots": [ctypes.c_char_p, _P],
    "akv_map_slots_args_bytes": [],
    "akv_qk_norm_rope": [ctypes.c_char_p, _P],
    "akv_qk_norm_rope_args_bytes": [],
    "akv_tree_attention_units": [],
    "akv_tree_attention": [ctypes.c_char_p, _P],
    "akv_tree_attention_args_bytes": [],
    "akv_context_attention_query_block": [],
    "akv_context_attention": [
        _P, _I64, _I64, _P, _P, _I64, _I64, _I64, _I64, _I64, _P, _P, _P, _P, _P, _P, _P,
        ctypes.c_float, _I64, _I32, _I32, _I32, _P, _I32, _P, _I64, _I64, _P, _P, _I32, _P,
    ],
}
RESTYPES = {
    "akv_tree_attention_args_bytes": _I64,
    "akv_qk_norm_rope_args_bytes": _I64,
    "akv_map_slots_args_bytes": _I64,
    "akv_version": ctypes.c_char_p,
    "akv_drop_compact_tile_tokens": _I64,
    "akv_drop_compact_workspace_bytes": _I64,
    "akv_drop_compact_static_max_requests": _I64,
    "akv_drop_compact_static_max_tiles": _I64,
    "akv_compile_layouts_max_repositions": _I64,
    "akv_compile_layouts_workspace_bytes": _I64,
    "akv_compile_layouts_batch_bytes": _I64,
    "akv_decode_attention_ctas_per_sm": _I32,
    "akv_tree_attention_units": _I32,
    "akv_context_attention_query_block": _I64,
    "akv_active_slots_chunk": _I64,
    "akv_gather_slots_chunk": _I64,
}


def _load():
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is not built; run `python -m akv_b200.build` (nvcc, sm_100a). "
            "akv_b200 has no CPU or Triton fallback."
        )
    lib = ctypes.CDLL(LIB_PATH)
    for name, args in SIGNATURES.items():
        fn = getattr(lib, name)
        fn.argtypes = args
        fn.restype = RESTYPES.get(name, ctypes.c_int)
    return lib


lib = _load()
# fields(ndim, tensor, ...) -> address, device, type code, sizes and strides of each, and the
# type codes.  The drafted-token step alone uses it; without it the rest works.
INT32 = INT64 = None
FIELD_CODE = {}  # type code -> AKV_* element type
try:
    from . import _tensor_fields

    if getattr(_tensor_fields, "BUILT_FOR", None) != torch.__version__:
        raise ImportError("it was built for another torch")
    fields = _tensor_fields.fields
    INT32, INT64 = _tensor_fields.INT32, _tensor_fields.INT64
    FIELD_CODE = {_tensor_fields.F16: AKV_F16, _tensor_fields.BF16: AKV_BF16,
                  _tensor_fields.F32: AKV_F32}
except ImportError as e:
    _no_fields = f"akv_b200._tensor_fields cannot be used ({e}); run `python -m akv_b200.build`"

    def fields(*args):
        raise ImportError(_no_fields)


def ptr(t):
    """Device address of a tensor (None -> NULL)."""
    return None if t is None else ctypes.c_void_p(t.data_ptr())


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)


def stream_of(device) -> ctypes.c_void_p:
    """The current torch stream of ``device`` as a cudaStream_t."""
    if _raw_stream is not None:
        if isinstance(device, int):
            return ctypes.c_void_p(_raw_stream(device))
        d = device if isinstance(device, torch.device) else torch.device(device)
        if d.type == "cuda":
            index = d.index if d.index is not None else torch.cuda.current_device()
            return ctypes.c_void_p(_raw_stream(index))
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def capturing(index: int) -> bool:
    """Whether the current torch stream of CUDA device ``index`` is being captured."""
    if torch._C._cuda_getDevice() == index:
        return torch._C._cuda_isCurrentStreamCapturing()
    with torch.cuda.device(index):
        return torch.cuda.is_current_stream_capturing()


def launch(index: int, fn, args) -> int:
    """``fn(args, stream)`` on the current torch stream of CUDA device
    ``index``, which is made the current device for the call if it is not
    (a kernel must be launched from its stream's device)."""
    if torch.cuda.current_device() == index:
        return fn(args, _raw_stream(index) if _raw_stream is not None
                  else torch.cuda.current_stream(index).cuda_stream)
    with torch.cuda.device(index):
        return fn(args, torch.cuda.current_stream(index).cuda_stream)


def check(status: int, what: str) -> None:
    if status == AKV_OK:
        return
    if status == AKV_ERR_INVALID:
        raise ValueError(f"{what}: invalid arguments")
    if status == AKV_ERR_UNSUPPORTED:
        raise ValueError(f"{what}: unsupported configuration")
    raise RuntimeError(f"{what}: CUDA launch failed (status {status})")


def is64(t) -> int:
    if t.dtype == torch.int64:
        return 1
    if t.dtype == torch.int32:
        return 0
    raise ValueError(f"index tensors must be int32 or int64, got {t.dtype}")
