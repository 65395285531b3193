"""Argument refusals of the drafted-token step's C entry points: reported on
the host, before any launch (no GPU needed)."""

import ctypes

import pytest

_HOST = (ctypes.c_int64 * 64)()  # only its address is used
BUF = ctypes.c_void_p((ctypes.addressof(_HOST) + 15) & ~15)


def slots_args(**change):
    a = dict(req_to_token=BUF, row_stride=8, rows=2, columns=8, row_ids=BUF, row_ids_is64=1,
             raw_lens=BUF, raw_lens_is64=1, new_lens=BUF, new_lens_is64=1, batch=2, page_size=4,
             ring=BUF, ring_state=BUF, ring_capacity=4, next_positions=None, next_is64=0, parents=None,
             capacity=4, new_offsets=BUF, slots=BUF, positions=BUF, tree_mask=None,
             block_table=None, table_stride=0, table_columns=0, totals=BUF, status=BUF,
             workspace=BUF, commit=1)
    assert set(change) <= set(a)
    return [*{**a, **change}.values(), None]


@pytest.mark.parametrize("change", [
    dict(page_size=0), dict(page_size=2), dict(page_size=12), dict(page_size=256), dict(page_size=-4),
    dict(batch=-1), dict(batch=65536), dict(rows=-1), dict(columns=9), dict(ring_capacity=0),
    dict(capacity=-1), dict(capacity=1 << 31), dict(req_to_token=None), dict(row_ids=None),
    dict(raw_lens=None), dict(new_lens=None), dict(ring=None), dict(ring_state=None),
    dict(slots=None), dict(positions=None), dict(new_offsets=None), dict(totals=None),
    dict(status=None), dict(workspace=None), dict(parents=BUF),
    dict(block_table=BUF, table_stride=3, table_columns=4),
])
def test_map_slots_refuses(change):
    from akv_b200 import _native

    assert _native.lib.akv_map_slots(*slots_args(**change)) == _native.AKV_ERR_INVALID


def test_map_slots_of_no_request_is_ok():
    from akv_b200 import _native

    assert _native.lib.akv_map_slots(*slots_args(batch=0)) == _native.AKV_OK


def rope_args(**change):
    a = dict(q=BUF, q_st=512, q_sh=64, k=BUF, k_st=128, k_sh=64, v=None, v_st=0, v_sh=0, dtype=1,
             tokens=3, hq=8, hkv=2, dim=64, rotary=64, neox=1, wq=None, wk=None, wdtype=1, eps=1e-6,
             positions=BUF, positions_is64=0, table=BUF, table_dtype=2, table_stride=64,
             max_position=10, q_out=BUF, qo_st=512, qo_sh=64, k_out=BUF, ko_st=128, ko_sh=64,
             k_pool=None, kp_ss=0, kp_sh=0, v_pool=None, vp_ss=0, vp_sh=0, num_slots=0, slots=None,
             slots_is64=0, flag=None)
    assert set(change) <= set(a)
    return [*{**a, **change}.values(), None]


ODD = ctypes.c_void_p(BUF.value + 8)  # not on a 16-byte boundary


@pytest.mark.parametrize("change", [
    dict(tokens=-1), dict(hq=0), dict(hkv=0), dict(dim=8), dict(dim=72), dict(dim=528), dict(rotary=0),
    dict(rotary=80), dict(rotary=24), dict(dtype=3), dict(dtype=-1), dict(table_dtype=3),
    dict(wq=BUF, wdtype=0), dict(q=None), dict(k=None), dict(q_out=None), dict(positions=None),
    dict(table=None), dict(max_position=0), dict(k_out=None), dict(v=BUF),
    dict(k_pool=BUF, v=BUF, slots=BUF, num_slots=4), dict(k_pool=BUF, v_pool=BUF, v=BUF, num_slots=4),
    dict(k_pool=BUF, v_pool=BUF, slots=BUF, num_slots=4),
    dict(k_pool=BUF, v_pool=BUF, v=BUF, slots=BUF, num_slots=0), dict(q_st=516), dict(q_sh=60),
    dict(k_sh=66), dict(qo_st=514), dict(ko_sh=65), dict(table_stride=66), dict(q=ODD), dict(k=ODD),
    dict(q_out=ODD), dict(table=ODD),
])
def test_qk_norm_rope_refuses(change):
    from akv_b200 import _native

    assert _native.lib.akv_qk_norm_rope(*rope_args(**change)) == _native.AKV_ERR_INVALID


def test_qk_norm_rope_of_no_token_is_ok():
    from akv_b200 import _native

    assert _native.lib.akv_qk_norm_rope(*rope_args(tokens=0)) == _native.AKV_OK


def test_wrappers_refuse_cpu_tensors():
    import torch

    from akv_b200.context_rope import qk_norm_rope

    x = torch.zeros(2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(x, x, torch.zeros(2, dtype=torch.int32), torch.zeros(4, 64))
