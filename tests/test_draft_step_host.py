"""Argument refusals of the drafted-token step's C entry points: reported on
the host, before any launch (no GPU needed)."""

import ctypes

import pytest

_HOST = (ctypes.c_int64 * 64)()  # only its address is used
BUF = ctypes.c_void_p((ctypes.addressof(_HOST) + 15) & ~15)


def packed(struct, args, change):
    """The argument struct of ``args``, given in its members' order."""
    from akv_b200 import _native

    values = [getattr(v, "value", v) or 0 for v in {**args, **change}.values()]
    return getattr(_native, struct).pack(*values), None


def slots_args(**change):
    a = dict(req_to_token=BUF, row_stride=8, rows=2, columns=8, row_ids=BUF, row_ids_is64=1,
             raw_lens=BUF, raw_lens_is64=1, new_lens=BUF, new_lens_is64=1, batch=2, page_size=4,
             ring=BUF, ring_state=BUF, ring_capacity=4, next_positions=None, next_is64=0, parents=None,
             capacity=4, new_offsets=BUF, slots=BUF, positions=BUF, tree_mask=None,
             block_table=None, table_stride=0, table_columns=0, totals=BUF, status=BUF,
             workspace=BUF, commit=1)
    assert set(change) <= set(a)
    return packed("MAP_SLOTS", a, change)


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
    return packed("QK_NORM_ROPE", a, change)


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


def test_argument_structs_match_the_header():
    """Members in the header's order, doubles where it has doubles, its size;
    no struct is refused."""
    import os
    import re

    from akv_b200 import _native
    from conftest import ROOT

    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(ROOT, "include", "akv_b200.h")).read(),
                  flags=re.S)
    for name, mirror in (("akv_map_slots", _native.MAP_SLOTS),
                         ("akv_qk_norm_rope", _native.QK_NORM_ROPE),
                         ("akv_tree_attention", _native.TREE_ATTENTION)):
        end = text.index("} %s_args;" % name)
        members = text[text.rindex("{", 0, end) + 1: end].split(";")[:-1]
        assert [re.sub(r".*[ *]", "", m.strip()) for m in members] == mirror.names
        assert "".join("d" if m.split()[0] == "double" else "q" for m in members) == \
            mirror.struct.format
        assert getattr(_native.lib, name + "_args_bytes")() == mirror.struct.size
        assert getattr(_native.lib, name)(None, None) == _native.AKV_ERR_INVALID


def test_wrappers_refuse_cpu_tensors():
    import torch

    from akv_b200.context_rope import qk_norm_rope

    x = torch.zeros(2, 8, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(x, x, torch.zeros(2, dtype=torch.int32), torch.zeros(4, 64))


def test_fields_of_tensors_and_what_they_refuse():
    import torch

    from akv_b200 import _native

    a = torch.zeros(5, 6, dtype=torch.int32)
    b = torch.zeros(7, 8, dtype=torch.bfloat16)[::2, 1:]
    got = _native.fields(2, a, b)
    assert got == (a.data_ptr(), -1, _native.INT32, 5, 6, 6, 1,
                   b.data_ptr(), -1, got[9], 4, 7, 16, 1)
    assert _native.FIELD_CODE[got[9]] == _native.AKV_BF16 and _native.fields(2) == ()
    codes = [_native.fields(1, torch.zeros(1, dtype=t))[2]
             for t in (torch.int64, torch.float16, torch.float32)]
    assert codes[0] == _native.INT64
    assert [_native.FIELD_CODE[c] for c in codes[1:]] == [_native.AKV_F16, _native.AKV_F32]
    sparse = torch.zeros(2, 2).to_sparse()
    for bad in ((), (-1,), (9,), (2, [1]), (2, None), (1, a), (3, a), (2, a, 5), (2, sparse)):
        with pytest.raises(ValueError):
            _native.fields(*bad)
    with pytest.raises(TypeError):
        _native.fields("2", a)


def tree_args(**change):
    a = dict(q=BUF, q_st=512, q_sh=64, k=BUF, v=BUF, k_ss=128, k_sh=64, v_ss=128, v_sh=64, slots=8,
             dtype=1, tokens=8, keys=8, indices=BUF, draft=BUF, mask=BUF, qpos=None, kpos=None, window=-1, sinks=None,
             scale=1.0, hq=8, hkv=2, dim=64, items=BUF, cta_items=BUF, n_ctas=1, merges=None, n_merges=0,
             acc=None, ml=None, out=BUF, o_st=512, o_sh=64, lse=None, flag=None)
    assert set(change) <= set(a)
    return packed("TREE_ATTENTION", a, change)


@pytest.mark.parametrize("change", [
    dict(hkv=0), dict(hq=0), dict(hq=9), dict(n_ctas=-1), dict(tokens=-1), dict(keys=-1),
    dict(scale=0.0), dict(scale=float("nan")), dict(k_ss=-8), dict(v_ss=1 << 31), dict(slots=1 << 31), dict(n_merges=-1), dict(slots=0), dict(dtype=2),
    dict(q=None), dict(k=None), dict(v=None), dict(indices=None), dict(draft=None), dict(mask=None),
    dict(items=None), dict(cta_items=None), dict(out=None), dict(n_merges=1), dict(window=3),
    dict(window=3, qpos=BUF), dict(q=ODD), dict(k=ODD), dict(v=ODD), dict(out=ODD), dict(q_st=516),
    dict(k_ss=130), dict(v_sh=60), dict(o_sh=63),
])
def test_tree_attention_refuses(change):
    from akv_b200 import _native

    assert _native.lib.akv_tree_attention(*tree_args(**change)) == _native.AKV_ERR_INVALID


@pytest.mark.parametrize("scale", [1e-50, 1e39, float("inf"), float("nan")])
def test_tree_attention_refuses_scales_that_fp32_does_not_hold(scale):
    from akv_b200 import _native

    assert _native.lib.akv_tree_attention(*tree_args(scale=scale)) == _native.AKV_ERR_INVALID


def test_tree_attention_of_nothing_is_ok_and_other_head_dims_are_unsupported():
    from akv_b200 import _native

    assert _native.lib.akv_tree_attention(*tree_args(n_ctas=0)) == _native.AKV_OK
    assert _native.lib.akv_tree_attention(*tree_args(dim=96)) == _native.AKV_ERR_UNSUPPORTED
    assert _native.lib.akv_tree_attention_units() == 2


@pytest.mark.parametrize("pair_heads", [False, True])
@pytest.mark.parametrize("hkv,group", [(8, 8), (1, 8), (3, 5), (2, 40)])
@pytest.mark.parametrize("ctas", [1, 7, 296])
def test_tree_work_list_covers_every_key_of_every_row_once(pair_heads, hkv, group, ctas):
    import numpy as np

    from akv_b200.context_tree import tree_work_list

    rng = np.random.default_rng(pair_heads + 2 * hkv + ctas)
    cached = np.r_[0, 1, 128, rng.integers(0, 3000, 9)]
    new = np.r_[1, 0, 64, rng.integers(0, 65, 9)]
    kv, dr = (np.concatenate(([0], np.cumsum(x))) for x in (cached, new))
    items, cta_items, merges, partials = tree_work_list(kv, dr, group, hkv, pair_heads, ctas)
    seen, parts = {}, {}
    for q0, n, kv0, prefix, lo, hi, h0, t0, hs, ts, u_n, partial in items.tolist():
        b = int(np.searchsorted(dr, q0, side="right")) - 1
        assert (q0, n, kv0, prefix) == (dr[b], new[b], kv[b], cached[b]) and n > 0
        assert u_n in (1, 2) and hs + ts == u_n - 1 and lo % 128 == 0 and lo < hi <= prefix + n
        assert pair_heads or not hs
        for u in range(u_n):
            key = (b, h0 + u * hs, t0 + u * ts)
            assert key[1] < hkv and key[2] * 128 < n * group
            seen.setdefault(key, []).append((lo, hi))
            parts.setdefault(key, []).append(-1 if partial < 0 else partial + u)
    for b in range(len(new)):
        for h in range(hkv):
            for t in range(-(-int(new[b]) * group // 128)):
                runs = sorted(seen.pop((b, h, t)))
                assert runs[0][0] == 0 and runs[-1][1] == cached[b] + new[b]
                assert all(x[1] == y[0] for x, y in zip(runs, runs[1:]))
    assert not seen
    used = sorted(p for v in parts.values() for p in v if p >= 0)
    assert len(set(used)) == len(used) and (not used or used[-1] < partials)
    assert partials <= 4 * ctas
    joined = set()
    for q0, n, h0, t0, steps, first, count, _ in merges.tolist():
        b = int(np.searchsorted(dr, q0, side="right")) - 1
        assert n == new[b] and count > 1
        for u in range(steps >> 2):
            key = (b, h0 + u * (steps & 1), t0 + u * (steps >> 1 & 1))
            assert sorted(parts[key]) == [first + u + 2 * i for i in range(count)]
            joined.add(key)
    assert joined == {k for k, v in parts.items() if v[0] >= 0}
    assert all(len(v) == 1 for k, v in parts.items() if k not in joined)
    assert cta_items[0] == 0 and cta_items[-1] == len(items) and np.all(np.diff(cta_items) >= 0)
    cost = -(-(items[:, 5] - items[:, 4]) // 128) * items[:, 10]
    load = [cost[a:b].sum() for a, b in zip(cta_items, cta_items[1:])]
    # Equal shares, each end off by less than two tiles of a pair.
    assert max(load) <= -(-cost.sum() // len(load)) + 6


def test_tree_work_list_refuses():
    from akv_b200.context_tree import tree_work_list

    for kv, dr in (([0, 5], [0]), ([0, 5], [0, 65]), ([5, 0], [0, 1]), ([0, 5], [1, 0]), ([], []),
                   ([0, 1 << 31], [0, 1])):
        with pytest.raises(ValueError):
            tree_work_list(kv, dr, 8, 8, True, 10)
