"""The drafted-token step of a fixed size over a compacted cache: a mapper and
projections larger than the batch, a full and a sliding-window layer, page
size 1 and more, eager and from one graph over several batches.  Tolerances
as in test_draft_step_gpu.py."""

import numpy as np
import pytest
import torch

import test_tree_gpu as tree
from test_qk_rope_gpu import formula, near

pytestmark = pytest.mark.gpu

HKV, GROUP, D, BATCH, ROOM, WINDOW = 2, 8, 64, 3, 48, 300
HQ = HKV * GROUP


@pytest.mark.parametrize("page", [1, 16])
def test_a_padded_step_with_a_window_layer(page):
    from akv_b200.context_drop import DropCompactor, FreeSlotRing
    from akv_b200.context_rope import qk_norm_rope
    from akv_b200.context_slots import SlotMapper
    from akv_b200.context_tree import TreeAttention
    from akv_b200.rope import rope_cos_sin_cache

    rng = np.random.default_rng(page)
    g = torch.Generator(device="cuda").manual_seed(page)
    rand = lambda *a: torch.randn(*a, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    counts = np.array([640, 1000, 70], np.int64)
    ranges = np.array([50, 200, 300, 420, 100, 900, 10, 20], np.int32)
    used = -(-counts // page)
    ids = rng.permutation(int(used.sum()) + 200).astype(np.int32) + 1
    rows = np.zeros((5, 1200), np.int32)
    row_ids = np.array([3, 1, 4], np.int64)
    at = 0
    for b, n in enumerate(counts):
        own = ids[at: at + used[b]]
        at += used[b]
        rows[row_ids[b], :n] = (np.repeat(own * page, page) + np.tile(np.arange(page), used[b]))[:n]
    rows = torch.from_numpy(rows).cuda()
    ring = FreeSlotRing(torch.from_numpy(ids[at:]), capacity=len(ids) + 1200, device="cuda")
    drop = DropCompactor(int(counts.sum()), 3, 4, torch.device("cuda", 0)).run(
        counts, np.array([0, 2, 3, 4]), ranges, rows, row_ids, ring, page_size=page)
    drop.check()
    kv = drop.active_offsets.cpu().numpy().astype(np.int64)
    row_ids = torch.from_numpy(row_ids).cuda()
    owner = torch.repeat_interleave(row_ids, torch.from_numpy(np.diff(kv)).cuda())
    kv_indices = rows[owner, drop.raw_indices[: kv[-1]].long()].contiguous()
    kv_positions = drop.active_positions[: kv[-1]]     # in the order of kv_indices

    slots = (int(ids.max()) + 1) * page
    pools = [(rand(slots, HKV, D), rand(slots, HKV, D)) for _ in range(2)]
    windows = [-1, WINDOW]
    qkv = [rand(ROOM, (HQ + 2 * HKV) * D) for _ in pools]
    queries = [torch.zeros(ROOM, HQ, D, dtype=torch.bfloat16, device="cuda") for _ in pools]
    outs = [torch.zeros_like(q) for q in queries]
    weight = 1 + 0.2 * rand(D)
    sinks = torch.randn(HQ, generator=g, device="cuda")
    table = rope_cos_sin_cache(2048, D, 10000.0).cuda()
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    raw_lens, new_lens = torch.from_numpy(counts).cuda(), torch.zeros(BATCH, dtype=torch.int64, device="cuda")
    up = torch.zeros(ROOM, dtype=torch.int32, device="cuda")
    mapper = SlotMapper(BATCH, ROOM, "cuda", page_size=page)
    attn = TreeAttention(HQ, HKV, D, BATCH, "cuda")

    def step():
        view = mapper.run(rows, row_ids, raw_lens, new_lens, ring, next_positions=drop.next_position,
                          parents=up, commit=False, keep_offsets=True)
        for (kp, vp), x, q_out, out, window in zip(pools, qkv, queries, outs, windows):
            q, k, v = (t.view(ROOM, -1, D) for t in x.split([HQ * D, HKV * D, HKV * D], 1))
            qk_norm_rope(q, k, view.positions, table, q_weight=weight, k_weight=weight, v=v, k_pool=kp,
                         v_pool=vp, slots=view.slots, q_out=q_out, error_flag=flag)
            attn.run(q_out, kp, vp, kv_indices, view.slots, view.tree_mask, sinks=sinks, window=window,
                     q_positions=view.positions, kv_positions=kv_positions, out=out)
        return view

    def batch(new):
        """Sets the step's inputs; returns what it may not change."""
        parents = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(n)] for n in new]
                                 + [[]]).astype(np.int32)
        up[: len(parents)] = torch.from_numpy(parents).cuda()
        new_lens.copy_(torch.tensor(new))
        for x in qkv:
            x.copy_(rand(*x.shape))
        for out in outs:
            out.fill_(5)
        dr = np.concatenate(([0], np.cumsum(new))).astype(np.int64)
        attn.plan(kv, dr)
        return parents, dr, [[p.clone() for p in layer] for layer in pools]

    def check(view, parents, dr, before):
        view.check()
        attn.check()
        total = int(dr[-1])
        assert int(flag) == 0 and view.slots[total:].tolist() == [-1] * (ROOM - total)
        at = view.slots[:total].long()
        assert len(set(at.tolist()) | set(kv_indices.tolist())) == total + int(kv[-1])
        rest = torch.ones(slots, dtype=torch.bool, device="cuda")
        rest[at] = False
        positions = view.positions[:total]
        for n, (kp, vp) in enumerate(pools):
            q, k, v = (t.view(ROOM, -1, D)[:total] for t in qkv[n].split([HQ * D, HKV * D, HKV * D], 1))
            near(queries[n][:total], *formula(q, weight, table, positions, True, 1e-6), D)
            near(kp[at], *formula(k, weight, table, positions, True, 1e-6), D)
            assert torch.equal(vp[at], v)
            for pool, old in zip((kp, vp), before[n]):
                assert torch.equal(pool[rest], old[rest])
            assert bool((outs[n][total:] == 5).all())
            case = dict(q=queries[n][:total], k=kp, v=vp, kv=kv, dr=dr, indices=kv_indices,
                        draft=view.slots[:total], mask=torch.from_numpy(tree.masks(parents, dr)[0]).cuda(),
                        window=windows[n], qpos=positions, kpos=kv_positions, sinks=sinks, hkv=HKV,
                        group=GROUP, d=D, dtype=torch.bfloat16)
            want, _, mean, size = tree.exact(case)
            e32 = (D + 4) * 2.0**-23 * size + 2.0**-21 + 1100 * 2.0**-24
            bound = 2.0**-8 * want.abs() + (2.0**-8 + 2 * e32[..., None]) * mean + 2.0**-24
            assert bool(((outs[n][:total].double() - want).abs() <= bound * 1.01).all())

    inputs = batch([9, 16, 5])
    check(step(), *inputs)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        view = step()
    for new in ([16, 16, 16], [1, 0, 3], [0, 0, 0], [7, 30, 1]):
        inputs = batch(new)
        graph.replay()
        check(view, *inputs)
