"""The drafted-token step as a server runs it, over a cache that a Drop and a
Reposition have compacted: slot maps of the drafted trees, then per layer the
Q/K norms with the rotation and the store, then the tree attention.  Every
layer's output is checked against the formulas in 64 bits.

Tolerance: the stored keys and the queries are checked to one rounding in
test_qk_rope_gpu.py; here the attention of what was stored is compared with
test_tree_gpu.py's bound."""

import numpy as np
import pytest
import torch

import test_tree_gpu as tree
from test_qk_rope_gpu import formula, near

pytestmark = pytest.mark.gpu

HKV, GROUP, D, LAYERS = 2, 8, 64, 2
HQ = HKV * GROUP


def compacted(page, seed):
    """Three requests after a Drop + Reposition of a paged pool, with room in
    their rows: what the server holds before it drafts."""
    from akv_b200.context_drop import DropCompactor, FreeSlotRing

    rng = np.random.default_rng(seed)
    counts = np.array([640, 1000, 70], np.int64)
    ranges = np.array([50, 200, 300, 420, 100, 900, 10, 20], np.int32)
    range_offsets = np.array([0, 2, 3, 4], np.int64)
    width = int(counts.max()) + 64
    pages = -(-(counts + 64) // page)
    ids = rng.permutation(int(pages.sum()) + 40).astype(np.int32) + 1
    table = np.zeros((5, width), np.int32)
    row_ids = np.array([3, 1, 4], np.int64)
    at = 0
    for b, n in enumerate(counts):
        used = -(-int(n) // page)
        own = ids[at: at + used]
        at += used
        table[row_ids[b], :n] = (np.repeat(own * page, page) + np.tile(np.arange(page), used))[:n]
    req_to_token = torch.from_numpy(table).cuda()
    ring = FreeSlotRing(torch.from_numpy(ids[at:]), capacity=len(ids) + 200, device="cuda")
    comp = DropCompactor(int(counts.sum()), 3, len(ranges) // 2, torch.device("cuda", 0))
    res = comp.run(counts, range_offsets, ranges, req_to_token, row_ids, ring, page_size=page)
    torch.cuda.synchronize()
    assert int(res.status[0]) == 0
    slots = (int(ids.max()) + 1) * page
    return dict(rng=rng, counts=counts, row_ids=torch.from_numpy(row_ids).cuda(), ring=ring,
                rows=req_to_token, offsets=res.active_offsets.clone(),
                raw=res.raw_indices.clone(), next=res.next_position.clone(), slots=slots)


@pytest.mark.parametrize("page", [4, 16])
def test_a_step_after_a_drop(page):
    from akv_b200.context_rope import qk_norm_rope
    from akv_b200.context_slots import SlotMapper
    from akv_b200.context_tree import TreeAttention
    from akv_b200.rope import rope_cos_sin_cache

    s = compacted(page, page)
    new = np.array([9, 16, 5], np.int64)
    total = int(new.sum())
    kv = s["offsets"].cpu().numpy().astype(np.int64)[:4]
    dr = np.concatenate(([0], np.cumsum(new)))
    parents = np.concatenate([[s["rng"].integers(-1, i) if i else -1 for i in range(n)] for n in new])
    g = torch.Generator(device="cuda").manual_seed(page)
    rand = lambda *a: torch.randn(*a, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    pools = [(rand(s["slots"], HKV, D), rand(s["slots"], HKV, D)) for _ in range(LAYERS)]
    qkv = [rand(total, (HQ + 2 * HKV) * D) for _ in range(LAYERS)]
    wq, wk = 1 + 0.2 * rand(D), 1 + 0.2 * rand(D)
    sinks = torch.randn(HQ, generator=g, device="cuda")
    table = rope_cos_sin_cache(2048, D, 10000.0).cuda()
    # The cached keys' slots, from the compacted view.
    req = torch.repeat_interleave(s["row_ids"], torch.from_numpy(np.diff(kv)).cuda())
    kv_indices = s["rows"][req, s["raw"][: kv[-1]].long()].contiguous()

    mapper = SlotMapper(3, total, "cuda", page_size=page)
    attn = TreeAttention(HQ, HKV, D, 3, "cuda").plan(kv, dr)
    raw_lens = torch.from_numpy(s["counts"]).cuda()
    new_lens, up = torch.from_numpy(new).cuda(), torch.from_numpy(parents.astype(np.int32)).cuda()
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    queries = [torch.empty(total, HQ, D, dtype=torch.bfloat16, device="cuda") for _ in range(LAYERS)]
    outs = [torch.empty_like(q) for q in queries]

    def step():
        view = mapper.run(s["rows"], s["row_ids"], raw_lens, new_lens, s["ring"],
                          next_positions=s["next"], parents=up, commit=False)
        for layer, (kp, vp) in enumerate(pools):
            q, k, v = (t.view(total, -1, D) for t in
                       qkv[layer].split([HQ * D, HKV * D, HKV * D], 1))
            qk_norm_rope(q, k, view.positions, table, q_weight=wq, k_weight=wk, v=v, k_pool=kp,
                         v_pool=vp, slots=view.slots, q_out=queries[layer], error_flag=flag)
            attn.run(queries[layer], kp, vp, kv_indices, view.slots, view.tree_mask, sinks=sinks,
                     out=outs[layer])
        return view

    def check(view):
        view.check()
        attn.check()
        assert int(flag) == 0
        mask, depth = tree.masks(parents, dr)
        assert np.array_equal(view.tree_mask.cpu().numpy(), mask)
        positions = np.repeat(s["next"].cpu().numpy()[:3], new) + depth
        assert view.positions.tolist() == positions.tolist()
        assert len(set(view.slots.tolist()) | set(kv_indices.tolist())) == total + int(kv[-1])
        pos = torch.from_numpy(positions).cuda()
        for layer, (kp, vp) in enumerate(pools):
            q, k, v = (t.view(total, -1, D) for t in
                       qkv[layer].split([HQ * D, HKV * D, HKV * D], 1))
            near(queries[layer], *formula(q, wq, table, pos, True, 1e-6), D)
            near(kp[view.slots.long()], *formula(k, wk, table, pos, True, 1e-6), D)
            assert torch.equal(vp[view.slots.long()], v)
            case = dict(q=queries[layer], k=kp, v=vp, kv=kv, dr=dr, indices=kv_indices,
                        draft=view.slots, mask=view.tree_mask, window=-1, qpos=view.positions,
                        kpos=None, sinks=sinks, hkv=HKV, group=GROUP, d=D, dtype=torch.bfloat16)
            want, _, mean, size = tree.exact(case)
            e32 = (D + 4) * 2.0**-23 * size + 2.0**-21 + 1100 * 2.0**-24
            bound = 2.0**-8 * want.abs() + (2.0**-8 + 2 * e32[..., None]) * mean + 2.0**-24
            assert bool(((outs[layer].double() - want).abs() <= bound * 1.01).all())

    check(step())
    # The whole step again from a graph, with other projections and trees.
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        view = step()
    for t in qkv:
        t.copy_(rand(*t.shape))
    parents[:] = np.concatenate([np.arange(n) - 1 for n in new])
    up.copy_(torch.from_numpy(parents.astype(np.int32)))
    for out in outs:
        out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    check(view)
