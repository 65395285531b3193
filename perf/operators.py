"""The speculative-decoding step over a paged cache, operator by operator.

One step of a server that drafts a tree of tokens for each request and
verifies them in one forward pass runs, once: the slot maps, positions, tree
masks and block tables of the drafted tokens (``op`` "slots"); and in every
layer: the per-head norms of Q and K with the position rotation and the store
into the cache ("rope"), then the attention of the drafted tokens over the
cache and over their own ancestors ("tree").  Prompt chunks use the first two
in the same way with thousands of new tokens and no tree.

``run`` computes each operator in plain torch (``own`` false) or by this
repository's entry points (``own`` true).
"""

import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
THETA = 150000.0


# ---------------------------------------------------------------- cases

def listed():
    return [
        # One user, a short draft tree, a pool of single slots: latency.
        {"name": "slots_one", "op": "slots", "batch": 1, "page": 1, "new_lo": 8, "new_hi": 8,
         "len_lo": 4096, "len_hi": 4096, "tree": True, "table": False, "ragged": 1},
        # An ordinary serving batch over a paged pool, block tables for a paged reader.
        {"name": "slots_pages", "op": "slots", "batch": 64, "page": 16, "new_lo": 16, "new_hi": 16,
         "len_lo": 2048, "len_hi": 32768, "tree": True, "table": True, "ragged": 2},
        # A large batch with requests that draft nothing, few or 64 tokens.
        {"name": "slots_ragged", "op": "slots", "batch": 512, "page": 1, "new_lo": 0, "new_hi": 64,
         "len_lo": 0, "len_hi": 16384, "tree": True, "table": True, "ragged": 3},
        # Prompt chunks of up to 8191 tokens behind cached prefixes; no tree.
        {"name": "slots_prompt", "op": "slots", "batch": 16, "page": 64, "new_lo": 1, "new_hi": 8191,
         "len_lo": 0, "len_hi": 65536, "tree": False, "table": True, "ragged": 4},
        # One decoded token of a 64-head model: latency.
        {"name": "rope_token", "op": "rope", "tokens": 1, "hq": 64, "hkv": 8, "dim": 64, "rotary": 64,
         "neox": True, "dtype": "bf16", "store": True, "pad": 0},
        # 128 requests of 16 drafted tokens, some of them padding without a slot.
        {"name": "rope_draft", "op": "rope", "tokens": 2048, "hq": 64, "hkv": 8, "dim": 64, "rotary": 64,
         "neox": True, "dtype": "bf16", "store": True, "pad": 37},
        # A prompt chunk of head_dim 128, an odd number of tokens.
        {"name": "rope_prompt", "op": "rope", "tokens": 16411, "hq": 64, "hkv": 8, "dim": 128,
         "rotary": 128, "neox": True, "dtype": "bf16", "store": True, "pad": 0},
        # fp16, half of each head rotated in adjacent pairs, keys returned instead of stored.
        {"name": "rope_pairs", "op": "rope", "tokens": 4097, "hq": 32, "hkv": 4, "dim": 128,
         "rotary": 64, "neox": False, "dtype": "fp16", "store": False, "pad": 0},
        # One user, four drafted tokens over a short cache: latency.
        {"name": "tree_one", "op": "tree", "batch": 1, "new_lo": 4, "new_hi": 4, "len_lo": 1000,
         "len_hi": 1000, "hkv": 8, "group": 8, "dim": 64, "dtype": "bf16", "sinks": True,
         "window": -1, "lse": False, "ragged": 5},
        # The ordinary verification step: 64 requests of 16 drafted tokens.
        {"name": "tree_batch", "op": "tree", "batch": 64, "new_lo": 16, "new_hi": 16, "len_lo": 4096,
         "len_hi": 12288, "hkv": 8, "group": 8, "dim": 64, "dtype": "bf16", "sinks": True,
         "window": -1, "lse": False, "ragged": 6},
        # Wide trees over long caches, head_dim 128.
        {"name": "tree_wide", "op": "tree", "batch": 8, "new_lo": 33, "new_hi": 64, "len_lo": 16384,
         "len_hi": 32768, "hkv": 8, "group": 8, "dim": 128, "dtype": "bf16", "sinks": False,
         "window": -1, "lse": True, "ragged": 7},
        # A sliding-window layer: the window's keys of 128 requests, in fp16.
        {"name": "tree_window", "op": "tree", "batch": 128, "new_lo": 8, "new_hi": 8, "len_lo": 100,
         "len_hi": 140, "hkv": 8, "group": 8, "dim": 64, "dtype": "fp16", "sinks": True,
         "window": 128, "lse": False, "ragged": 8},
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["slots", "rope", "tree"])
    if op == "slots":
        tree = rng.random() < 0.7
        batch = _log(rng, 1, 512)
        new_hi = _log(rng, 1, 64) if tree else _log(rng, 1, min(8191, max(1, 131072 // batch)))
        len_hi = _log(rng, 1, min(65536, (512 * 16384) // batch))
        return {"op": op, "batch": batch, "page": rng.choice([1, 4, 16, 64, 128]),
                "new_lo": rng.randint(0, new_hi), "new_hi": new_hi,
                "len_lo": rng.randint(0, len_hi), "len_hi": len_hi, "tree": tree,
                "table": rng.random() < 0.7, "ragged": rng.randint(0, 1 << 30)}
    if op == "rope":
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4, 5, 8, 16])
        dim = rng.choice([64, 128, 256])
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        rotary = rng.choice([dim, dim, dim // 2])
        top = (16411 * 80 * 128 * 2) // ((hq + 2 * hkv) * dim * DTYPES[dtype].itemsize)
        tokens = _log(rng, 1, min(65536, top))
        return {"op": op, "tokens": tokens, "hq": hq, "hkv": hkv, "dim": dim, "rotary": rotary,
                "neox": rng.random() < 0.7, "dtype": dtype, "store": rng.random() < 0.7,
                "pad": rng.randint(0, tokens // 8)}
    hkv, group = rng.choice([1, 2, 4, 8]), rng.choice([1, 2, 4, 5, 8, 8, 8, 16])
    dim = rng.choice([64, 128])
    new_hi = _log(rng, 1, 64)
    batch = _log(rng, 1, 128)
    # Not above the listed cases' scores (batch x rows x keys) or gathered keys.
    scores = 8 * 8 * 512 * 24576
    keys = 64 * 8192 * 8 * 64
    top = min(32768, scores // (batch * hkv * group * new_hi), keys // (batch * hkv * dim))
    len_hi = _log(rng, 1, max(1, top))
    window = rng.choice([-1, -1, -1, 128, 1024])
    if window >= 0:
        len_hi = min(len_hi, window + 12)
    return {"op": op, "batch": batch, "new_lo": rng.randint(1, new_hi), "new_hi": new_hi,
            "len_lo": rng.randint(len_hi // 2, len_hi), "len_hi": len_hi, "hkv": hkv,
            "group": group, "dim": dim, "dtype": rng.choice(["bf16", "bf16", "fp16"]),
            "sinks": rng.random() < 0.5, "window": window, "lse": rng.random() < 0.5,
            "ragged": rng.randint(0, 1 << 30)}


def _lengths(case):
    """Cached and new lengths of each request: of the case alone, not of the seed."""
    r = np.random.default_rng(case["ragged"])
    cached = r.integers(case["len_lo"], case["len_hi"] + 1, case["batch"])
    new = r.integers(case["new_lo"], case["new_hi"] + 1, case["batch"])
    if new.sum() == 0:
        new[0] = 1
    return cached.astype(np.int64), new.astype(np.int64)


def work(case):
    if case["op"] == "slots":
        cached, new = _lengths(case)
        page, total = case["page"], int(new.sum())
        pages_old = int((-(-cached // page)).sum())
        pages = int((-(-(cached + new) // page)).sum())
        moved = 20 * case["batch"] + 4 * (pages - pages_old)   # lengths, positions, rows; lent pages
        moved += total * (4 + 4 + 4)                           # row entries, slot map, positions
        if case["tree"]:
            moved += total * (4 + 8)                           # parents in, masks out
        if case["table"]:
            moved += 4 * pages_old + 4 * pages                 # one row entry a page in, the table out
        return {"bytes": moved, "flops": 0}
    if case["op"] == "rope":
        t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
        size = DTYPES[case["dtype"]].itemsize
        heads = hq + 2 * hkv if case["store"] else hq + hkv
        return {"bytes": 2 * t * heads * d * size + t * (4 * case["rotary"] + 4)
                + (4 * t if case["store"] else 0) + 2 * d * size,
                "flops": t * (hq + hkv) * (4 * d + 3 * case["rotary"])}
    cached, new = _lengths(case)
    hkv, hq, d = case["hkv"], case["hkv"] * case["group"], case["dim"]
    keys, total = int((cached + new).sum()), int(new.sum())
    return {"bytes": keys * (hkv * d * 4 + 4) + total * (hq * d * 4 + 8)
            + (4 * keys if case["window"] >= 0 else 0),
            "flops": 4 * hq * d * int((new * (cached + 1)).sum())}


# ---------------------------------------------------------------- inputs

def _indptr(n):
    return np.concatenate(([0], np.cumsum(n))).astype(np.int64)


def _parents(rng, new):
    """Draft trees in topological order: node 0 the root, a later node's parent one of the eight
    nodes before it; -1 for a root.  int32, node numbers of the request."""
    i = np.concatenate([np.arange(n) for n in new])
    back = rng.integers(1, 9, len(i))
    return np.where(i == 0, -1, np.maximum(i - back, 0)).astype(np.int32)


def _masks(parents, indptr):
    """One 64-bit word per node: the bits of its ancestors and its own; and the depths."""
    mask = np.zeros(len(parents), np.uint64)
    depth = np.zeros(len(parents), np.int32)
    start = np.repeat(indptr[:-1], np.diff(indptr))
    node = np.arange(len(parents)) - start
    for i in range(int(node.max()) + 1):
        at = np.nonzero(node == i)[0]
        up = start[at] + np.maximum(parents[at], 0)
        has = parents[at] >= 0
        mask[at] = np.where(has, mask[up], np.uint64(0)) | (np.uint64(1) << np.uint64(i))
        depth[at] = np.where(has, depth[up] + 1, 0)
    return mask.view(np.int64), depth


def prepare(case, seed):
    return {"slots": _prepare_slots, "rope": _prepare_rope, "tree": _prepare_tree}[case["op"]](case, seed)


def _prepare_slots(case, seed):
    rng = np.random.default_rng(seed)
    cached, new = _lengths(case)
    page, batch, total = case["page"], case["batch"], int(new.sum())
    old_pages = -(-cached // page)
    all_pages = -(-(cached + new) // page)
    lent = int((all_pages - old_pages).sum())
    width = (int((cached + new).max()) + 63) // 64 * 64
    rows = batch + 3
    ids = rng.permutation(int(old_pages.sum()) + lent + 64).astype(np.int32) + 1
    # Rows of the cached tokens, each request at a row of its own.
    row_ids = rng.permutation(rows)[:batch].astype(np.int64)
    table = np.zeros((rows, width), np.int32)
    at = _indptr(old_pages)
    for b in range(batch):
        pages = ids[at[b]: at[b + 1]]
        table[row_ids[b], : cached[b]] = (np.repeat(pages * page, page)
                                          + np.tile(np.arange(page, dtype=np.int32), len(pages)))[: cached[b]]
    free = ids[int(old_pages.sum()):]
    head = int(rng.integers(0, len(free)))
    dev = "cuda"
    state = {
        "case": case,
        "req_to_token": torch.from_numpy(table).to(dev),
        "row_ids": torch.from_numpy(row_ids).to(dev),
        "raw_lens": torch.from_numpy(cached).to(dev),
        "new_lens": torch.from_numpy(new).to(dev),
        # Positions follow the compacted cache, which dropped tokens left shorter than the row.
        "next_positions": torch.from_numpy((cached - rng.integers(0, cached // 4 + 1)).astype(np.int32)).to(dev),
        "parents": torch.from_numpy(_parents(rng, new)).to(dev) if case["tree"] else None,
        # The free list as a ring: entry (head + k) % capacity is the k-th free page.
        "ring": torch.from_numpy(np.roll(free, head)).to(dev),
        "ring_state": torch.tensor([head, head + len(free)], dtype=torch.int64, device=dev),
        "block_table": torch.full((batch, int(all_pages.max()) + 5), -1, dtype=torch.int32, device=dev)
        if case["table"] else None,
        "total": total,
    }
    if own:
        from akv_b200.context_drop import FreeSlotRing
        from akv_b200.context_slots import SlotMapper

        free_ring = FreeSlotRing([], capacity=len(free), device=dev)
        free_ring.ring.copy_(state["ring"])
        free_ring.state.copy_(state["ring_state"])
        state["free_ring"] = free_ring
        state["mapper"] = SlotMapper(batch, total, dev, page_size=page)
    return state


def _prepare_rope(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    t, hq, hkv, d = case["tokens"], case["hq"], case["hkv"], case["dim"]
    dtype, dev = DTYPES[case["dtype"]], "cuda"
    # The fused projection's output: Q, K and V are views of it.
    qkv = torch.randn(t, (hq + 2 * hkv) * d, generator=g, device=dev).mul_(2.0).to(dtype)
    q, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=1)
    inv = 1.0 / THETA ** (torch.arange(0, case["rotary"], 2, dtype=torch.float64, device=dev) / case["rotary"])
    angle = torch.arange(131072, dtype=torch.float64, device=dev)[:, None] * inv
    slots = t + 61
    where = rng.permutation(slots - 1)[:t].astype(np.int32) + 1   # slot 0 stays free, as a pool keeps it
    if case["pad"]:
        where[rng.permutation(t)[: case["pad"]]] = -1             # padding tokens have no slot
    return {
        "case": case,
        "q": q.view(t, hq, d), "k": k.view(t, hkv, d), "v": v.view(t, hkv, d),
        "positions": torch.from_numpy(rng.integers(0, 131072, t).astype(np.int32)).to(dev),
        "cos_sin": torch.cat((angle.cos(), angle.sin()), 1).float(),
        "q_weight": (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dtype),
        "k_weight": (1 + 0.2 * torch.randn(d, generator=g, device=dev)).to(dtype),
        "k_pool": torch.randn(slots, hkv, d, generator=g, device=dev).to(dtype) if case["store"] else None,
        "v_pool": torch.randn(slots, hkv, d, generator=g, device=dev).to(dtype) if case["store"] else None,
        "slots": torch.from_numpy(where).to(dev) if case["store"] else None,
    }


def _prepare_tree(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rng = np.random.default_rng(seed)
    cached, new = _lengths(case)
    hkv, hq, d = case["hkv"], case["hkv"] * case["group"], case["dim"]
    dtype, dev = DTYPES[case["dtype"]], "cuda"
    kv_indptr, draft_indptr = _indptr(cached), _indptr(new)
    keys, total = int(kv_indptr[-1]), int(draft_indptr[-1])
    slots = keys + total + 64
    place = rng.permutation(slots).astype(np.int32)   # every token at a slot of its own, in no order
    mask, depth = _masks(_parents(rng, new), draft_indptr)
    # Positions of the cached keys, with the gaps that dropped spans leave; the draft goes on behind.
    steps = rng.integers(1, 3, keys) if case["window"] >= 0 else np.ones(keys, np.int64)
    run_of = np.cumsum(steps)
    first = np.concatenate(([0], run_of))[kv_indptr[:-1]]
    kv_pos = run_of - np.repeat(first, cached)
    end = np.array([kv_pos[kv_indptr[b + 1] - 1] if cached[b] else 0 for b in range(len(cached))])
    q_pos = np.repeat(end + 1, new) + depth
    state = {
        "case": case,
        "q": torch.randn(total, hq, d, generator=g, device=dev).mul_(1.5).to(dtype),
        "k_pool": torch.randn(slots, hkv, d, generator=g, device=dev).to(dtype),
        "v_pool": torch.randn(slots, hkv, d, generator=g, device=dev).to(dtype),
        "kv_indptr_host": kv_indptr, "draft_indptr_host": draft_indptr,
        "kv_indptr": torch.from_numpy(kv_indptr).to(dev),
        "draft_indptr": torch.from_numpy(draft_indptr).to(dev),
        "kv_indices": torch.from_numpy(place[:keys]).to(dev),
        "draft_slots": torch.from_numpy(place[keys: keys + total]).to(dev),
        "tree_mask": torch.from_numpy(mask).to(dev),
        "kv_positions": torch.from_numpy(kv_pos.astype(np.int32)).to(dev),
        "q_positions": torch.from_numpy(q_pos.astype(np.int32)).to(dev),
        "sinks": torch.randn(hq, generator=g, device=dev) if case["sinks"] else None,
        "key_top": int(cached.max()), "new_top": int(new.max()), "total": total,
    }
    if own:
        from akv_b200.context_tree import TreeAttention

        state["attn"] = TreeAttention(hq, hkv, d, len(cached), dev, dtype=dtype)
        state["attn"].plan(kv_indptr, draft_indptr)
    return state


# ---------------------------------------------------------------- one pass

def run(state):
    return {"slots": _run_slots, "rope": _run_rope, "tree": _run_tree}[state["case"]["op"]](state)


def _run_slots(s):
    page = s["case"]["page"]
    if own:
        # The pages are lent: taken for good once the accepted tokens are known.
        view = s["mapper"].run(s["req_to_token"], s["row_ids"], s["raw_lens"], s["new_lens"],
                               s["free_ring"], next_positions=s["next_positions"],
                               parents=s["parents"], block_table=s["block_table"], commit=False)
        return {"offsets": view.new_offsets, "slots": view.slots, "positions": view.positions,
                "mask": view.tree_mask, "rows": s["req_to_token"], "table": s["block_table"],
                "status": view.status}
    dev, batch, total = s["row_ids"].device, len(s["row_ids"]), s["total"]
    cached, new, table = s["raw_lens"], s["new_lens"], s["req_to_token"]
    old_pages, all_pages = (cached + page - 1) // page, (cached + new + page - 1) // page
    need = all_pages - old_pages
    base = need.cumsum(0) - need
    offsets = torch.zeros(batch + 1, dtype=torch.int32, device=dev)
    offsets[1:] = new.cumsum(0)
    req = torch.repeat_interleave(torch.arange(batch, device=dev), new, output_size=total)
    i = torch.arange(total, device=dev) - offsets[req]
    t = cached[req] + i
    row = s["row_ids"][req]
    last = table[row, (cached[req] - 1).clamp(min=0)].long() // page     # the page that the row ends in
    k = base[req] + t // page - old_pages[req]
    head, capacity = s["ring_state"][0], len(s["ring"])
    fresh = s["ring"][(head + k.clamp(min=0)) % capacity].long()
    slots = (torch.where(t // page < old_pages[req], last, fresh) * page + t % page).int()
    table[row, t] = slots
    mask = None
    step = i
    if s["parents"] is not None:
        up = s["parents"].long()
        link = torch.zeros(batch, 64, 64, device=dev)
        link[req, i, up.clamp(min=0)] = (up >= 0).float()
        link += torch.eye(64, device=dev)
        seen = torch.linalg.matrix_power(link, 64)[req, i] > 0           # ancestors, and the node
        step = seen.sum(1) - 1
        mask = (seen.long() << torch.arange(64, device=dev)).sum(1)
    positions = (s["next_positions"][req] + step).int()
    if s["block_table"] is not None:
        out = s["block_table"]
        g = torch.arange(out.shape[1], device=dev)[None]
        at = (g * page).clamp(max=table.shape[1] - 1)
        ids = table[s["row_ids"][:, None], at] // page
        out.copy_(torch.where(g < all_pages[:, None], ids, out))
    enough = need.sum() <= s["ring_state"][1] - head
    return {"offsets": offsets, "slots": slots, "positions": positions, "mask": mask, "rows": table,
            "table": s["block_table"], "status": (~enough).int()[None]}


def _run_rope(s):
    case = s["case"]
    if own:
        from akv_b200.context_rope import qk_norm_rope

        q, k = qk_norm_rope(s["q"], s["k"], s["positions"], s["cos_sin"], q_weight=s["q_weight"],
                            k_weight=s["k_weight"], eps=1e-6, is_neox_style=case["neox"],
                            v=s["v"] if case["store"] else None, k_pool=s["k_pool"],
                            v_pool=s["v_pool"], slots=s["slots"])
        return {"q": q, "k": k, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}
    half = case["rotary"] // 2
    table = s["cos_sin"][s["positions"].long()][:, None]
    cos, sin = table[..., :half], table[..., half:]

    def turn(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
        r = x[..., : 2 * half]
        if case["neox"]:
            a, b = r[..., :half], r[..., half:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        else:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        return torch.cat((r, x[..., 2 * half:]), -1).to(s["q"].dtype)

    q, k = turn(s["q"], s["q_weight"]), turn(s["k"], s["k_weight"])
    if not case["store"]:
        return {"q": q, "k": k, "k_pool": None, "v_pool": None}
    # Tokens without a slot write slot 0's own rows back to it.
    at = s["slots"].long().clamp(min=0)
    real = (s["slots"] >= 0)[:, None, None]
    s["k_pool"][at] = torch.where(real, k, s["k_pool"][0])
    s["v_pool"][at] = torch.where(real, s["v"], s["v_pool"][0])
    return {"q": q, "k": None, "k_pool": s["k_pool"], "v_pool": s["v_pool"]}


def _run_tree(s):
    case = s["case"]
    if own:
        out, lse = s["attn"].run(
            s["q"], s["k_pool"], s["v_pool"], s["kv_indices"], s["draft_slots"], s["tree_mask"],
            sinks=s["sinks"], window=case["window"], q_positions=s["q_positions"],
            kv_positions=s["kv_positions"], return_lse=True) if case["lse"] else (s["attn"].run(
                s["q"], s["k_pool"], s["v_pool"], s["kv_indices"], s["draft_slots"], s["tree_mask"],
                sinks=s["sinks"], window=case["window"], q_positions=s["q_positions"],
                kv_positions=s["kv_positions"]), None)
        return {"out": out, "lse": lse}
    hkv, group, d = case["hkv"], case["group"], case["dim"]
    dev, batch, total = s["q"].device, len(s["kv_indptr"]) - 1, s["total"]
    L, n = s["key_top"], s["new_top"]
    kv0, d0 = s["kv_indptr"], s["draft_indptr"]
    lens, new = kv0.diff(), d0.diff()
    # Everything padded to the longest request: [prefix | draft] keys, and queries.
    j = torch.arange(L, device=dev)[None]
    i = torch.arange(n, device=dev)[None]
    has_key, has_node = j < lens[:, None], i < new[:, None]
    key_at = (kv0[:-1, None] + j).clamp(max=max(0, len(s["kv_indices"]) - 1))
    node_at = (d0[:-1, None] + i).clamp(max=total - 1)
    prefix = torch.where(has_key, s["kv_indices"][key_at].long(), 0) if len(s["kv_indices"]) else \
        torch.zeros(batch, L, dtype=torch.long, device=dev)
    slot = torch.cat((prefix, torch.where(has_node, s["draft_slots"][node_at].long(), 0)), 1)
    keys = s["k_pool"][slot].float().permute(0, 2, 3, 1)                         # [B, Hkv, D, T]
    q = s["q"][node_at].float().view(batch, n, hkv, group, d).permute(0, 2, 1, 3, 4)
    scores = (q.reshape(batch, hkv, n * group, d) @ keys) / math.sqrt(d)
    del keys
    bits = (s["tree_mask"][node_at][:, :, None] >> torch.arange(n, device=dev)) & 1
    seen = torch.cat((has_key[:, None].expand(-1, n, -1), (bits > 0) & has_node[:, None]), 2)
    if case["window"] >= 0:
        qp = s["q_positions"][node_at]
        kp = torch.cat((s["kv_positions"][key_at], qp), 1) if len(s["kv_indices"]) else \
            torch.cat((torch.zeros(batch, L, dtype=torch.int32, device=dev), qp), 1)
        seen = seen & (qp[:, :, None] - kp[:, None] <= case["window"])
    scores = scores.view(batch, hkv, n, group, L + n).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    if s["sinks"] is not None:
        sink = s["sinks"].view(1, hkv, 1, group, 1)
        top = torch.maximum(top, sink)
    top = torch.where(top == -math.inf, 0.0, top)
    p = scores.sub_(top).exp_()
    den = p.sum(-1, keepdim=True)
    if s["sinks"] is not None:
        den = den + torch.exp(sink - top)
    values = s["v_pool"][slot].float().permute(0, 2, 1, 3)                       # [B, Hkv, T, D]
    o = (p.view(batch, hkv, n * group, L + n) @ values).view(batch, hkv, n, group, d)
    o = o / torch.where(den > 0, den, 1.0)
    req = torch.repeat_interleave(torch.arange(batch, device=dev), new, output_size=total)
    node = torch.arange(total, device=dev) - d0[req]
    out = o[req, :, node].reshape(total, hkv * group, d).to(s["q"].dtype)
    lse = (top + den.log())[req, :, node].reshape(total, hkv * group) if case["lse"] else None
    return {"out": out, "lse": lse}


# ---------------------------------------------------------------- 64 bits

def exact(case, seed):
    return {"slots": _exact_slots, "rope": _exact_rope, "tree": _exact_tree}[case["op"]](case, seed)


def _exact_slots(case, seed):
    s = _prepare_slots(case, seed)
    page = case["page"]
    table, ring = s["req_to_token"].cpu().numpy(), s["ring"].cpu().numpy()
    blocks = s["block_table"].cpu().numpy() if case["table"] else None
    head, tail = s["ring_state"].tolist()
    rows, cached, new = (s[k].tolist() for k in ("row_ids", "raw_lens", "new_lens"))
    at, slots, positions, masks, offsets = head, [], [], [], [0]
    parents = s["parents"].tolist() if case["tree"] else None
    for b, r in enumerate(rows):
        start, mask, depth = s["next_positions"][b].item(), [], []
        for i in range(new[b]):
            t = cached[b] + i
            if t % page:
                slot = table[r, t - 1] + 1
            else:
                slot = ring[at % len(ring)] * page
                at += 1
            table[r, t] = slot
            slots.append(slot)
            if parents is not None:
                up = parents[offsets[-1] + i]
                mask.append((mask[up] if up >= 0 else 0) | 1 << i)
                depth.append(depth[up] + 1 if up >= 0 else 0)
            positions.append(start + (depth[i] if parents is not None else i))
        masks += mask
        offsets.append(offsets[-1] + new[b])
        if blocks is not None:
            used = -(-(cached[b] + new[b]) // page)
            blocks[b, :used] = table[r, : used * page: page] // page
    return {"offsets": np.array(offsets, np.int32), "slots": np.array(slots, np.int32),
            "positions": np.array(positions, np.int32),
            "mask": np.array(masks, np.uint64).view(np.int64) if case["tree"] else None,
            "rows": table, "table": blocks, "status": np.array([int(at > tail)], np.int32)}


def _exact_rope(case, seed):
    s = _prepare_rope(case, seed)
    t, d, half = case["tokens"], case["dim"], case["rotary"] // 2
    angle = s["cos_sin"].double()[s["positions"].long()]
    first = torch.arange(half, device="cuda")
    first, second = (first, first + half) if case["neox"] else (2 * first, 2 * first + 1)

    def head(x, w):
        x = x.double()
        y = x / torch.sqrt((x * x).sum(-1, keepdim=True) / d + 1e-6) * w.double()
        z = torch.complex(y[..., first], y[..., second]) * torch.complex(angle[:, :half], angle[:, half:])[:, None]
        y[..., first], y[..., second] = z.real, z.imag
        return y

    q, k = head(s["q"], s["q_weight"]), head(s["k"], s["k_weight"])
    if not case["store"]:
        return {"q": q, "k": k, "k_pool": None, "v_pool": None}
    keys, values = s["k_pool"].double(), s["v_pool"].double()
    real = s["slots"] >= 0
    keys[s["slots"][real].long()] = k[real]
    values[s["slots"][real].long()] = s["v"][real].double()
    return {"q": q, "k": None, "k_pool": keys, "v_pool": values}


def _exact_tree(case, seed):
    s = _prepare_tree(case, seed)
    hkv, group, d = case["hkv"], case["group"], case["dim"]
    out = torch.zeros(s["total"], hkv * group, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(s["total"], hkv * group, dtype=torch.float64, device="cuda")
    kv0, d0 = s["kv_indptr_host"], s["draft_indptr_host"]
    for b in range(len(kv0) - 1):
        lo, hi, x, y = int(kv0[b]), int(kv0[b + 1]), int(d0[b]), int(d0[b + 1])
        if x == y:
            continue
        at = torch.cat((s["kv_indices"][lo:hi], s["draft_slots"][x:y])).long()
        tree = s["tree_mask"][x:y, None] >> torch.arange(y - x, device="cuda") & 1
        open_ = torch.cat((torch.ones(y - x, hi - lo, device="cuda").bool(), tree.bool()), 1)
        if case["window"] >= 0:
            pos = torch.cat((s["kv_positions"][lo:hi], s["q_positions"][x:y]))
            open_ &= s["q_positions"][x:y, None] - pos <= case["window"]
        for h in range(hkv * group):
            k, v = s["k_pool"][at, h // group].double(), s["v_pool"][at, h // group].double()
            e = s["q"][x:y, h].double() @ k.T / math.sqrt(d)
            e = torch.where(open_, e, torch.full_like(e, -math.inf))
            if s["sinks"] is not None:
                e = torch.cat((e, s["sinks"][h].double().expand(y - x, 1)), 1)
            z = torch.logsumexp(e, 1)
            lse[x:y, h] = z
            w = torch.exp(e - z[:, None]).nan_to_num(0.0)[:, : len(at)]
            out[x:y, h] = w @ v
    return {"out": out, "lse": lse if case["lse"] else None}
