"""Slot maps of new tokens (C ABI akv_map_slots): every output is an integer
and must equal a plain statement of the rules, token by token."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

CODES = dict(underflow=1, capacity=2, request=4, page=8, parent=16)


def case(rng, cached, new, page, *, tree=False, table=False, extra_columns=0):
    cached, new = np.asarray(cached, np.int64), np.asarray(new, np.int64)
    batch = len(cached)
    old = -(-cached // page)
    used = -(-(cached + new) // page)
    lent = int((used - old).sum())
    ids = rng.permutation(int(old.sum()) + lent + 9).astype(np.int32) + 1
    rows = batch + 2
    row_ids = rng.permutation(rows)[:batch].astype(np.int64)
    table_rows = np.full((rows, int((cached + new).max()) + 3 + extra_columns), -7, np.int32)
    at = 0
    for b in range(batch):
        for t in range(cached[b]):
            if t % page == 0:
                at += 1
            table_rows[row_ids[b], t] = ids[at - 1] * page + t % page
    free = ids[at:]
    head = int(rng.integers(0, 3 * len(free)))
    ring = np.empty_like(free)
    ring[(head + np.arange(len(free))) % len(free)] = free
    parents = None
    if tree:
        parents = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(n)] for n in new]
                                 + [[]]).astype(np.int32)
    return dict(page=page, row_ids=row_ids, cached=cached, new=new, rows=table_rows, ring=ring,
                head=head, tail=head + len(free), parents=parents,
                next=rng.integers(0, 1 << 20, batch).astype(np.int32),
                table=np.full((batch, int(used.max()) + 2), -5, np.int32) if table else None)


def expected(c):
    """The rules, one token at a time."""
    page, rows = c["page"], c["rows"].copy()
    table = None if c["table"] is None else c["table"].copy()
    at, offsets, slots, positions, masks = c["head"], [0], [], [], []
    for b, r in enumerate(c["row_ids"]):
        mask = []
        for i in range(c["new"][b]):
            t = c["cached"][b] + i
            if t % page:
                slot = rows[r, t - 1] + 1
            else:
                slot = c["ring"][at % len(c["ring"])] * page
                at += 1
            rows[r, t] = slot
            slots.append(slot)
            step = i
            if c["parents"] is not None:
                up = c["parents"][offsets[-1] + i]
                mask.append(1 << i | (mask[up] if up >= 0 else 0))
                step = bin(mask[-1]).count("1") - 1
            positions.append(c["next"][b] + step)
        masks += mask
        offsets.append(offsets[-1] + c["new"][b])
        if table is not None:
            for g in range(-(-(c["cached"][b] + c["new"][b]) // page)):
                table[b, g] = rows[r, g * page] // page
    return dict(offsets=offsets, slots=slots, positions=positions, rows=rows, table=table,
                masks=np.array(masks, np.uint64).view(np.int64), pages=at - c["head"])


def launch(c, *, commit=True, capacity=None, mapper=None, lens64=True, dev="cuda", lay=lambda x: x):
    from akv_b200.context_drop import FreeSlotRing
    from akv_b200.context_slots import SlotMapper

    total = int(c["new"].sum())
    capacity = total if capacity is None else capacity
    mapper = mapper or SlotMapper(len(c["row_ids"]), capacity, dev, page_size=c["page"])
    ring = FreeSlotRing([], capacity=len(c["ring"]), device=dev)
    ring.ring.copy_(torch.from_numpy(c["ring"]))
    ring.state.copy_(torch.tensor([c["head"], c["tail"]]))
    index = torch.int64 if lens64 else torch.int32
    t = dict(rows=lay(torch.from_numpy(c["rows"]).to(dev)),
             row_ids=torch.from_numpy(c["row_ids"]).to(dev, index),
             cached=torch.from_numpy(c["cached"]).to(dev, index),
             new=torch.from_numpy(c["new"]).to(dev, index),
             next=torch.from_numpy(c["next"]).to(dev), ring=ring)
    parents = c["parents"]
    if parents is not None:
        parents = np.concatenate((parents, np.zeros(max(0, capacity - len(parents)), np.int32)))
        parents = torch.from_numpy(parents).to(dev)
    t["table"] = None if c["table"] is None else lay(torch.from_numpy(c["table"]).to(dev))
    view = mapper.run(t["rows"], t["row_ids"], t["cached"], t["new"], ring,
                      next_positions=t["next"], parents=parents, block_table=t["table"],
                      commit=commit)
    return view, t


def check(c, view, t, commit):
    want = expected(c)
    n = len(want["slots"])
    assert int(view.status.item()) == 0
    assert view.new_offsets.tolist() == want["offsets"]
    assert view.slots[:n].tolist() == want["slots"]
    assert view.positions[:n].tolist() == want["positions"]
    assert view.totals.tolist() == [n, want["pages"]]
    np.testing.assert_array_equal(t["rows"].cpu().numpy(), want["rows"])
    if c["parents"] is not None:
        np.testing.assert_array_equal(view.tree_mask[:n].cpu().numpy(), want["masks"])
    if c["table"] is not None:
        np.testing.assert_array_equal(t["table"].cpu().numpy(), want["table"])
    head = c["head"] + (want["pages"] if commit else 0)
    assert t["ring"].state.tolist() == [head, c["tail"]]


@pytest.mark.parametrize("page", [1, 4, 16, 128])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("table", [False, True])
def test_slot_map_matches_the_rules(page, tree, table):
    rng = np.random.default_rng(page * 4 + tree * 2 + table)
    # empty rows, no new tokens, whole pages, one token short of a page, one past
    cached = [0, 0, 1, page, page - 1, page + 1, 777, 5 * page]
    new = [0, 1, 64, page if page <= 64 else 64, 1, 2, 33, 0]
    c = case(rng, cached, new, page, tree=tree, table=table)
    for commit in (True, False):
        view, t = launch(c, commit=commit, lens64=commit)
        check(c, view, t, commit)


@pytest.mark.parametrize("batch", [1, 255, 257, 900])
def test_slot_map_batches(batch):
    rng = np.random.default_rng(batch)
    c = case(rng, rng.integers(0, 90, batch), rng.integers(0, 65, batch), 16, tree=True, table=True)
    check(c, *launch(c), True)


@pytest.mark.parametrize("offset", [0, 1, 2, 4])
@pytest.mark.parametrize("pad", [0, 1, 3, 4])
def test_long_block_tables_at_any_alignment(offset, pad):
    """Pages of one slot: rows that may be copied 16 bytes at a time and rows
    that may not, some of each in one call."""
    rng = np.random.default_rng(8 * offset + pad)
    c = case(rng, [4096, 4099, 0, 3, 5000, 1022, 12288], [1, 9, 5, 2, 64, 0, 33], 1, tree=True, table=True)

    def lay(x):
        n, m = x.shape
        wide = torch.full((n, m + offset + pad), -7, dtype=x.dtype, device=x.device)
        wide[:, offset: offset + m] = x
        return wide[:, offset: offset + m]

    view, t = launch(c, lay=lay)
    check(c, view, t, True)
    for x in (t["rows"], t["table"]):
        edge = torch.as_strided(x, (x.shape[0], offset), (x.stride(0), 1),
                                x.storage_offset() - offset)
        assert bool((edge == -7).all())


def test_slot_map_prompt_chunks():
    rng = np.random.default_rng(5)
    c = case(rng, [0, 5000, 17], [9000, 1, 4095], 64, table=True)
    check(c, *launch(c), True)


def test_outputs_behind_the_last_token_stay():
    rng = np.random.default_rng(6)
    c = case(rng, [3, 9], [2, 4], 4, tree=True)
    from akv_b200.context_slots import SlotMapper

    mapper = SlotMapper(5, 40, "cuda", page_size=4)
    for b in (mapper._slots, mapper._positions, mapper._mask):
        b.fill_(-99)
    view, t = launch(c, mapper=mapper, capacity=40)
    check(c, view, t, True)
    for b in (view.slots, view.positions, view.tree_mask):
        assert bool((b[6:] == -99).all())


def test_deep_and_flat_trees():
    rng = np.random.default_rng(7)
    c = case(rng, [10, 10, 10], [64, 64, 64], 1, tree=True)
    c["parents"] = np.concatenate((np.arange(64) - 1, np.r_[-1, np.zeros(63)],
                                   np.full(64, -1))).astype(np.int32)
    check(c, *launch(c), True)


def test_lent_pages_come_again_and_taken_pages_do_not():
    rng = np.random.default_rng(8)
    c = case(rng, [5, 6], [8, 8], 4)
    view, t = launch(c, commit=False)
    first = view.slots.tolist()
    view, t2 = launch({**c, "rows": t["rows"].cpu().numpy()}, commit=False)
    assert view.slots.tolist() == first


def test_refused_calls_leave_rows_ring_and_table():
    rng = np.random.default_rng(9)
    c = case(rng, [5, 6], [8, 8], 4, table=True)
    short = {**c, "tail": c["head"] + 1}
    view, t = launch(short)
    assert int(view.status.item()) == CODES["underflow"]
    assert view.slots.tolist() == [-1] * 16 and view.totals.tolist() == [16, 0]
    np.testing.assert_array_equal(t["rows"].cpu().numpy(), c["rows"])
    np.testing.assert_array_equal(t["table"].cpu().numpy(), c["table"])
    assert t["ring"].state.tolist() == [short["head"], short["tail"]]
    view, t = launch(c, capacity=15)
    assert int(view.status.item()) == CODES["capacity"]
    assert view.new_offsets.tolist() == [0, 0, 0] and view.totals.tolist() == [0, 0]
    assert view.slots.tolist() == [-1] * 15
    np.testing.assert_array_equal(t["rows"].cpu().numpy(), c["rows"])
    with pytest.raises(RuntimeError, match="max_new_tokens"):
        view.check()


@pytest.mark.parametrize("what", ["row", "negative", "length", "tree", "table"])
def test_a_bad_request_is_one_without_new_tokens(what):
    rng = np.random.default_rng(10)
    c = case(rng, [5, 6, 7], [3, 3, 3], 1, tree=True, table=True)
    bad = {**c, "row_ids": c["row_ids"].copy(), "cached": c["cached"].copy(), "new": c["new"].copy(),
           "rows": c["rows"]}
    if what == "row":
        bad["row_ids"][1] = len(c["rows"])
    elif what == "negative":
        bad["cached"][1] = -4
    elif what == "length":
        bad["new"][1] = 1 << 40
    elif what == "tree":
        bad["new"][1] = 65
        c["rows"] = bad["rows"] = np.pad(c["rows"], ((0, 0), (0, 90)), constant_values=-7)
        c["table"] = bad["table"] = np.pad(c["table"], ((0, 0), (0, 90)), constant_values=-5)
    else:
        bad["cached"][1] = c["table"].shape[1] - 2
        c["rows"] = bad["rows"] = np.pad(c["rows"], ((0, 0), (0, 90)), constant_values=-7)
    view, t = launch(bad, capacity=9)
    assert int(view.status.item()) == CODES["request"]
    good = {**c, "new": c["new"].copy()}
    good["new"][1] = 0
    good["parents"] = c["parents"][:6]
    want = expected(good)
    assert view.new_offsets.tolist() == want["offsets"]
    assert view.slots[:6].tolist() == want["slots"]
    np.testing.assert_array_equal(t["rows"].cpu().numpy(), want["rows"])


def test_bad_page_and_bad_parent():
    rng = np.random.default_rng(11)
    c = case(rng, [5, 6], [3, 3], 4, tree=True, table=True)
    c["rows"][c["row_ids"][0], 4] += 1            # the last slot off its place in the page
    c["parents"][:] = [-1, 5, 0, -1, 0, 2]        # token 1's parent comes after it; token 5's is itself
    view, t = launch(c)
    assert int(view.status.item()) == CODES["page"] | CODES["parent"]
    assert view.slots[:3].tolist() == [-1] * 3 and view.slots[3:].min() >= 0
    assert view.tree_mask.tolist() == [1, 2, 5, 1, 3, 4]
    np.testing.assert_array_equal(t["rows"][c["row_ids"][0]].cpu().numpy(), c["rows"][c["row_ids"][0]])
    assert bool((t["table"][0] == -5).all())
    view, t = launch(case(rng, [5], [3], 4))       # a status is the call's own
    assert int(view.status.item()) == 0


def test_captured_calls_replay_on_grown_lengths():
    from akv_b200.context_drop import FreeSlotRing
    from akv_b200.context_slots import SlotMapper

    dev = torch.device("cuda")
    rows = torch.zeros(3, 64, dtype=torch.int32, device=dev)
    ring = FreeSlotRing(torch.arange(1, 33), device=dev)
    ids = torch.tensor([2, 0], device=dev)
    cached = torch.zeros(2, dtype=torch.int64, device=dev)
    new = torch.tensor([3, 2], device=dev)
    mapper = SlotMapper(2, 8, dev, page_size=4)
    run = lambda: mapper.run(rows, ids, cached, new, ring)  # noqa: E731
    run()
    torch.cuda.synchronize()
    rows.zero_()
    ring.state.copy_(torch.tensor([0, 32]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        view = run()
    for _ in range(3):
        graph.replay()
        cached += new
    torch.cuda.synchronize()
    assert int(view.status.item()) == 0
    pages = lambda r, n: [r[i] // 4 for i in range(0, n, 4)]  # noqa: E731
    a, b = rows[2].tolist(), rows[0].tolist()
    assert [s % 4 for s in a[:9]] == [t % 4 for t in range(9)]
    assert sorted(pages(a, 9) + pages(b, 6)) == [1, 2, 3, 4, 5]
    assert ring.state.tolist() == [5, 32]


def test_wrapper_refusals():
    from akv_b200.context_drop import FreeSlotRing
    from akv_b200.context_slots import SlotMapper

    for page in (2, 3, 256, 0):
        with pytest.raises(ValueError):
            SlotMapper(1, 1, "cuda", page_size=page)
    mapper = SlotMapper(2, 4, "cuda")
    ring = FreeSlotRing(torch.arange(8), device="cuda")
    rows = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    two = torch.zeros(2, dtype=torch.int64, device="cuda")
    ok = dict(req_to_token=rows, row_ids=two, raw_lens=two, new_lens=two, ring=ring)
    for change in (dict(req_to_token=rows.long()), dict(req_to_token=rows.t()), dict(raw_lens=two[:1]),
                   dict(new_lens=two.float()), dict(raw_lens=two.cpu()),
                   dict(parents=torch.zeros(3, dtype=torch.int32, device="cuda")),
                   dict(block_table=rows[:1]), dict(block_table=rows.long()),
                   dict(row_ids=torch.zeros(3, dtype=torch.int64, device="cuda"))):
        with pytest.raises(ValueError):
            mapper.run(**{**ok, **change})
    none = two[:0]
    view = mapper.run(rows, none, none, none, ring)
    assert view.new_offsets.tolist() == [0] and view.totals.tolist() == [0, 0]
