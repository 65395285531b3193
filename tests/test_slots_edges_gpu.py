"""Slot maps at the edges of the mapper's contract: entries behind the last
token, rows that cannot go on, requests that are not in order."""

import numpy as np
import pytest
import torch

from test_slots_gpu import CODES, case, check, expected, launch

pytestmark = pytest.mark.gpu


def test_no_slot_of_another_call_is_left_behind_the_last_token():
    """A mapper larger than its batch: what follows the last token holds no
    slot and no position, on a first call, after a larger call that took its
    pages, eager and replayed, in a refused call and in one of no request."""
    from akv_b200.context_drop import FreeSlotRing
    from akv_b200.context_slots import SlotMapper

    ring = FreeSlotRing(torch.arange(10, 74), device="cuda")
    rows = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    ids, none = torch.tensor([0, 1], device="cuda"), torch.zeros(0, dtype=torch.int64, device="cuda")
    lens = torch.zeros(2, dtype=torch.int64, device="cuda")
    mapper = SlotMapper(2, 16, "cuda")

    def run(new, commit=True):
        view = mapper.run(rows, ids, lens, new, ring, commit=commit)
        return view

    def tail_is_free(view, n):
        assert int((view.slots >= 0).sum()) == n and bool((view.slots[:n] >= 0).all())
        assert view.slots[n:].tolist() == [-1] * (16 - n)
        assert view.positions[n:].tolist() == [0] * (16 - n)

    few, many = torch.tensor([1, 2], device="cuda"), torch.tensor([9, 7], device="cuda")
    tail_is_free(run(few, commit=False), 3)
    tail_is_free(run(many), 16)
    lens += many
    tail_is_free(run(few), 3)
    lens += few
    tail_is_free(run(many, commit=False), 16)
    new = few.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        view = run(new, commit=False)
    for n in ([9, 7], [1, 0], [0, 0], [3, 3]):
        new.copy_(torch.tensor(n, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        tail_is_free(view, sum(n))
    ring.state[0] = ring.state[1]       # no page is free
    refused = run(few)
    assert int(refused.status) == CODES["underflow"]
    assert refused.slots.tolist() == [-1] * 16 and refused.positions[3:].tolist() == [0] * 13
    ring.state[0] -= 32
    tail_is_free(run(many, commit=False), 16)
    tail_is_free(mapper.run(rows, none, none, none, ring), 0)


def test_padded_rows_behind_the_last_token_are_not_stored():
    """The whole of the mapper's vectors with padded projections, as a step of
    a fixed size passes them: no row of the pools changes but the new tokens'."""
    from akv_b200.context_drop import FreeSlotRing
    from akv_b200.context_rope import qk_norm_rope
    from akv_b200.context_slots import SlotMapper

    ring = FreeSlotRing(torch.arange(5, 69), device="cuda")
    rows = torch.zeros(2, 64, dtype=torch.int32, device="cuda")
    ids, lens = torch.tensor([1, 0], device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda")
    mapper = SlotMapper(2, 16, "cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    pools = [torch.randn(80, 2, 64, generator=g, device="cuda").half() for _ in range(2)]
    q, k, v = (torch.randn(16, h, 64, generator=g, device="cuda").half() for h in (4, 2, 2))
    table = torch.randn(100, 64, generator=g, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    new = torch.zeros(2, dtype=torch.int64, device="cuda")

    def step():
        view = mapper.run(rows, ids, lens, new, ring)
        qk_norm_rope(q, k, view.positions, table, v=v, k_pool=pools[0], v_pool=pools[1],
                     slots=view.slots, error_flag=flag)
        return view

    def check(n):
        before = [p.clone() for p in pools]
        new.copy_(torch.tensor(n, device="cuda"))
        yield
        at = view.slots[: sum(n)].long()
        assert int(flag) == 0 and len(set(at.tolist())) == sum(n)
        assert torch.equal(pools[1][at], v[: sum(n)])
        rest = torch.ones(80, dtype=torch.bool, device="cuda")
        rest[at] = False
        for pool, old in zip(pools, before):
            assert torch.equal(pool[rest], old[rest])
        lens.add_(new)

    for n in ([1, 2], [9, 7], [1, 0], [2, 2]):
        run = check(n)
        next(run)
        view = step()
        next(run, None)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        view = step()
    for n in ([8, 7], [2, 1], [0, 0], [3, 1]):
        run = check(n)
        next(run)
        graph.replay()
        next(run, None)


@pytest.mark.parametrize("bad_rows", [[0], [1], [2], [0, 2], [0, 1, 2, 3], [3]])
@pytest.mark.parametrize("page", [4, 16])
@pytest.mark.parametrize("full", [False, True])
def test_pages_of_a_row_with_a_bad_end_are_not_lost(bad_rows, page, full):
    """The ring's head moves by the pages that rows hold, and what is left in
    the ring with what was given out is what it held before, each page once."""
    rng = np.random.default_rng(page)
    n_new = 3 * page + 1
    c = case(rng, [page + 1, 2, 3 * page + 2, 1], [n_new] * 4, page, table=True)
    if full:                                   # every entry of the ring is a free page
        assert c["tail"] - c["head"] == len(c["ring"])
    else:
        c["ring"] = np.concatenate((c["ring"][c["head"] % len(c["ring"]):],
                                    c["ring"][: c["head"] % len(c["ring"])], np.full(5, 1 << 20, np.int32)))
        c["tail"] -= c["head"]
        c["head"] = 0
    for b in bad_rows:
        r, end = c["row_ids"][b], c["cached"][b] - 1
        c["rows"][r, end] += 1
    size = len(c["ring"])
    before = [int(c["ring"][i % size]) for i in range(c["head"], c["tail"])]
    view, t = launch(c)
    assert int(view.status.item()) == CODES["page"]
    head, tail = t["ring"].state.tolist()
    left = [int(t["ring"].ring[i % size]) for i in range(head, tail)]
    slots, offsets = view.slots.tolist(), view.new_offsets.tolist()
    given = []
    for b in range(4):
        mine = slots[offsets[b]: offsets[b + 1]]
        assert len(mine) == n_new
        if b in bad_rows:
            assert mine == [-1] * n_new
        else:
            fresh = [s // page for i, s in enumerate(mine) if (c["cached"][b] + i) % page == 0]
            given += fresh
            assert t["rows"][c["row_ids"][b], c["cached"][b]: c["cached"][b] + n_new].tolist() == mine
    assert tail == c["tail"] and head - c["head"] == len(given) == int(view.totals[1])
    assert sorted(left + given) == sorted(before) and len(set(before)) == len(before)
    view, t = launch(c, commit=False)          # lent: the ring is as it was
    assert t["ring"].state.tolist() == [c["head"], c["tail"]]
    np.testing.assert_array_equal(t["ring"].ring.cpu().numpy(), c["ring"])


def test_pages_of_many_rows_with_bad_ends_are_not_lost():
    rng = np.random.default_rng(12)
    batch, page = 700, 4
    c = case(rng, rng.integers(0, 30, batch), rng.integers(0, 30, batch), page)
    ends = [b for b in range(batch) if c["cached"][b] % page and rng.random() < 0.4]
    for b in ends:
        c["rows"][c["row_ids"][b], c["cached"][b] - 1] += 1
    size = len(c["ring"])
    before = sorted(int(c["ring"][i % size]) for i in range(c["head"], c["tail"]))
    view, t = launch(c)
    assert int(view.status.item()) == CODES["page"]
    head, tail = t["ring"].state.tolist()
    ring = t["ring"].ring.cpu().numpy()
    left = [int(ring[i % size]) for i in range(head, tail)]
    rows, given = t["rows"].cpu().numpy(), []
    for b in range(batch):
        for i in range(c["cached"][b], c["cached"][b] + c["new"][b]):
            if b not in ends and i % page == 0:
                given.append(int(rows[c["row_ids"][b], i]) // page)
    assert sorted(left + given) == before and int(view.totals[1]) == len(given)


class Kept:
    """A mapper whose calls keep the offsets of the lengths."""

    def __init__(self, batch, tokens, page):
        from akv_b200.context_slots import SlotMapper

        self.mapper = SlotMapper(batch, tokens, "cuda", page_size=page)

    def run(self, *args, **kw):
        return self.mapper.run(*args, keep_offsets=True, **kw)


@pytest.mark.parametrize("what", ["row", "negative", "columns", "table"])
@pytest.mark.parametrize("tree", [False, True])
def test_kept_offsets_are_those_of_the_lengths(what, tree):
    """With keep_offsets a bad request keeps its entries, without slots, and the
    others' slots, parents and masks stay where the caller's tokens are."""
    rng = np.random.default_rng(13)
    c = case(rng, [5, 6, 7, 2], [3, 4, 5, 2], 4, tree=tree, table=True)
    bad = {**c, "row_ids": c["row_ids"].copy(), "cached": c["cached"].copy()}
    if what == "row":
        bad["row_ids"][1] = -1
    elif what == "negative":
        bad["cached"][1] = -4
    elif what == "columns":
        bad["cached"][1] = c["rows"].shape[1] - 1
    else:
        c["rows"] = bad["rows"] = np.pad(c["rows"], ((0, 0), (0, 90)), constant_values=-7)
        bad["cached"][1] = 4 * c["table"].shape[1] - 2
    view, t = launch(bad, mapper=Kept(4, 14, 4))
    assert int(view.status.item()) == CODES["request"]
    assert view.new_offsets.tolist() == [0, 3, 7, 12, 14]
    # The rules without request 1, whose tokens take no page.
    rest = {**c, "new": c["new"].copy()}
    rest["new"][1] = 0
    if tree:
        rest["parents"] = np.delete(c["parents"], [3, 4, 5, 6])
    want = expected(rest)
    keep = [i for i in range(14) if not 3 <= i < 7]
    assert view.slots[keep].tolist() == want["slots"]
    assert view.slots[3:7].tolist() == [-1] * 4
    assert view.positions[keep].tolist() == want["positions"]
    assert bool((view.positions[3:7] >= 0).all()) and bool((view.positions[3:7] < 4).all())
    if tree:
        assert view.tree_mask[keep].tolist() == want["masks"].tolist()
    np.testing.assert_array_equal(t["rows"].cpu().numpy(), want["rows"])
    # Without bad requests both ways are the same.
    check(c, *launch(c, mapper=Kept(4, 14, 4)), True)


@pytest.mark.parametrize("new", [1 << 40, -1, 65])
def test_kept_offsets_refuse_lengths_that_leave_none(new):
    rng = np.random.default_rng(14)
    c = case(rng, [5, 6, 7], [3, 3, 3], 1, tree=True, table=True)
    c["rows"] = np.pad(c["rows"], ((0, 0), (0, 90)), constant_values=-7)
    c["table"] = np.pad(c["table"], ((0, 0), (0, 90)), constant_values=-5)
    bad = {**c, "new": c["new"].copy()}
    bad["new"][1] = new
    view, t = launch(bad, capacity=9, mapper=Kept(3, 9, 1))
    assert int(view.status.item()) == CODES["request"]
    assert view.new_offsets.tolist() == [0] * 4 and view.totals.tolist() == [0, 0]
    assert view.slots.tolist() == [-1] * 9
    np.testing.assert_array_equal(t["rows"].cpu().numpy(), c["rows"])
    np.testing.assert_array_equal(t["table"].cpu().numpy(), c["table"])
    assert t["ring"].state.tolist() == [c["head"], c["tail"]]


def test_rings_of_other_types_are_refused():
    from akv_b200.context_drop import FreeSlotRing
    from akv_b200.context_slots import SlotMapper

    mapper = SlotMapper(1, 4, "cuda")
    rows = torch.zeros(2, 8, dtype=torch.int32, device="cuda")
    one = torch.ones(1, dtype=torch.int64, device="cuda")
    for field, value in (("ring", torch.arange(8, device="cuda")),
                         ("ring", torch.arange(16, dtype=torch.int32, device="cuda")[::2]),
                         ("ring", torch.arange(7, dtype=torch.int32, device="cuda")),
                         ("state", torch.zeros(2, dtype=torch.int32, device="cuda")),
                         ("state", torch.zeros(4, dtype=torch.int64, device="cuda")[::2])):
        ring = FreeSlotRing(torch.arange(8), device="cuda")
        setattr(ring, field, value)
        with pytest.raises(ValueError, match="free ring"):
            mapper.run(rows, one - 1, one - 1, one, ring)


@pytest.mark.parametrize("batch", [1, 3, 90])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("spare", [1, 5, 1023, 40000])
def test_every_entry_behind_the_last_token_of_a_large_mapper(batch, tree, spare):
    from akv_b200.context_slots import SlotMapper

    rng = np.random.default_rng(spare + batch)
    c = case(rng, rng.integers(0, 40, batch), rng.integers(1, 9, batch), 4, tree=tree, table=True)
    total = int(c["new"].sum())
    mapper = SlotMapper(batch + 2, total + spare, "cuda", page_size=4)
    mapper._slots.copy_(torch.arange(total + spare))
    mapper._positions.copy_(torch.arange(total + spare) + 3)
    view, t = launch(c, mapper=mapper, capacity=total + spare)
    check(c, view, t, True)
    assert bool((view.slots[total:] == -1).all()) and bool((view.positions[total:] == 0).all())
