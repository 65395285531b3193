"""Taking a verified tree into the rows: draft, store, accept one root path per
request, move its K/V, go on.  Everything here is a copy of stored values or an
integer, so all comparisons are exact."""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

HQ, HKV, D = 4, 2, 64


@pytest.mark.parametrize("page", [1, 4, 16])
@pytest.mark.parametrize("tree", [True, False])
def test_accepted_paths_over_many_steps(page, tree):
    from akv_b200.context_drop import FreeSlotRing
    from akv_b200.context_rope import qk_norm_rope
    from akv_b200.context_slots import SlotMapper

    rng = np.random.default_rng(page + 100 * tree)
    g = torch.Generator(device="cuda").manual_seed(page)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda").bfloat16()  # noqa: E731
    batch, room, pages = 5, 40, 1000 if page == 1 else 200
    ids = rng.permutation(pages) + 1
    ring = FreeSlotRing(torch.from_numpy(ids.astype(np.int32)), device="cuda")
    rows = torch.zeros(batch + 1, 512, dtype=torch.int32, device="cuda")
    row_ids = torch.from_numpy(rng.permutation(batch + 1)[:batch]).cuda()
    raw = torch.zeros(batch, dtype=torch.int64, device="cuda")
    # Tokens dropped before leave the positions behind the columns.
    behind = torch.zeros(batch, dtype=torch.int64, device="cuda")
    table = torch.randn(600, D, generator=g, device="cuda")
    layers = [[rand((pages + 1) * page, HKV, D) for _ in range(2)] for _ in range(2)]
    mapper = SlotMapper(batch, batch * room, "cuda", page_size=page)
    want = [[[] for _ in range(batch)] for _ in layers]     # each request's K and V, column by column
    starts = lambda n: np.concatenate(([0], np.cumsum(n)))  # noqa: E731

    def store(view, n):
        """Every layer's new tokens; returns what a store of each alone holds."""
        kv = []
        for kp, vp in layers:
            q, k, v = rand(n, HQ, D), rand(n, HKV, D), rand(n, HKV, D)
            qk_norm_rope(q, k, view.positions, table, v=v, k_pool=kp, v_pool=vp, slots=view.slots)
            kv.append((k, v))
        return kv

    def rotated(k, positions):
        return qk_norm_rope(k.new_zeros(len(k), HQ, D), k, positions, table)[1]

    # A prompt chunk takes its pages at once.
    new = rng.integers(0, 30, batch)
    view = mapper.run(rows, row_ids, raw, torch.from_numpy(new).cuda(), ring)
    view.check()
    for layer, (k, v) in enumerate(store(view, int(new.sum()))):
        k = rotated(k, view.positions[: len(k)].clone())
        for b, (x, y) in enumerate(zip(starts(new)[:-1], starts(new)[1:])):
            want[layer][b] += [(k[t], v[t]) for t in range(x, y)]
    raw += torch.from_numpy(new).cuda()
    behind.copy_(torch.from_numpy(rng.integers(0, new + 1)))

    for _ in range(6):
        new = rng.integers(0, 17, batch)
        at = starts(new)
        parents = np.concatenate([[rng.integers(max(-1, i - 4), i) if tree else i - 1 for i in range(n)]
                                  for n in new] + [[]]).astype(np.int32)
        up = torch.zeros(batch * room, dtype=torch.int32, device="cuda")
        up[: len(parents)] = torch.from_numpy(parents).cuda()
        view = mapper.run(rows, row_ids, raw, torch.from_numpy(new).cuda(), ring,
                          next_positions=raw - behind, parents=up, commit=False, keep_offsets=True)
        view.check()
        kv = store(view, int(new.sum()))
        # Verified: one path from a root per request, or none.
        nodes, taken = [], []
        for b, n in enumerate(new):
            path, node = [], int(rng.integers(-1, n)) if n else -1
            while node >= 0:
                path.insert(0, at[b] + node)
                node = int(parents[at[b] + node])
            nodes += path
            taken.append(len(path))
        nodes, taken = torch.tensor(nodes, dtype=torch.int64, device="cuda"), torch.tensor(taken, device="cuda")
        # The accepted nodes' slots are read before the mapper's next call.
        source = view.slots[nodes].long()
        first = (raw - behind).tolist()
        got = mapper.run(rows, row_ids, raw, taken, ring, next_positions=raw - behind, commit=True)
        got.check()
        target = got.slots[: len(nodes)].long()
        for kp, vp in layers:
            kp[target], vp[target] = kp[source], vp[source]
        raw += taken
        # What the rows hold now: the accepted nodes, rotated at the positions of their columns.
        ends = starts(taken.tolist())
        position = torch.tensor([first[b] + i for b, n in enumerate(taken.tolist()) for i in range(n)],
                                dtype=torch.int64, device="cuda")
        for layer, (k, v) in enumerate(kv):
            k, v = rotated(k[nodes].contiguous(), position), v[nodes]
            for b in range(batch):
                want[layer][b] += [(k[t], v[t]) for t in range(ends[b], ends[b + 1])]
        held = []
        for b in range(batch):
            slots = rows[row_ids[b], : int(raw[b])].long()
            held += slots.tolist()
            assert bool((slots % page == torch.arange(len(slots), device="cuda") % page).all())
            for layer, (kp, vp) in enumerate(layers):
                assert len(slots) == len(want[layer][b])
                for pool, kind in ((kp, 0), (vp, 1)):
                    if len(slots):
                        assert torch.equal(pool[slots], torch.stack([x[kind] for x in want[layer][b]]))
        assert len(set(held)) == len(held)
        free = set(ring.snapshot().tolist())
        mine = {s // page for s in held}
        assert not free & mine and sorted(free | mine) == sorted(ids.tolist())
