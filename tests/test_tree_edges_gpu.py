"""Tree attention at its edges: infinities and NaN in long windows and in many
items of one CTA, graphs replayed on other plans, small weights in fp16."""

import numpy as np
import pytest
import torch

from test_tree_gpu import attention, compare, exact, launch, make

pytestmark = pytest.mark.gpu


def seen_keys(c, b):
    """[tokens, cached + drafted keys] of request b."""
    lo, hi, x, y = (int(v) for v in (*c["kv"][b: b + 2], *c["dr"][b: b + 2]))
    bits = (c["mask"][x:y, None] >> torch.arange(y - x, device="cuda")) & 1
    seen = torch.cat((torch.ones(y - x, hi - lo, dtype=torch.bool, device="cuda"), bits.bool()), 1)
    if c["window"] >= 0:
        at = torch.cat((c["kpos"][lo:hi], c["qpos"][x:y]))
        seen &= c["qpos"][x:y, None] - at <= c["window"]
    return seen


def check_bad_values(c, places, ctas=None):
    """V elements ``places`` [(request, key, head, dim, value)] that are not
    finite change those elements of the rows that see them, and nothing else:
    all others are what zeros in their place give, bit for bit."""
    attn = attention(c, ctas)
    zero, bad = c["v"].clone(), c["v"].clone()
    special = torch.zeros(len(c["q"]), c["hkv"], c["d"], dtype=torch.float64, device="cuda")
    views = {b: seen_keys(c, b) for b in {p[0] for p in places}}
    for b, key, head, dim, value in places:
        lo, hi, x, y = (int(v) for v in (*c["kv"][b: b + 2], *c["dr"][b: b + 2]))
        slot = int(c["indices"][lo + key] if key < hi - lo else c["draft"][x + key - (hi - lo)])
        zero[slot, head, dim], bad[slot, head, dim] = 0, value
        rows = views[b][:, key].nonzero().flatten() + x
        special[rows, head, dim] += value
    want, want_lse = launch({**c, "v": zero}, attn, return_lse=True)
    out, lse = launch({**c, "v": bad}, attn, return_lse=True)
    assert int(attn.error_flag) == 0
    special = special.repeat_interleave(c["group"], 1)
    hit = special != 0
    assert bool(hit.any()) and torch.equal(lse, want_lse)
    assert torch.equal(out[~hit], want[~hit])
    got, sure = out[hit].double(), special[hit]
    assert torch.equal(got.isnan(), sure.isnan())
    assert torch.equal(got.nan_to_num(0.5), sure.nan_to_num(0.5))


BAD = [float("nan"), float("inf"), -float("inf")]


def draws(c, rng, n):
    """n bad elements at keys that some row sees."""
    out = []
    while len(out) < n:
        b = int(rng.integers(len(c["kv"]) - 1))
        keys = seen_keys(c, b).any(0).nonzero().flatten()
        if len(keys):
            out.append((b, int(keys[int(rng.integers(len(keys)))]), int(rng.integers(c["hkv"])),
                        int(rng.integers(c["d"])), BAD[int(rng.integers(3))]))
    return out


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_bad_draft_element_behind_a_long_window_leaves_the_others(d, dtype):
    """30,000 keys in a large window, all of it and a second request one CTA's work."""
    c = make([30000, 700], [16, 9], 2, 8, d, dtype, seed=21, window=100000)
    for value in BAD:
        check_bad_values(c, [(0, 30000 + 3, 1, 5, value)], ctas=1)
        check_bad_values(c, [(0, 30000 + 3, 1, 5, value)])


@pytest.mark.parametrize("ctas", [1, 5])
@pytest.mark.parametrize("d", [64, 128])
def test_bad_elements_all_over_a_long_window(d, ctas):
    """More tiles than an item's word has bits, hidden keys in every tile."""
    c = make([20000, 300, 9000], [16, 64, 3], 2, 5, d, torch.bfloat16, seed=22, window=30000)
    g = torch.Generator(device="cuda").manual_seed(1)
    for b in range(3):  # positions in no order: every tile has hidden keys
        part = slice(int(c["kv"][b]), int(c["kv"][b + 1]))
        c["kpos"][part] = c["kpos"][part][torch.randperm(int(c["kv"][b + 1] - c["kv"][b]), generator=g,
                                                         device="cuda")]
    rng = np.random.default_rng(23)
    check_bad_values(c, draws(c, rng, 40), ctas)


@pytest.mark.parametrize("window", [-1, 60])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 8, 16])
def test_bad_elements_in_many_short_items_of_one_cta(d, window, group):
    rng = np.random.default_rng(24)
    c = make(rng.integers(0, 200, 40), rng.integers(1, 20, 40), 3, group, d, torch.bfloat16, seed=25,
             window=window)
    # Without a window an infinity that all rows of a tile see takes the ordinary way, as its
    # product with a weight above 0; the weights of this test are.
    for ctas in (1, 3, None):
        check_bad_values(c, draws(c, rng, 30), ctas)


@pytest.mark.parametrize("d", [64, 128])
def test_a_request_of_nothing_but_nan_leaves_the_others(d):
    """Every V of a long request is NaN, with hidden keys in every tile."""
    c = make([12000, 40, 300], [16, 8, 33], 2, 8, d, torch.bfloat16, seed=26, window=15000)
    part = slice(0, 12000)
    g = torch.Generator(device="cuda").manual_seed(2)
    c["kpos"][part] = c["kpos"][part][torch.randperm(12000, generator=g, device="cuda")]
    v = c["v"].clone()
    v[c["indices"][part].long()] = float("nan")
    for ctas in (1, None):
        attn = attention(c, ctas)
        want, want_lse = launch(c, attn, return_lse=True)
        out, lse = launch({**c, "v": v}, attn, return_lse=True)
        assert int(attn.error_flag) == 0 and torch.equal(lse, want_lse)
        assert bool(out[:16].isnan().all()) and torch.equal(out[16:], want[16:])


def test_work_behind_a_merge_that_joins_nothing_waits_for_its_pieces():
    """A replay on a plan whose every merge lies past the call's tokens: what
    follows in the stream sees the error bits of the pieces' kernel."""
    c = make([4000], [8], 2, 8, 64, torch.bfloat16, seed=27)
    attn = attention(c, 8)
    out = torch.empty_like(c["q"])
    launch(c, attn, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch(c, attn, out=out)
    attn.plan([0, 4000], [0, 64])       # 64 tokens where the call has 8
    for _ in range(20):
        attn.error_flag.zero_()
        graph.replay()
        seen = attn.error_flag.clone()
        assert int(seen) == 4
    attn.plan(c["kv"], c["dr"])
    attn.error_flag.zero_()
    graph.replay()
    assert int(attn.error_flag) == 0
    compare(c, out, launch(c, attn, return_lse=True)[1])


def grown(c, cached, new, room_keys, room_tokens):
    """The same pools under other lengths, vectors copied into ones of a fixed size."""
    def wide(t, n):
        out = t.new_zeros((n, *t.shape[1:]))
        out[: len(t)] = t
        return out

    keys, total = int(sum(cached)), int(sum(new))
    x = make(cached, new, c["hkv"], c["group"], c["d"], c["dtype"], seed=keys + total, sinks=True,
             window=c["window"], extra_slots=len(c["k"]) - keys - total)
    return x, {n: wide(x[n], room_tokens if n in ("q", "draft", "mask", "qpos") else room_keys)
               for n in ("q", "draft", "mask", "qpos", "indices", "kpos")}


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("window", [-1, 900])
def test_one_graph_over_growing_caches_and_other_batches(d, window):
    """Captured once and replayed on plans of other lengths, batches, CTA and
    merge counts, an empty one among them: always what an eager run gives."""
    rng = np.random.default_rng(31)
    room_keys, room_tokens, batch = 12000, 120, 12
    lens = rng.integers(0, 900, batch)
    c = make(lens, [8] * batch, 2, 8, d, torch.bfloat16, seed=32, window=window, sinks=True,
             extra_slots=16000)
    from akv_b200.context_tree import TreeAttention

    attn = TreeAttention(16, 2, d, batch, "cuda", ctas=23).plan(c["kv"], c["dr"])
    fixed = grown(c, lens, [8] * batch, room_keys, room_tokens)[1]
    buffers = {n: t.clone() for n, t in fixed.items()}
    pools = dict(k=torch.zeros_like(c["k"]), v=torch.zeros_like(c["v"]))
    sinks = torch.zeros(16, device="cuda")
    out = torch.empty(room_tokens, 16, d, dtype=torch.bfloat16, device="cuda")

    def run():
        return attn.run(buffers["q"], pools["k"], pools["v"], buffers["indices"], buffers["draft"],
                        buffers["mask"], sinks=sinks, window=window, q_positions=buffers["qpos"],
                        kv_positions=buffers["kpos"], out=out)

    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run()
    steps, counts = [], set()
    for _ in range(20):                                     # a cache that grows
        lens = lens + rng.integers(0, 6, batch)
        steps.append((lens.copy(), rng.integers(1, 10, batch)))
    steps += [([5000], [64]), ([], []), ([0, 3], [1, 0]), ([40] * 12, [1] * 12), ([9000, 70], [3, 64]),
              ([room_keys], [1]), ([1, 2], [64, 56])]
    for cached, new in steps:
        x, vectors = grown(c, cached, new, room_keys, room_tokens)
        for n, t in vectors.items():
            buffers[n].copy_(t)
        pools["k"].copy_(x["k"])
        pools["v"].copy_(x["v"])
        sinks.copy_(x["sinks"])
        attn.plan(x["kv"], x["dr"])
        counts.add((attn.n_ctas, attn.n_merges))
        out.fill_(7)
        graph.replay()
        total = int(sum(new))
        assert int(attn.error_flag) == 0 and bool((out[total:] == 7).all())
        fresh = TreeAttention(16, 2, d, batch, "cuda", ctas=23).plan(x["kv"], x["dr"])
        want = launch(x, fresh)
        assert torch.equal(out[:total], want)
    assert len({n for n, _ in counts}) > 2 and len({m for _, m in counts}) > 2
    for cached, new in (([room_keys, 1], [1, 1]), ([3, 3], [64, 57])):    # a key, a token too many
        kv, dr = (np.concatenate(([0], np.cumsum(n))) for n in (cached, new))
        attn.plan(kv, dr)
        graph.replay()
        with pytest.raises(RuntimeError, match="tensors hold"):
            attn.check()


def test_a_graph_captured_on_an_empty_plan():
    c = make([300, 20], [5, 9], 2, 8, 64, torch.bfloat16, seed=33)
    attn = attention(c)
    want = launch(c, attention(c))
    out = torch.zeros_like(want)
    launch(c, attn, out=out)
    attn.plan([0], [0])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch(c, attn, out=out)
    out.zero_()
    graph.replay()
    assert not bool(out.any())
    attn.plan(c["kv"], c["dr"])
    graph.replay()
    assert torch.equal(out, want) and int(attn.error_flag) == 0


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctas", [1, None])
def test_many_small_weights_in_fp16(d, ctas):
    """One key of score 0 with V 0 and 150,000 of weight 2^-26 with V 1: half of
    fp16's smallest P, but 0.2 % of the sum.  Tolerance as compare() without its
    term for subnormal P: a P of at least 2^-14 (base 2^7 up: weights of 2^-21
    and more) keeps 11 bits, one below is off by at most 2^-25 in those units,
    2^-32 of the row's largest weight, per key."""
    n = 150000
    c = make([n], [3], 1, 8, d, torch.float16, seed=41)
    c["mask"].zero_()                       # cached keys alone
    c["q"].zero_()
    c["q"][:, :, 0] = 1.0
    c["k"].zero_()
    c["v"].fill_(1.0)
    # score = q0 k0 / sqrt(d) + q1 k1 / sqrt(d): 26 ln 2 below, to fp16's steps
    c["k"][:, :, 0] = -26 * np.log(2) * d**0.5
    at = int(c["indices"][n // 3])
    c["k"][at], c["v"][at] = 0.0, 0.0
    out, lse = launch(c, attention(c, ctas), return_lse=True)
    want, want_lse, mean, size = exact(c)
    assert float(want.max()) > 1e-3
    u = 2.0**-11
    e32 = (d + 4) * 2.0**-23 * size + 2.0**-21 + n * 2.0**-24
    bound = u * want.abs() + (u + 2 * e32[..., None]) * mean + n * 2.0**-32 + 2.0**-24
    assert bool(((out.double() - want).abs() <= bound * (1 + u)).all())
