"""Attention of drafted token trees (C ABI akv_tree_attention), against the
definition in 64 bits.

Tolerance, with u = eps(type) / 2, A = sum_j p_j |v_j| / l and S the row's
largest sum_d |q_d k_d| * scale:
  * the output is rounded once:                         u |want|
  * each p is rounded to the type before P.V:            u A
  * a score is a dot product of D terms in fp32: off by at most (D + 4) 2^-23 S,
    which is p's relative error, in the numerator and in l;
  * exponentials to 2 ulp and sums of `keys` terms in fp32: 2^-21 + keys 2^-24,
    in the numerator and in l.
"""

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def masks(parents, indptr):
    out = np.zeros(len(parents), np.uint64)
    depth = np.zeros(len(parents), np.int64)
    for b in range(len(indptr) - 1):
        for i in range(indptr[b + 1] - indptr[b]):
            up = parents[indptr[b] + i]
            at = indptr[b] + i
            out[at] = np.uint64(1) << np.uint64(i)
            if up >= 0:
                out[at] |= out[indptr[b] + up]
                depth[at] = depth[indptr[b] + up] + 1
    return out.view(np.int64), depth


def make(cached, new, hkv, group, d, dtype, *, seed=0, sinks=False, window=-1, scale=1.5,
         extra_slots=9):
    rng = np.random.default_rng(seed)
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    kv, dr = (np.concatenate(([0], np.cumsum(x))).astype(np.int64) for x in (cached, new))
    keys, total = int(kv[-1]), int(dr[-1])
    slots = keys + total + extra_slots
    place = torch.from_numpy(rng.permutation(slots).astype(np.int32)).cuda()
    parents = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(n)] for n in new]
                             + [[]]).astype(np.int64)
    mask, depth = masks(parents, dr)
    pos = np.concatenate([np.cumsum(rng.integers(1, 4, n)) for n in cached] + [[]]).astype(np.int32)
    last = [int(pos[kv[b + 1] - 1]) if cached[b] else 0 for b in range(len(cached))]
    qpos = (np.repeat(np.array(last, np.int64), new) + 1 + depth).astype(np.int32)
    return dict(q=(scale * rand(total, hkv * group, d)).to(dtype), k=rand(slots, hkv, d).to(dtype),
                v=rand(slots, hkv, d).to(dtype), kv=kv, dr=dr, indices=place[:keys],
                draft=place[keys: keys + total], mask=torch.from_numpy(mask).cuda(), window=window,
                qpos=torch.from_numpy(qpos).cuda(), kpos=torch.from_numpy(pos).cuda(),
                sinks=rand(hkv * group) if sinks else None, hkv=hkv, group=group, d=d, dtype=dtype)


def exact(c):
    """(out, lse, A, S) in 64 bits; masked keys take no part at all."""
    hkv, group, d = c["hkv"], c["group"], c["d"]
    total = c["q"].shape[0]
    out = torch.zeros(total, hkv * group, d, dtype=torch.float64, device="cuda")
    mean = torch.zeros_like(out)
    lse = torch.full((total, hkv * group), -np.inf, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(lse)
    for b in range(len(c["kv"]) - 1):
        lo, hi, x, y = (int(v) for v in (*c["kv"][b: b + 2], *c["dr"][b: b + 2]))
        pad = c["draft"][x:y] < 0
        at = torch.cat((c["indices"][lo:hi], c["draft"][x:y].clamp(min=0))).long()
        k, v = c["k"][at].double(), c["v"][at].double()
        k[hi - lo:][pad], v[hi - lo:][pad] = 0, 0
        for i in range(x, y):
            bits = (c["mask"][i] >> torch.arange(y - x, device="cuda")) & 1
            seen = torch.cat((torch.ones(hi - lo, device="cuda"), bits)).bool()
            if c["window"] >= 0:
                p = torch.cat((c["kpos"][lo:hi], c["qpos"][x:y]))
                seen &= c["qpos"][i] - p <= c["window"]
            if not bool(seen.any()):
                if c["sinks"] is not None:
                    lse[i] = c["sinks"].double()
                continue
            kk, vv = k[seen], v[seen]
            qq = c["q"][i].double().view(hkv, group, d)
            s = torch.einsum("hgd,nhd->hgn", qq, kk) * d**-0.5
            size[i] = (torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()) * d**-0.5).amax(-1).view(-1)
            z = torch.logsumexp(s, -1)
            if c["sinks"] is not None:
                z = torch.logaddexp(z, c["sinks"].double().view(hkv, group))
            w = torch.exp(s - z[..., None])
            out[i] = torch.einsum("hgn,nhd->hgd", w, vv).reshape(-1, d)
            mean[i] = torch.einsum("hgn,nhd->hgd", w, vv.abs()).reshape(-1, d)
            lse[i] = z.view(-1)
    return out, lse, mean, size


def attention(c, ctas=None):
    from akv_b200.context_tree import TreeAttention

    return TreeAttention(c["hkv"] * c["group"], c["hkv"], c["d"], len(c["kv"]) - 1, "cuda",
                         dtype=c["dtype"], ctas=ctas).plan(c["kv"], c["dr"])


def launch(c, attn, **more):
    return attn.run(c["q"], c["k"], c["v"], c["indices"], c["draft"], c["mask"], sinks=c["sinks"],
                    window=c["window"], q_positions=c["qpos"], kv_positions=c["kpos"], **more)


def compare(c, out, lse):
    want, want_lse, mean, size = exact(c)
    u = torch.finfo(c["dtype"]).eps / 2
    keys = int((np.diff(c["kv"]) + np.diff(c["dr"])).max()) if len(c["kv"]) > 1 else 0
    e32 = (c["d"] + 4) * 2.0**-23 * size + 2.0**-21 + keys * 2.0**-24
    # fp16's subnormal P: half its smallest step per key, of rows whose maximum weighs 1
    tiny = keys * 2.0**-25 if c["dtype"] == torch.float16 else 0.0
    bound = u * want.abs() + (u + 2 * e32[..., None]) * mean + tiny + 2.0**-24
    bad = ~((out.double() - want).abs() <= bound * (1 + u))
    assert not bool(bad.any()), (int(bad.sum()), float((out.double() - want).abs().max()))
    finite = torch.isfinite(want_lse)
    assert torch.equal(torch.isfinite(lse), finite)
    err = (lse.double() - want_lse)[finite].abs()
    assert bool((err <= (e32 + 2.0**-22 * want_lse.abs() + 2.0**-20)[finite]).all())


def check(c, ctas=None):
    attn = attention(c, ctas)
    out, lse = launch(c, attn, return_lse=True)
    torch.cuda.synchronize()
    assert int(attn.error_flag) == 0
    compare(c, out, lse)
    return out, lse


LENGTHS = [0, 1, 63, 64, 65, 300, 129]
NEW = [1, 64, 16, 17, 1, 5, 0]


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("hkv,group", [(8, 8), (1, 8), (3, 5), (2, 1), (2, 16), (1, 40)])
@pytest.mark.parametrize("sinks", [False, True])
def test_tree_attention_matches_the_definition(d, hkv, group, sinks):
    check(make(LENGTHS, NEW, hkv, group, d, torch.bfloat16, seed=hkv + group, sinks=sinks))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ctas", [1, 3, 37, None])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_requests_cut_into_pieces(d, ctas, dtype):
    check(make([2000, 5, 700, 0, 4097], [3, 9, 40, 2, 16], 2, 8, d, dtype, seed=3, sinks=True), ctas)


@pytest.mark.parametrize("window", [0, 1, 7, 128, 100000])
@pytest.mark.parametrize("d", [64, 128])
def test_windows(window, d):
    check(make([0, 3, 64, 200, 500], [5, 64, 16, 9, 33], 2, 8, d, torch.bfloat16, seed=window,
               window=window))


@pytest.mark.parametrize("new", [1, 2, 15, 16, 31, 32, 33, 48, 63, 64])
def test_every_row_tile_boundary(new):
    check(make([130, 64], [new, max(1, new - 1)], 4, 8, 64, torch.bfloat16, seed=new, sinks=True))
    check(make([130], [new], 2, 8, 128, torch.float16, seed=new))


def test_large_scores_and_rising_maxima():
    """Scores of +-100s: the running maximum moves in steps past every threshold."""
    c = make([900, 70], [16, 3], 2, 8, 64, torch.bfloat16, seed=1, scale=40.0)
    order = torch.argsort((c["q"][0, 0].float() @ c["k"][c["indices"][:900].long(), 0].float().T))
    c["indices"][:900] = c["indices"][:900][order]
    check(c)
    check(make([900, 70], [16, 3], 2, 8, 128, torch.float16, seed=2, scale=20.0))


@pytest.mark.parametrize("sinks", [False, True])
def test_rows_that_see_nothing(sinks):
    c = make([0, 0, 70], [4, 64, 2], 2, 8, 64, torch.bfloat16, seed=4, sinks=sinks)
    c["mask"][1], c["mask"][10], c["mask"][-1] = 0, 0, 0
    out, lse = check(c)
    assert bool((out[1] == 0).all())
    assert sinks or bool((lse[1] == -np.inf).all())   # with sinks: compare() bounds it


@pytest.mark.parametrize("sink", [200.0, -200.0, -float("inf")])
def test_sinks_far_from_every_score(sink):
    c = make([0, 70, 900], [4, 16, 2], 2, 8, 64, torch.bfloat16, seed=4, sinks=True)
    c["mask"][1] = 0
    c["sinks"][::3] = sink
    check(c)
    check(c, 1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("window", [-1, 9])
def test_masked_keys_may_hold_anything(d, bad, window):
    """Infinities and NaN in drafted tokens that a row does not see (another
    branch, another request's slots, keys out of the window) do not reach it."""
    c = make([70, 3, 130], [16, 64, 5], 2, 8, d, torch.bfloat16, seed=5, window=window)
    node = 3  # of request 0; only rows with its bit may see it
    slot = int(c["draft"][node])
    rows = torch.nonzero((c["mask"][:16] >> node) & 1).flatten()
    for pool in ("k", "v"):
        d_ = {**c, pool: c[pool].clone()}
        d_[pool][slot] = bad
        attn = attention(c)
        out, lse = launch(d_, attn, return_lse=True)
        clean, clean_lse = launch(c, attn, return_lse=True)
        keep = torch.ones(85, dtype=torch.bool, device="cuda")
        keep[rows] = False
        assert torch.equal(out[keep], clean[keep]) and torch.equal(lse[keep], clean_lse[keep])
        if pool == "v":
            assert not bool(out[rows].isfinite().any())
    if window >= 0:  # the first cached key of request 2 lies outside every window
        for pool in ("k", "v"):
            d_ = {**c, pool: c[pool].clone()}
            d_[pool][int(c["indices"][73])] = bad
            out, lse = launch(d_, attn, return_lse=True)
            assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [8, 5])
@pytest.mark.parametrize("shuffled", [False, True])
def test_windows_over_many_tiles(d, group, shuffled):
    """Tiles wholly inside, wholly outside and across the windows, also with
    positions that do not rise along the row, and tokens far apart."""
    c = make([1500, 900, 128, 2000], [16, 33, 4, 64], 3, group, d, torch.float16, seed=9, window=1300,
             sinks=True)
    if shuffled:
        g = torch.Generator(device="cuda").manual_seed(3)
        c["kpos"] = c["kpos"][torch.randperm(len(c["kpos"]), generator=g, device="cuda")].contiguous()
        c["qpos"] = c["qpos"] + 150 * (torch.arange(len(c["qpos"]), device="cuda") % 3).int()
    check(c)
    check(c, ctas=5)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_bad_values_inside_and_outside_long_windows(d, bad):
    """One bad V element at a key that every row sees, that some rows see and
    that none sees, each in a tile of its own: it changes that element of the
    rows that see it and nothing else."""
    c = make([1000, 300], [16, 5], 2, 8, d, torch.bfloat16, seed=10, window=700)
    c["qpos"][:16] = int(c["kpos"][999]) + 1 + 40 * torch.arange(16, device="cuda").int()
    attn = attention(c)
    clean, clean_lse = launch(c, attn, return_lse=True)
    seen_by = lambda j: c["qpos"][:16] - c["kpos"][j] <= 700  # noqa: E731
    counts = torch.stack([seen_by(j).sum() for j in range(1000)])
    for keys in ((counts == 16), (counts > 0) & (counts < 16), (counts == 0)):
        j = int(torch.nonzero(keys).flatten()[int(keys.sum()) // 2])
        v = c["v"].clone()
        v[int(c["indices"][j]), 1, 7] = bad
        out, lse = launch({**c, "v": v}, attn, return_lse=True)
        hit = torch.zeros_like(out, dtype=torch.bool)
        hit[:16][seen_by(j), 8:, 7] = True
        assert torch.equal(lse, clean_lse) and torch.equal(out[~hit], clean[~hit])
        want = torch.full_like(out, bad)
        assert torch.equal(out[hit].isnan(), want[hit].isnan())
        assert torch.equal(out[hit].nan_to_num(0.5), want[hit].nan_to_num(0.5))


def test_one_infinite_element_of_a_visible_key():
    c = make([70], [3], 2, 8, 64, torch.bfloat16, seed=6)
    c["mask"].copy_(torch.tensor([1, 3, 5]))
    c["v"][int(c["draft"][1]), 1, 7] = float("inf")
    out = launch(c, attention(c))
    hit = torch.zeros_like(out, dtype=torch.bool)
    hit[1, 8:, 7] = True
    assert bool((out[hit] == float("inf")).all()) and bool(out[~hit].isfinite().all())


def test_padding_tokens_read_as_zeros_and_bad_slots_are_reported():
    c = make([40, 9], [8, 8], 2, 8, 64, torch.bfloat16, seed=7)
    c["draft"][5:8] = -1          # seen by their own rows only: their mask stays
    c["draft"][12] = -7
    c["mask"][13:16] = 0
    check(c)
    attn = attention(c)
    c["indices"][3] = c["k"].shape[0]
    launch(c, attn)
    with pytest.raises(RuntimeError, match="outside the KV pools"):
        attn.check()
    attn.check()
    c["indices"][3] = -1
    launch(c, attn)
    assert int(attn.error_flag) == 1


def test_strided_pools_and_outputs():
    """K and V interleaved in one buffer, heads before slots, q and out views."""
    c = make([300, 20], [16, 40], 4, 8, 64, torch.bfloat16, seed=8, sinks=True)
    want, _ = check(c)
    slots = c["k"].shape[0]
    both = torch.empty(slots, 2, 4, 64, dtype=c["dtype"], device="cuda")
    both[:, 0], both[:, 1] = c["k"], c["v"]
    by_head = c["k"].transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.full((60, 40, 128), 5.0, dtype=c["dtype"], device="cuda")
    q = torch.zeros(60, 40, 64, dtype=c["dtype"], device="cuda")
    q[:56, :32] = c["q"]
    attn = attention(c)
    for k, v in ((both[:, 0], both[:, 1]), (by_head, c["v"])):
        out = attn.run(q[:, :32], k, v, c["indices"], c["draft"], c["mask"], sinks=c["sinks"],
                       out=wide[:, :32, 64:])
        assert torch.equal(out[:56], want)
    assert bool((wide[56:] == 5).all()) and bool((wide[..., :64] == 5).all())


def test_slots_past_32_bits_of_elements():
    slots = (1 << 31) // (8 * 128) + 11
    c = make([200, 31], [16, 3], 8, 8, 128, torch.bfloat16, seed=9)
    n = c["k"].shape[0]
    big = {**c, "k": torch.zeros(slots, 8, 128, dtype=c["dtype"], device="cuda"),
           "v": torch.zeros(slots, 8, 128, dtype=c["dtype"], device="cuda")}
    big["k"][slots - n:], big["v"][slots - n:] = c["k"], c["v"]
    big["indices"], big["draft"] = c["indices"] + (slots - n), c["draft"] + (slots - n)
    assert torch.equal(launch(big, attention(big)), launch(c, attention(c)))


def test_replayed_graphs_follow_masks_slots_and_plans():
    c = make([100, 200], [8, 8], 2, 8, 64, torch.bfloat16, seed=10)
    attn = attention(c)
    out = torch.empty_like(c["q"])
    launch(c, attn, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        launch(c, attn, out=out)
    other = make([100, 200], [8, 8], 2, 8, 64, torch.bfloat16, seed=11)
    for name in ("q", "k", "v", "indices", "draft", "mask"):
        c[name].copy_(other[name])
    out.zero_()
    graph.replay()
    assert torch.equal(out, launch(other, attention(other)))


def test_a_replay_on_a_larger_plan_stays_in_its_tensors():
    """The captured call's vectors bound it, whatever plan the device holds."""
    c = make([100, 200], [8, 8], 2, 8, 64, torch.bfloat16, seed=10)
    attn = attention(c)
    wide = torch.full((200, 16, 64), 3.0, dtype=c["dtype"], device="cuda")
    graph = torch.cuda.CUDAGraph()
    launch(c, attn, out=wide)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        launch(c, attn, out=wide)
    attn.plan([0, 100, 400], [0, 64, 128])
    graph.replay()
    torch.cuda.synchronize()
    assert bool((wide[16:] == 3).all())
    with pytest.raises(RuntimeError, match="replayed"):
        attn.check()
    attn.plan(c["kv"], c["dr"])
    graph.replay()
    assert torch.equal(wide[:16], launch(c, attention(c)))


def test_visible_nan_keys_make_their_rows_nan():
    c = make([700, 5], [16, 3], 2, 8, 64, torch.bfloat16, seed=16)
    for at in (3, 40, 333, 699):        # columns of every kind of a tile
        k = c["k"].clone()
        k[int(c["indices"][at]), 1, 9] = float("nan")
        out, lse = launch({**c, "k": k}, attention(c), return_lse=True)
        assert bool(out[:16, 8:].isnan().all()) and bool(lse[:16, 8:].isnan().all())
        assert bool(out[:16, :8].isfinite().all()) and bool(out[16:].isfinite().all())


def test_results_do_not_change_from_run_to_run():
    c = make([3000, 10, 517], [16, 33, 1], 8, 8, 64, torch.bfloat16, seed=12, sinks=True)
    attn = attention(c)
    first = launch(c, attn)
    for _ in range(5):
        assert torch.equal(launch(c, attn), first)


@pytest.mark.parametrize("ctas", [None, 2, 1])
def test_the_output_may_be_the_queries(ctas):
    c = make([700, 30, 0, 1500], [16, 64, 3, 5], 3, 5, 64, torch.bfloat16, sinks=True)
    want = launch(c, attention(c, ctas))
    mine = {**c, "q": c["q"].clone()}
    got = launch(mine, attention(c, ctas), out=mine["q"])
    assert got is mine["q"] and torch.equal(got, want)


def test_two_instances_on_two_streams():
    cases = [make([1500, 40], [16, 20], 4, 8, 64, torch.bfloat16, seed=s) for s in (13, 14)]
    attns = [attention(c) for c in cases]
    want = [launch(c, a) for c, a in zip(cases, attns)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [None, None]
    for _ in range(4):
        for n in range(2):
            with torch.cuda.stream(streams[n]):
                got[n] = launch(cases[n], attns[n])
    torch.cuda.synchronize()
    for n in range(2):
        assert torch.equal(got[n], want[n])


def test_batches_of_the_serving_kind():
    rng = np.random.default_rng(15)
    check(make(rng.integers(1, 1500, 40), rng.integers(0, 20, 40), 8, 8, 64, torch.bfloat16, seed=15,
               sinks=True))


def test_refusals():
    from akv_b200.context_tree import TreeAttention

    for bad in ((63, 8, 64), (64, 0, 64), (64, 8, 96), (64, 8, 256)):
        with pytest.raises(ValueError):
            TreeAttention(*bad, 4, "cuda")
    with pytest.raises(ValueError):
        TreeAttention(64, 8, 64, 4, "cuda", dtype=torch.float32)
    c = make([40, 9], [8, 8], 2, 8, 64, torch.bfloat16, window=5)
    attn = attention(c)
    with pytest.raises(ValueError):
        attn.plan([0, 1, 2, 3], [0, 1, 2, 3])     # above max_batch
    ok = dict(q=c["q"], k_pool=c["k"], v_pool=c["v"], kv_indices=c["indices"], draft_slots=c["draft"],
              tree_mask=c["mask"])
    for change in (dict(q=c["q"].half()), dict(q=c["q"][:15]), dict(q=c["q"][:, :8]),
                   dict(k_pool=c["k"][:, :1]), dict(v_pool=c["v"].float()),
                   dict(kv_indices=c["indices"].long()), dict(kv_indices=c["indices"][:-1]),
                   dict(draft_slots=c["draft"][:-1]), dict(tree_mask=c["mask"].int()),
                   dict(tree_mask=c["mask"].cpu()), dict(sinks=torch.zeros(8, device="cuda")),
                   dict(sinks=torch.zeros(16, device="cuda").half()), dict(window=5),
                   dict(window=5, q_positions=c["qpos"], kv_positions=c["kpos"].long()),
                   dict(out=c["q"][:15]), dict(out=c["q"].float()),
                   dict(q=torch.zeros(16, 16, 68, dtype=c["dtype"], device="cuda")[..., 4:])):
        with pytest.raises(ValueError):
            attn.run(**{**ok, **change})
    none = attn.plan([0], [0])
    assert none.run(**ok).shape == (0, 16, 64)
