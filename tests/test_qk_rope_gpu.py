"""Q/K norm, rotation and cache store in one pass (C ABI akv_qk_norm_rope),
against the formula in 64 bits.

Tolerance: the kernel computes in fp32 and rounds once.  The rounding is off
by at most eps(type)/2 of the result.  In fp32 a row of D elements costs: the
sum of D squares, at most D roundings, (D/2) * 2^-24 relative on the root;
two products, the division, the root and the reciprocal root (2 ulp), and a rotation of
two products and a sum: under 16 * 2^-24 of |y| rotated, where the rotated
pair's size bounds both terms.  So |error| <= eps/2 |want| + (D/2 + 16) 2^-24
pair, with pair = |y0 c| + |y1 s|.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


def formula(x, w, table, pos, neox, eps):
    """(result, size of the terms) in 64 bits."""
    x = x.double()
    if w is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w.double()
    row = table.double()[pos.long()][:, None]
    half = table.shape[1] // 2
    c, s = row[..., :half], row[..., half:]
    i = torch.arange(half, device=x.device)
    a, b = (i, i + half) if neox else (2 * i, 2 * i + 1)
    y, size = x.clone(), x.abs()
    y[..., a] = x[..., a] * c - x[..., b] * s
    y[..., b] = x[..., b] * c + x[..., a] * s
    size[..., a] = (x[..., a] * c).abs() + (x[..., b] * s).abs()
    size[..., b] = (x[..., b] * c).abs() + (x[..., a] * s).abs()
    return y, size


def near(got, want, size, d):
    bound = torch.finfo(got.dtype).eps / 2 * want.abs() + (d / 2 + 16) * 2.0**-24 * size
    tiny = torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps  # a subnormal's half step
    assert bool(((got.double() - want).abs() <= bound * 1.0001 + tiny).all())


def inputs(tokens, hq, hkv, d, rotary, dtype, *, wdtype=None, cdtype=torch.float32, seed=0,
           magnitude=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    qkv = (2 * rand(tokens, (hq + 2 * hkv) * d)).to(dtype)
    q, k, v = (t.view(tokens, -1, d) for t in qkv.split([hq * d, hkv * d, hkv * d], 1))
    angle = 300 * torch.rand(500, rotary // 2, generator=g, device="cuda")
    return dict(q=q, k=k, v=v, table=(magnitude * torch.cat((angle.cos(), angle.sin()), 1)).to(cdtype),
                pos=torch.randint(0, 500, (tokens,), generator=g, device="cuda"),
                wq=(1 + 0.3 * rand(d)).to(wdtype or dtype), wk=(1 + 0.3 * rand(d)).to(wdtype or dtype),
                perm=torch.randperm(tokens + 5, generator=g, device="cuda")[:tokens])


SHAPES = [  # tokens, hq, hkv, head_dim, rotary_dim
    (1, 64, 8, 64, 64), (37, 8, 1, 128, 128), (5, 5, 3, 80, 48), (3, 9, 2, 96, 96),
    (7, 4, 4, 256, 128), (2, 1, 1, 16, 16), (4, 3, 1, 512, 512), (11, 6, 2, 32, 16),
    (129, 40, 8, 192, 64),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("neox", [True, False])
def test_matches_the_formula(shape, dtype, neox):
    from akv_b200.context_rope import qk_norm_rope

    tokens, hq, hkv, d, rotary = shape
    x = inputs(*shape, dtype, seed=tokens)
    kp = torch.full((tokens + 5, hkv, d), 7.0, dtype=dtype, device="cuda")
    vp = kp.clone()
    k_out = torch.empty(tokens, hkv, d, dtype=dtype, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, k = qk_norm_rope(x["q"], x["k"], x["pos"].int(), x["table"], q_weight=x["wq"],
                        k_weight=x["wk"], is_neox_style=neox, v=x["v"], k_pool=kp, v_pool=vp,
                        slots=x["perm"], k_out=k_out, error_flag=flag)
    assert k is k_out and int(flag) == 0
    near(q, *formula(x["q"], x["wq"], x["table"], x["pos"], neox, 1e-6), d)
    near(k, *formula(x["k"], x["wk"], x["table"], x["pos"], neox, 1e-6), d)
    assert torch.equal(kp[x["perm"]], k) and torch.equal(vp[x["perm"]], x["v"])
    rest = torch.ones(tokens + 5, dtype=torch.bool, device="cuda")
    rest[x["perm"]] = False
    assert bool((kp[rest] == 7).all()) and bool((vp[rest] == 7).all())


@pytest.mark.parametrize("wdtype", [None, torch.float32])
@pytest.mark.parametrize("cdtype", [torch.float32, torch.bfloat16, torch.float16])
def test_weight_and_table_types(wdtype, cdtype):
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(19, 16, 2, 64, 32, torch.bfloat16, wdtype=wdtype, cdtype=cdtype, magnitude=1.3)
    q, k = qk_norm_rope(x["q"], x["k"], x["pos"], x["table"], q_weight=x["wq"], k_weight=x["wk"],
                        eps=0.5)
    near(q, *formula(x["q"], x["wq"], x["table"], x["pos"], True, 0.5), 64)
    near(k, *formula(x["k"], x["wk"], x["table"], x["pos"], True, 0.5), 64)


def test_without_weights_rows_are_only_rotated_and_in_place_is_the_same():
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(33, 8, 8, 128, 64, torch.bfloat16)
    for weights in ({}, dict(q_weight=x["wq"]), dict(q_weight=x["wq"], k_weight=x["wk"])):
        q, k = qk_norm_rope(x["q"], x["k"], x["pos"], x["table"], **weights)
        near(q, *formula(x["q"], weights.get("q_weight"), x["table"], x["pos"], True, 1e-6), 128)
        near(k, *formula(x["k"], weights.get("k_weight"), x["table"], x["pos"], True, 1e-6), 128)
        mine = x["q"].clone(), x["k"].clone()
        qk_norm_rope(*mine, x["pos"], x["table"], q_out=mine[0], k_out=mine[1], **weights)
        assert torch.equal(mine[0], q) and torch.equal(mine[1], k)


def test_padding_bad_slots_and_bad_positions():
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(6, 8, 2, 64, 64, torch.float16)
    pool = torch.full((2, 6, 2, 64), 3.0, dtype=torch.float16, device="cuda")
    slots = torch.tensor([0, -1, 5, 6, 2, 1 << 40], device="cuda")
    pos = x["pos"].clone()
    pos[4], pos[0] = 500, 499
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    q, _ = qk_norm_rope(x["q"], x["k"], pos, x["table"], q_weight=x["wq"], k_weight=x["wk"],
                        v=x["v"], k_pool=pool[0], v_pool=pool[1], slots=slots, error_flag=flag)
    assert int(flag) == 1
    seen = pos.clone()
    seen[4] = 0
    near(q, *formula(x["q"], x["wq"], x["table"], seen, True, 1e-6), 64)
    want, size = formula(x["k"], x["wk"], x["table"], seen, True, 1e-6)
    near(pool[0][[0, 5]], want[[0, 2]], size[[0, 2]], 64)
    assert torch.equal(pool[1][[0, 5]], x["v"][[0, 2]])
    assert bool((pool[:, 1:5] == 3).all())
    flag.zero_()
    qk_norm_rope(x["q"][:3], x["k"][:3], pos[:3], x["table"], v=x["v"][:3], k_pool=pool[0],
                 v_pool=pool[1], slots=slots[:3].int(), error_flag=flag)
    assert int(flag) == 0   # padding is no error


def test_infinities_and_zero_rows():
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(3, 2, 2, 64, 64, torch.bfloat16)
    q = x["q"].clone()
    q[0, 0], q[1, 1, 5] = 0.0, float("nan")
    out, _ = qk_norm_rope(q, x["k"], x["pos"], x["table"], q_weight=x["wq"], k_weight=x["wk"])
    assert bool((out[0, 0] == 0).all()) and bool(out[1, 1].isnan().all())
    clean = torch.ones(3, 2, dtype=torch.bool)
    clean[1, 1] = False
    assert bool(out[clean].isfinite().all())


@pytest.mark.parametrize("neox", [True, False])
@pytest.mark.parametrize("d,rotary", [(128, 64), (80, 48), (256, 16)])
@pytest.mark.parametrize("normed", [False, True])
def test_dimensions_past_the_rotation_do_not_reach_one_another(neox, d, rotary, normed):
    """An infinity there changes its own element (and the norm), no other."""
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(d - rotary, 3, 2, d, rotary, torch.float16, seed=2)
    row = torch.arange(d - rotary, device="cuda")
    for t in (x["q"], x["k"]):  # token i: the i-th of these dimensions
        t[row, 1, rotary + row] = float("inf") if normed else float("nan")
        t[row, 0, rotary + row] = -float("inf")
    w = dict(q_weight=x["wq"], k_weight=x["wk"]) if normed else {}
    q, k = qk_norm_rope(x["q"], x["k"], x["pos"], x["table"], is_neox_style=neox, **w)
    for got, t, wt in ((q, x["q"], x["wq"]), (k, x["k"], x["wk"])):
        want, size = formula(t, wt if normed else None, x["table"], x["pos"], neox, 1e-6)
        odd = ~torch.isfinite(want)
        assert torch.equal(torch.isnan(got), torch.isnan(want))
        assert torch.equal(torch.isinf(got), torch.isinf(want))
        near(got.masked_fill(odd, 0), want.masked_fill(odd, 0), size.masked_fill(odd, 0), d)


def test_a_row_past_32_bits_of_elements():
    """Pool rows whose element offset passes 2^31."""
    from akv_b200.context_rope import qk_norm_rope

    slots = (1 << 31) // (8 * 128) + 7
    pool = torch.zeros(slots, 8, 128, dtype=torch.bfloat16, device="cuda")
    x = inputs(3, 8, 8, 128, 128, torch.bfloat16)
    at = torch.tensor([slots - 1, 0, slots - 6], device="cuda")
    _, k = qk_norm_rope(x["q"], x["k"], x["pos"], x["table"], k_weight=x["wk"], v=x["v"], k_pool=pool,
                        v_pool=pool.clone(), slots=at, k_out=torch.empty_like(x["k"].contiguous()))
    assert torch.equal(pool[at], k)
    pool[at] = 0
    assert not bool(pool.view(torch.int16).any())


def test_side_stream_and_graph():
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(40, 16, 4, 64, 64, torch.bfloat16)
    want, _ = qk_norm_rope(x["q"], x["k"], x["pos"], x["table"], q_weight=x["wq"])
    out = torch.zeros_like(want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        qk_norm_rope(x["q"], x["k"], x["pos"], x["table"], q_weight=x["wq"], q_out=out)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def test_refusals():
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(4, 8, 2, 64, 64, torch.bfloat16)
    ok = dict(q=x["q"], k=x["k"], positions=x["pos"], cos_sin_cache=x["table"])
    pool = torch.zeros(9, 2, 64, dtype=torch.bfloat16, device="cuda")
    store = dict(v=x["v"], k_pool=pool, v_pool=pool, slots=x["perm"])
    odd = torch.zeros(4, 8, 65, dtype=torch.bfloat16, device="cuda")[..., 1:]
    for change in (dict(q=x["q"].double()), dict(q=x["q"].cpu()), dict(k=x["k"][:3]), dict(k=x["k"].float()),
                   dict(q=odd), dict(positions=x["pos"][:2]), dict(positions=x["pos"].float()),
                   dict(cos_sin_cache=x["table"][:, :40]), dict(rotary_dim=32),
                   dict(cos_sin_cache=x["table"].double()), dict(q_weight=x["wq"].half()),
                   dict(q_weight=x["wq"], k_weight=x["wk"].float()), dict(q_weight=x["wq"][:32]),
                   {**store, "slots": None}, {**store, "v": x["v"][:2]}, {**store, "v": None},
                   {**store, "k_pool": pool[:, :1]}, {**store, "slots": x["perm"].float()},
                   dict(slots=x["perm"]), dict(q_out=x["k"]),
                   dict(q=x["q"][..., :40], k=x["k"][..., :40])):
        with pytest.raises(ValueError):
            qk_norm_rope(**{**ok, **change})
    q, k = qk_norm_rope(x["q"][:0], x["k"][:0], x["pos"][:0], x["table"])
    assert q.shape == (0, 8, 64) and k.shape == (0, 2, 64)
