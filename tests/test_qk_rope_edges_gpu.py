"""Q/K norm, rotation and store with the vectors of a larger slot map."""

import pytest
import torch

from test_qk_rope_gpu import inputs

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens", [1, 6])
def test_positions_and_slots_may_be_longer_than_the_tokens(index, tokens):
    """What follows the last token's entry is not read."""
    from akv_b200.context_rope import qk_norm_rope

    x = inputs(tokens, 4, 2, 64, 64, torch.bfloat16)
    pools = torch.full((2, 2, tokens + 5, 2, 64), 3.0, dtype=torch.bfloat16, device="cuda")
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    tail = torch.full((9,), 1 << 20, dtype=index, device="cuda")
    long = lambda t: torch.cat((t.to(index), tail))  # noqa: E731
    got = []
    for pool, pos, slots in ((pools[0], x["pos"], x["perm"]),
                             (pools[1], long(x["pos"]), long(x["perm"]))):
        got.append(qk_norm_rope(x["q"], x["k"], pos, x["table"], q_weight=x["wq"], k_weight=x["wk"],
                                v=x["v"], k_pool=pool[0], v_pool=pool[1], slots=slots,
                                error_flag=flag)[0])
    assert int(flag) == 0 and torch.equal(*got) and torch.equal(pools[0], pools[1])
    for bad in (dict(positions=x["pos"][: tokens - 1]), dict(positions=long(x["pos"])[::2])):
        if tokens > 1:
            with pytest.raises(ValueError):
                qk_norm_rope(**{**dict(q=x["q"], k=x["k"], positions=x["pos"],
                                       cos_sin_cache=x["table"]), **bad})
