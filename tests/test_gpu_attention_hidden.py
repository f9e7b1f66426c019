"""What a row of the attention must see, and what it must not: NaN and
infinities beside missing blocks.  Bounds: operator_helpers.attention_reference."""
import math

import pytest
import torch

from kvx_amd.abi import Status

from operator_helpers import AttentionCase, set_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("io,cache", [("bf16", None), ("f16", None), ("f32", None),
                                      ("f16", "e5m2"), ("bf16", "e4m3")])
@pytest.mark.parametrize("layout", ["nhd", "vllm"])
@pytest.mark.parametrize("table", ["packed", "ragged"])
@pytest.mark.parametrize("new,window", [([90], 0), ([90], 120), ([5], 0), ([1], 0)])
def test_infinities_beside_missing_blocks(io, cache, layout, table, new, window):
    """Elements of values that are not finite, in steps some of whose blocks are
    not there: every row that sees the token has them."""
    bad = math.inf if cache != "e4m3" else math.nan
    c = AttentionCase(io=io, cache=cache, layout=layout, table=table, lens=[200], new=new, D=64,
                      H=2, G=4, window=window, holes=[(0, 0), (0, 6), (0, 11)])
    want, _, tol, _ = c.reference()
    for t, h, d, sign in ((20, 0, 17, 1), (30, 1, 3, -1), (85, 1, 40, -1), (115, 0, 63, 1),
                          (170, 1, 5, 1)):
        c.rows[1][int(c.tb[0, t // 16]), t % 16, h, d] = sign * bad
        for i in range(new[0]):
            p = 200 - new[0] + i
            if t <= p and (window == 0 or t > p - window):
                want[i, h * c.G: (h + 1) * c.G, d] += sign * bad
    set_rows(c.cache.value_cache, c.cache.v_layout, c.rows[1])
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    got = c.out.cpu().double()
    fine = torch.isfinite(want)
    assert (~fine).any()
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    half = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}[io]
    over = (got - want).abs()[fine] - (tol + half * (want.abs() + tol) + 2.0 ** -25)[fine]
    assert (over <= 0).all()
