"""What a row of the attention must not see, and what it must: scales of pages
in front of its window or of nobody, scales that only other rows see, NaN and
infinities beside missing blocks.  Bounds: operator_helpers.attention_reference."""
import math

import pytest
import torch

from kvx_amd.abi import Status

from operator_helpers import AttentionCase, scale_rows, set_rows

pytestmark = pytest.mark.gpu

POISON = (math.nan, math.inf, -math.inf, 1e30)


def seen_blocks(c, window):
    """Blocks with a token that some row attends to."""
    live = torch.zeros(c.nb, dtype=torch.bool)
    for s, (n, m) in enumerate(zip(c.lens, c.new)):
        first = max(n - m + 1 - window, 0) if window else 0
        live[c.tb[s, first // c.bs: -(-n // c.bs)]] = True
    return live


@pytest.mark.parametrize("table,bs,layout,D", [("packed", 8, "nhd", 64), ("packed", 16, "nhd", 128),
                                               ("packed", 32, "vllm", 64), ("packed", 16, "hnd", 256),
                                               ("ragged", 16, "nhd", 64), ("ragged", 8, "vllm", 128),
                                               ("packed", 8, "nhd", 20)])
@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window", [17, 100])
@pytest.mark.parametrize("lens,new", [([100, 35, 2600], None), ([200, 35, 2600], [90, 3, 70])])
def test_scales_of_hidden_pages(lens, new, window, io, table, bs, layout, D):
    """Pages that slid out of the window, and pages of nobody, have scales that
    were never written."""
    for kind in ("block", "block_head"):
        c = AttentionCase(io=io, cache="e4m3", scales=kind, layout=layout, table=table, bs=bs, H=2,
                          G=2, D=D, lens=lens, new=new, window=window)
        dead = (~seen_blocks(c, window)).nonzero()[:, 0]
        assert dead.numel() > 3
        for s in c.kv_scales:
            for i, b in enumerate(dead.tolist()):
                s.values[b] = POISON[(i + b) % 4]
        assert c.run() == Status.OK
        c.check()


@pytest.mark.parametrize("poison", [math.nan, math.inf, 1e30])
@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new", [None, [40, 70]])
def test_one_kind_of_hidden_scale(io, new, poison):
    c = AttentionCase(io=io, cache="e5m2", scales="block", H=1, G=4, D=64, lens=[100, 300], new=new,
                      window=33)
    dead = ~seen_blocks(c, 33)
    for s in c.kv_scales:
        s.values[dead.to("cuda")] = poison
    assert c.run() == Status.OK
    c.check()


@pytest.mark.parametrize("poison", [math.nan, math.inf])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("table", ["packed", "ragged"])
@pytest.mark.parametrize("new,D", [([44], 64), ([7], 128), ([44], 20)])
def test_scales_that_some_rows_see(new, D, table, io, which, poison):
    """One page's scale is not finite: rows that attend to a token of it turn
    so, the others stay what they are.  An infinite scale of keys makes a negative
    product a logit of -infinity: a token that does not count."""
    window = 50
    for block in (11, 8):  # of the new tokens, and leaving the window
        c = AttentionCase(io=io, cache="e4m3", scales="block", H=2, G=2, D=D, lens=[190], new=new,
                          window=window, table=table)
        page = int(c.tb[0, block])
        c.kv_scales[which].values[page] = poison
        assert c.run() == Status.OK
        torch.cuda.synchronize()
        ref = list(c.reference())
        rows_of = c.rows_of
        c.rows_of = lambda s: (*rows_of(s)[:2], torch.arange(190) // 16 != block)
        without = c.reference()
        out, lse = c.out.cpu().double(), c.lse.cpu()
        sees = 0
        for i in range(new[0]):
            p = 190 - new[0] + i
            t = torch.arange(16 * block, 16 * block + 16)
            t = t[(t <= p) & (t > p - window)] % 16
            if t.numel() == 0:
                continue
            sees += 1
            for h in range(4):
                dots = c.rows[0][page, t, h // 2].double() @ c.q[i, h].double()
                if which == 0 and poison == math.inf and (dots < 0).all():
                    for x, y in zip(ref, without):
                        x[i, h] = y[i, h]
                    continue
                assert not torch.isfinite(out[i, h]).any()
                if which == 0:
                    assert not math.isfinite(lse[i, h])
                c.out[i, h] = ref[0][i, h].to(c.out.dtype).cuda()
                c.lse[i, h] = ref[1][i, h].float().cuda()
        assert sees > 0 or (block == 8 and new[0] == 7)
        c.reference = lambda: ref
        c.check()


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


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("cache", ["e4m3", "e5m2"])
@pytest.mark.parametrize("new", [None, [30, 1, 60]])
@pytest.mark.parametrize("table", ["packed", "ragged"])
def test_pages_of_very_different_scales(io, cache, new, table):
    """A page whose values have a scale 10^8 times the others', but whose tokens
    have weights near e^-28: its part is small, and the others keep their
    digits."""
    c = AttentionCase(io=io, cache=cache, scales="block", H=2, G=2, D=64, lens=[96, 40, 150],
                      new=new, table=table)
    ks = torch.ones(c.nb)
    vs = torch.full((c.nb,), 0.01)
    k = 0.5 * torch.randn(c.rows[0].shape, generator=torch.Generator().manual_seed(3))
    k[..., 0] = 0
    for s, j in ((0, 1), (1, 0), (2, 4)):
        b = int(c.tb[s, j])
        vs[b] = 1e6
        k[b, ..., 0] = -28.0
    c.q[..., 0] = 8.0
    c.q_dev.copy_(c.q)
    c.rows[0] = k.to(c.rows[0].dtype)
    set_rows(c.cache.key_cache, c.cache.k_layout, c.rows[0])
    for w, x in enumerate((ks, vs)):
        c.kv_scales[w].values.copy_(x)
        c.exact[w] = c.rows[w].double() * scale_rows(x, "block", c.nb, c.H)[:, None, :, None]
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    c.check()


@pytest.mark.parametrize("table,bs,layout", [("packed", 16, "nhd"), ("packed", 8, "vllm"),
                                             ("ragged", 16, "nhd"), ("ragged", 8, "vllm")])
@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new", [None, [40, 3]])
@pytest.mark.parametrize("window", [0, 2000])
def test_block_scales_of_split_sequences(window, new, io, table, bs, layout):
    """Contexts whose tokens are divided among workgroups; pages of nobody, and
    those in front of the window, have scales that were never written."""
    for kind in ("block", "block_head"):
        c = AttentionCase(io=io, cache="e4m3", scales=kind, layout=layout, table=table, bs=bs, H=1,
                          G=4, D=64, lens=[5000, 70], new=new, window=window)
        for s in c.kv_scales:
            for i, b in enumerate((~seen_blocks(c, window)).nonzero()[:, 0].tolist()):
                s.values[b] = POISON[(i + b) % 4]
        assert c.run() == Status.OK
        c.check()


@pytest.mark.parametrize("io,cache,D", [("bf16", None, 64), ("f16", None, 64), ("f32", None, 64),
                                        ("bf16", None, 20), ("f32", None, 20), ("f16", "e5m2", 20)])
@pytest.mark.parametrize("new", [[1], [40]])
@pytest.mark.parametrize("bad", [math.nan, math.inf])
def test_values_of_tokens_of_next_to_no_weight(io, cache, D, new, bad):
    """A token whose weight is e^-200 of the others' is attended to all the same:
    a value that is not finite reaches every row that sees it."""
    c = AttentionCase(io=io, cache=cache, D=D, lens=[130], new=new, H=1, G=2, scale=0.125)
    k = torch.zeros(c.rows[0].shape)
    t = 70
    page = int(c.tb[0, t // 16])
    one = 1.0 if cache is None else 1.0 / float(c.kv_scales[0].values[0])
    k[page, t % 16, :, 0] = -40.0 * one
    c.q[..., 0] = 40.0
    c.q_dev.copy_(c.q)
    c.rows[0] = k.to(c.rows[0].dtype)
    set_rows(c.cache.key_cache, c.cache.k_layout, c.rows[0])
    c.rows[1][page, t % 16, 0, 3] = bad
    set_rows(c.cache.value_cache, c.cache.v_layout, c.rows[1])
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    out = c.out.cpu().double()
    assert not torch.isfinite(out[..., 3]).any()
    out[..., 3] = 0
    assert torch.isfinite(out).all() and torch.isfinite(c.lse).all()
