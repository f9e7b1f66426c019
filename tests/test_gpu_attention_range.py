"""Softcaps of any size, and long contexts whose weights are small beside one:
against the definition in 64 bits.

Softcap.  With x the logit and c the cap, c tanh(x / c) is computed relative to
itself: in F32 and on the vector unit from tanhf (a few units of 2^-24); in 16 bits
with caps past 64 (F16) or 512 (BF16) by a polynomial for |x| < c / 2 (2^-26 and about eight
roundings), else as c (1 - 2 / (1 + e)) with e = exp(2 x / c): exp2 and the
reciprocal are good to 2^-23, the argument's rounding is worth |y| (1 - tanh^2 y)
2^-23 < 0.45 * 2^-23, in all less than 2^-22 of 1 and so 2^-21 of tanh(1/2).  Twice
that, 2^-20, is allowed.  Smaller caps in 16 bits take the latter form for all x
and are allowed 2^-21 of the cap, as in the other tests.

Weights.  An F16 weight below 2^-14 of the largest would lose digits, and one
below 2^-25 all of them; a long context has many."""
import math

import pytest
import torch

from kvx_amd import paged
from kvx_amd.abi import Layout, Status

from operator_helpers import AttentionCase, DT, scale_arg, set_rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("softcap", [1e-3, 2.0, 50.0, 64.0, 65.0, 512.0, 513.0, 1e3, 1e5, 1e6, 1e20, 3e38])
@pytest.mark.parametrize("io,cache,D", [("bf16", None, 64), ("f16", None, 64), ("f32", None, 64),
                                        ("f16", "e4m3", 128), ("f32", "e5m2", 64),
                                        ("bf16", None, 20), ("f32", None, 20)])
@pytest.mark.parametrize("new", [None, [80, 3]])
@pytest.mark.parametrize("scale", [0.2, -3.0])
def test_softcaps(softcap, io, cache, D, new, scale):
    c = AttentionCase(io=io, cache=cache, lens=[100, 64], new=new, D=D, softcap=softcap, scale=scale)
    if softcap > (512 if io == "bf16" else 64) or io == "f32" or D == 20:
        c.cap_rel = 2.0 ** -20
    assert c.run() == Status.OK
    c.check()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("D", [64, 20])
def test_smallest_softcap(io, D):
    """A cap that is subnormal: all logits are as good as 0."""
    c = AttentionCase(io=io, lens=[40, 90], new=[1, 60], D=D, softcap=1e-44)
    assert c.run() == Status.OK
    c.check()


def test_far_softcaps_of_chunks():
    """Far caps take the kernel for few rows, also for many tiles a sequence."""
    for kw in (dict(io="bf16", lens=[700, 40, 300], new=[500, 1, 129]),
               dict(io="f16", cache="e4m3", lens=[2500], new=[40], window=300),
               dict(io="f16", layout="vllm", lens=[90, 400], new=[90, 200])):
        c = AttentionCase(D=64, softcap=1e4, H=2, G=4, **kw)
        c.cap_rel = 2.0 ** -20
        assert c.run() == Status.OK
        c.check()
        size = paged.attention_workspace_size(c.cache, c.q_dev, c.table, c.lens_t, c.indptr,
                                              max_seq_len=max(c.lens), max_query_len=max(c.new),
                                              k_scale=c.kv_scales[0], v_scale=c.kv_scales[1])
        w = torch.empty(size, dtype=torch.uint8, device="cuda")
        assert c.run(workspace=w) == Status.OK
        c.check()


@pytest.mark.parametrize("io,cache,scales", [("f16", None, "tensor"), ("f16", "e4m3", "tensor"),
                                             ("f16", "e4m3", "block"), ("bf16", None, "tensor"),
                                             ("f32", None, "tensor")])
@pytest.mark.parametrize("kind", ["decode", "chunks"])
def test_many_small_weights_beside_one(io, cache, scales, kind):
    """Token 0 has a weight of 1 and a value of 0, all others weights of e^-17.75
    (2^-25.6) and values of 1: of n tokens out = (n - 1) e^-17.75 / (1 + (n - 1)
    e^-17.75).  All sequences share the pages.  Off by the rounding of the
    weights and of the output, and by F32 sums of n equal terms."""
    S, n, m = (128, 8192, 1) if kind == "decode" else (16, 32768, 128)
    H, G, D, bs = 8, 4, 64, 16
    if io == "f32" and kind == "chunks":
        S, n = 4, 8192
    nb = n // bs
    cdt = DT[cache or io]
    k = torch.zeros((nb, bs, H, D), dtype=torch.float32)
    k[0, 0, :, 0] = 1.0
    v = torch.ones((nb, bs, H, D), dtype=torch.float32)
    v[0, 0] = 0.0
    kv = paged.PagedCache(k.to(cdt).cuda(), v.to(cdt).cuda(), Layout.BLOCK_NHD, Layout.BLOCK_NHD,
                          nb, bs, H, D)
    q = torch.zeros((S * m, H * G, D), dtype=DT[io], device="cuda")
    q[..., 0] = 17.75
    out = torch.empty_like(q)
    lse = torch.empty((S * m, H * G), dtype=torch.float32, device="cuda")
    table = torch.arange(nb, dtype=torch.int32, device="cuda").expand(S, nb).contiguous()
    lens = torch.full((S,), n, dtype=torch.int32, device="cuda")
    indptr = None if m == 1 else torch.arange(S + 1, dtype=torch.int32, device="cuda") * m
    one = None
    if cache:
        one = scale_arg(torch.ones(1 if scales == "tensor" else nb, device="cuda"), scales)
    assert paged.attention(kv, q, out, table, lens, indptr, scale=1.0, lse=lse, max_seq_len=n,
                           max_query_len=m, k_scale=one, v_scale=one) == Status.OK
    torch.cuda.synchronize()
    others = torch.arange(n - m, n, dtype=torch.float64).repeat(S)  # each row's tokens but one
    w = math.exp(-17.75)
    want = (others * w / (1 + others * w))[:, None, None]
    half = torch.finfo(DT[io]).eps / 2
    tol = (2 * half + (n + 100) * 2.0 ** -24 + 2 * 17.75 * 2.0 ** -23) * want
    assert ((out.cpu().double() - want).abs() <= tol).all()
    want_l = 17.75 + torch.log1p(others * w)[:, None]
    assert ((lse.cpu().double() - want_l).abs() <= (n + 100) * 2.0 ** -24 + 4 * 17.75 * 2.0 ** -24).all()


@pytest.mark.parametrize("io,cache,D", [("f16", None, 64), ("f16", "e4m3", 64), ("bf16", None, 128),
                                        ("f32", None, 64), ("f16", None, 20)])
@pytest.mark.parametrize("new", [None, [60, 3]])
@pytest.mark.parametrize("scale", [1e3, 5e4, 3e5])
def test_logits_past_the_digits_of_f32(io, cache, D, new, scale):
    """Logits so large that F32 does not tell neighbours apart: the weights stay
    in their type's range.  One token's logit is far above the others': every row
    that sees it has its value, the rounding of weight and output aside.  F16
    weights hold out to logits of 9e7 (2^27 in units of log2, whose rounding is 2^3),
    others to 1e9 (2^31)."""
    if io == "f16" and D != 20:
        scale = min(scale, 5e4)
    c = AttentionCase(io=io, cache=cache, lens=[130, 90], new=new, H=2, G=4, D=D, scale=scale)
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    assert torch.isfinite(c.out.double()).all() and torch.isfinite(c.lse).all()
    for s in range(2):
        b = int(c.tb[s, 1])
        c.rows[0][b, 3, :, 0] = 400.0 if cache is None else 448.0
    c.q[..., 0] = 3.0 + torch.rand(c.q.shape[:-1]).to(c.q.dtype)
    c.q_dev.copy_(c.q)
    set_rows(c.cache.key_cache, c.cache.k_layout, c.rows[0])
    if cache:
        c.kv_scales[0].values.fill_(0.9)
        c.rows[0][...] = (c.rows[0].float() / 448).to(c.rows[0].dtype)
        for s in range(2):
            c.rows[0][int(c.tb[s, 1]), 3, :, 0] = 448.0
        set_rows(c.cache.key_cache, c.cache.k_layout, c.rows[0])
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    out, row = c.out.cpu().double(), 0
    half = torch.finfo(DT[io]).eps / 2
    for s, (n, m) in enumerate(zip(c.lens, c.new)):
        v = c.exact[1][int(c.tb[s, 1]), 3].repeat_interleave(c.G, 0)
        for i in range(m):
            if n - m + i >= 19:
                assert ((out[row] - v).abs() <= 4 * half * v.abs() + 2.0 ** -24).all()
            row += 1
