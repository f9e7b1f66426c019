"""Long contexts whose weights are small beside one, against the definition in
64 bits: an F16 weight below 2^-14 of the largest would lose digits, and one below
2^-25 all of them."""
import math

import pytest
import torch

from kvx_amd import paged
from kvx_amd.abi import Layout, Status

from operator_helpers import DT, scale_arg

pytestmark = pytest.mark.gpu


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
