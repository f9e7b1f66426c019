"""Rotary positions with the paged write (paged.rope_write_kv) against the
rotation in 64 bits.

Bounds.  An angle a is exact to 3 * 2^-53 |a| (its products are rounded to 64
bits: 2^-13 radians at a position of 2^40, where a bound without that term did
not hold), sines and cosines to 4 units of 2^-24 (their f32 value, its rest
term, the magnitude); a product, an
fma and the magnitude's rounding add 3 more, on |x0| + |x1| at most.  The
result is rounded once: half a step of the io type, or through the quotient by
the scale (correctly rounded to f32, 2^-24) half a step of the FP8 type, whose
smallest steps are 2^-10 (E4M3) and 2^-17 (E5M2) halves."""
import math

import pytest
import torch

from kvx_amd import abi, paged
from kvx_amd.abi import Status

from operator_helpers import (DT, HALF, TOP, U32, fp8, get_rows, make_cache, raw, scale_arg,
                              scale_rows)

pytestmark = pytest.mark.gpu
TINY = {"e4m3": 2.0 ** -10, "e5m2": 2.0 ** -17, "f16": 2.0 ** -25, "bf16": 0.0, "f32": 0.0}


class Case:
    def __init__(self, *, io="bf16", cache=None, layout="nhd", T=9, H=2, G=3, D=64, rot=None,
                 inter=False, bs=16, mag=1.0, far=5000, fused=True, scales="tensor",
                 index=torch.int64, query=True, padded=2, seed=0, positions=None, x=None):
        g = torch.Generator().manual_seed(seed)
        self.io, self.cdt = io, cache or io
        self.T, self.H, self.G, self.D = T, H, G, D
        self.rot, self.inter, self.mag = D if rot is None else rot, inter, mag
        nb = -(-T // bs) * 2 + 2
        self.nb, self.bs = nb, bs
        qkv = torch.randn((T, H * (G + 2), D), generator=g).to(DT[io])
        dev = qkv.cuda()
        self.q, self.k, self.v = qkv.split([H * G, H, H], 1)
        parts = dev.split([H * G, H, H], 1)
        self.dev = parts if fused else [p.contiguous() for p in parts]
        self.positions = (torch.randint(0, far, (T,), generator=g) if positions is None
                          else torch.tensor(positions))
        slots = torch.randperm(nb * bs, generator=g)[:T]
        slots[torch.randperm(T, generator=g)[:padded]] = -1
        if 1 < padded < T - 1:
            slots[(slots >= 0).nonzero()[0]] = nb * bs + 3  # past the pool: skipped too
        self.slots = slots
        self.cache = make_cache(layout, nb, bs, H, D, self.cdt, "cuda", x)
        self.before = []
        for t in (self.cache.key_cache, self.cache.value_cache):
            raw(t).copy_(torch.randint(0, 100, raw(t).shape, generator=g).to(raw(t).dtype))
        self.before = [get_rows(self.cache.key_cache, self.cache.k_layout).cpu().clone(),
                       get_rows(self.cache.value_cache, self.cache.v_layout).cpu().clone()]
        self.inv = paged.rope_frequencies(self.rot, 10000.0)[0] if self.rot else torch.zeros(0)
        self.rope = paged.Rope(self.inv.cuda(), inter, mag)
        self.sc = [None, None]
        self.sv = [None, None]
        if self.cdt in TOP:
            shape = {"tensor": (1,), "head": (H,), "block": (nb,), "block_head": (nb, H)}[scales]
            for i in range(2):
                s = (0.5 + torch.rand(shape, generator=g)) * 4.0 / TOP[self.cdt]
                self.sv[i] = scale_rows(s.float(), scales, nb, H)
                self.sc[i] = scale_arg(s.float().cuda(), scales)
        self.index = index
        self.query = query

    def run(self, q_out=None, **kw):
        q, k, v = self.dev
        return paged.rope_write_kv(self.cache, q if self.query else None, k, v,
                                   self.positions.to("cuda", self.index), self.rope,
                                   self.slots.to("cuda", self.index), query_out=q_out,
                                   k_scale=self.sc[0], v_scale=self.sc[1], **kw)

    def rotated(self, x):
        r = self.rot
        x = x.double()
        a = torch.outer(self.positions.double(), self.inv.double())
        c, s = (a.cos() * self.mag)[:, None], (a.sin() * self.mag)[:, None]
        y, tol = x.clone(), torch.zeros_like(x)
        i0, i1 = ((torch.arange(0, r, 2), torch.arange(0, r, 2) + 1) if self.inter
                  else (torch.arange(r // 2), torch.arange(r // 2, r)))
        x0, x1 = x[..., i0], x[..., i1]
        y[..., i0], y[..., i1] = x0 * c - x1 * s, x1 * c + x0 * s
        # one rounding of the angle in the reference, two in the kernel: 2^-53 each
        rel = 8 * U32 + 3 * 2.0 ** -53 * a.abs()[:, None]
        tol[..., i0] = tol[..., i1] = rel * abs(self.mag) * (x0.abs() + x1.abs())
        return y, tol

    def check_rows(self, got, ref, tol, dt):
        tol = tol + HALF[dt] * (ref.abs() + tol) + TINY[dt] + 1e-38
        assert ((got.double() - ref).abs() <= tol).all()

    def check(self, q_out):
        torch.cuda.synchronize()
        if self.query:
            ref, tol = self.rotated(self.q)
            self.check_rows(q_out.cpu(), ref, tol, self.io)
            assert torch.equal(q_out.cpu()[..., self.rot:], self.q[..., self.rot:])
        kept = (self.slots >= 0) & (self.slots < self.nb * self.bs)
        b, o = self.slots[kept] // self.bs, self.slots[kept] % self.bs
        for i, (t, lay, src) in enumerate(((self.cache.key_cache, self.cache.k_layout, self.k),
                                           (self.cache.value_cache, self.cache.v_layout, self.v))):
            ref, tol = self.rotated(src) if i == 0 else (src.double(), torch.zeros(src.shape))
            ref, tol = ref[kept], tol[kept]
            after = get_rows(t, lay).cpu()
            if self.sv[i] is not None:
                s = self.sv[i][b][..., None]
                ref, tol = ref / s, (tol + U32 * ref.abs()) / s
                ref = ref.clamp(-TOP[self.cdt], TOP[self.cdt])
            self.check_rows(raw(after)[b, o].view(after.dtype), ref, tol, self.cdt)
            if i == 1 and self.cdt == self.io:
                assert torch.equal(after[b, o], src[kept])
            rest = torch.ones((self.nb, self.bs), dtype=torch.bool)
            rest[b, o] = False
            assert torch.equal(raw(after)[rest], raw(self.before[i])[rest])


def go(**kw):
    c = Case(**kw)
    q_out = torch.zeros((c.T, c.H * c.G, c.D), dtype=DT[c.io], device="cuda")
    assert c.run(q_out if c.query else None) == Status.OK
    c.check(q_out)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "packed", "packed_k", "vllm", "dim_outer"])
@pytest.mark.parametrize("io,cache", [("bf16", None), ("f16", None), ("f32", None),
                                      ("bf16", "e4m3"), ("f16", "e5m2"), ("f32", "e4m3"),
                                      ("f32", "e5m2")])
@pytest.mark.parametrize("inter", [False, True])
def test_types_and_layouts(io, cache, layout, inter):
    go(io=io, cache=cache, layout=layout, inter=inter, T=21)


@pytest.mark.parametrize("D,rot", [(64, 32), (128, 128), (128, 16), (80, 20), (80, 80), (96, 48),
                                   (256, 64), (17, 16), (17, 2), (1, 0), (72, 0), (100, 100),
                                   (576, 64), (8, 6), (1024, 1024)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_head_and_rotated_dims(D, rot, inter, io):
    go(io=io, D=D, rot=rot, inter=inter, T=7)
    go(io=io, cache="e4m3", D=D, rot=rot, inter=inter, T=3, H=1, G=1, layout="hnd")


@pytest.mark.parametrize("T", [1, 2, 4, 5, 63, 300, 1500, 5000])
@pytest.mark.parametrize("H,G", [(1, 1), (8, 4), (3, 5)])
def test_token_counts(T, H, G):
    go(T=T, H=H, G=G, D=128, far=200000)


@pytest.mark.parametrize("scales", ["tensor", "head", "block", "block_head"])
def test_scales(scales):
    go(io="bf16", cache="e4m3", scales=scales, T=40, H=3)


def test_far_positions():
    """Angles of positions up to 2^31 - 1 and beyond, and negative ones: an
    angle kept in 32 bits would be off by whole radians."""
    go(io="f32", T=6, positions=[0, 1, 1_000_003, 16_777_217, 2 ** 31 - 1, -5], padded=0)
    c = Case(io="bf16", T=3, positions=[2 ** 33 + 1, 2 ** 40 + 3, 7], padded=0)
    q_out = torch.empty_like(c.dev[0])
    assert c.run(q_out) == Status.OK
    c.check(q_out)


def test_magnitude_and_in_place():
    c = Case(mag=1.37, T=33)
    q = c.dev[0]
    assert c.run() == Status.OK  # in place, in the fused projection
    c.check(q)
    c = Case(mag=0.25, T=33, fused=False, inter=True, io="f16")
    assert c.run() == Status.OK
    c.check(c.dev[0])


def test_without_queries_and_index_types():
    go(query=False, T=12)
    go(index=torch.int32, T=12)
    go(T=50, padded=50)  # nothing is written
    go(fused=False, T=12, io="f16")


def test_wide_batch_of_one_head_each():
    go(T=700, H=1, G=1, D=64, rot=32, inter=True)


def test_unaligned_rows():
    c = Case(T=10, D=64)
    flat = torch.zeros(c.T * c.H * c.G * c.D + 1, dtype=torch.bfloat16, device="cuda")
    q = flat[1:].view(c.T, c.H * c.G, c.D)
    q.copy_(c.dev[0])
    c.dev = (q, c.dev[1], c.dev[2])
    out = torch.empty_like(c.dev[0])
    assert c.run(out) == Status.OK
    c.check(out)


def test_same_as_the_write():
    """At position 0, or with nothing rotated, the cache gets what write_kv
    writes, bit for bit, FP8 codes and NaN and saturation among them."""
    for io, cdt in (("bf16", "bf16"), ("bf16", "e4m3"), ("f16", "e5m2"), ("f32", "e4m3")):
        for rot in (0, 64):
            c = Case(io=io, cache=cdt, T=30, positions=[0] * 30, rot=rot, fused=False, layout="hnd")
            for t in c.dev[1:]:
                t[3, 0, :4] = torch.tensor([float("nan"), float("inf"), -float("inf"), 6e4])
            other = make_cache("hnd", c.nb, c.bs, c.H, c.D, c.cdt, "cuda")
            raw(other.key_cache).copy_(raw(c.cache.key_cache))
            raw(other.value_cache).copy_(raw(c.cache.value_cache))
            slots = c.slots.cuda()
            assert paged.write_kv(other, c.dev[1], c.dev[2], slots, k_scale=c.sc[0],
                                  v_scale=c.sc[1]) == Status.OK
            # an infinite element turns its pair into NaN: compare without it
            if rot:
                for t in (c.dev[1],):
                    t[3, 0, :4] = 0
                assert paged.write_kv(other, c.dev[1], c.dev[2], slots, k_scale=c.sc[0],
                                      v_scale=c.sc[1]) == Status.OK
            assert c.run(torch.empty_like(c.dev[0])) == Status.OK
            torch.cuda.synchronize()
            same = lambda a, b: torch.equal(a.view(torch.uint8), b.view(torch.uint8))  # noqa: E731
            if io == cdt:  # a NaN's payload is not kept by a rotation's rounding
                same = lambda a, b: torch.equal(torch.nan_to_num(a.float(), 9.0),  # noqa: E731
                                                torch.nan_to_num(b.float(), 9.0))
            assert same(other.key_cache, c.cache.key_cache)
            assert same(other.value_cache, c.cache.value_cache)


def test_graph():
    c = Case(T=64, H=8, G=4, D=128)
    out = torch.zeros((c.T, 32, 128), dtype=torch.bfloat16, device="cuda")
    pos, slots = c.positions.cuda(), c.slots.cuda()

    def call():
        return paged.rope_write_kv(c.cache, *c.dev, pos, c.rope, slots, query_out=out)

    assert call() == Status.OK
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert call() == Status.OK
    for shift in (0, 17, 400):
        c.positions = (c.positions + shift) % 90000
        pos.copy_(c.positions)
        out.zero_()
        graph.replay()
        c.check(out)


def test_refusals_on_device():
    c = Case(T=10)
    q, k, v = c.dev
    pos, slots = c.positions.cuda(), c.slots.cuda()
    call = lambda *a, **kw: paged.rope_write_kv(c.cache, *a, **kw)  # noqa: E731
    out = torch.zeros((c.T, c.H * c.G, c.D), dtype=q.dtype, device="cuda")
    with pytest.raises(ValueError):
        call(q, k, v, c.positions, c.rope, slots, query_out=out)
    with pytest.raises(ValueError):
        call(q, k, v, pos[:5], c.rope, slots, query_out=out)
    with pytest.raises(ValueError):
        call(q, k, v, pos, paged.Rope(c.inv.double().cuda()), slots, query_out=out)
    assert call(q[:5], k, v, pos, c.rope, slots, query_out=out) == Status.INVALID_ARGUMENT
    assert call(q.half(), k, v, pos, c.rope, slots, query_out=out) == Status.UNSUPPORTED
    assert call(q, k, v, pos, paged.Rope(torch.ones(33, device="cuda")), slots,
                query_out=out) == Status.INVALID_ARGUMENT  # rot_dim 66 > 64
    assert call(q, k, v, pos, c.rope, slots,
                query_out=out[:, :1].expand(-1, 6, -1)) == Status.UNSUPPORTED
    assert call(q[..., ::2], k, v, pos, c.rope, slots, query_out=out) == Status.INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert (out == 0).all()
