"""rope_write_kv, attention and copy_blocks together, as a server runs them: a
prefill of two sequences in every layer, a fork whose last page is copied, and
decode steps of all three, eagerly and as one captured graph.

Bounds.  A rotated row differs from the exact one by at most e = 16 * 2^-24 of
its length (8 * 2^-24 (|x0| + |x1|) for both elements of a pair), and by u more
where it is rounded to 16 bits.  A logit is then off by 2 (e + u) |q| |k| scale
beside the bound of attention_reference, a weight by twice that, relative, and
the output by that times the largest value."""
import pytest
import torch

from kvx_amd import paged
from kvx_amd.abi import Status

from operator_helpers import DT, HALF, U32, attention_reference, make_cache

pytestmark = pytest.mark.gpu

H, G, D, BS, BLOCKS, LAYERS = 2, 3, 64, 16, 12, 2


class Server:
    def __init__(self, io, layout):
        self.io, self.gen = io, torch.Generator().manual_seed(3)
        self.caches = [make_cache(layout, BLOCKS, BS, H, D, io, "cuda") for _ in range(LAYERS)]
        for c in self.caches:  # pages of a pool hold whatever was there
            c.key_cache.fill_(float("nan"))
            c.value_cache.fill_(float("nan"))
        inv, _ = paged.rope_frequencies(D, 10000.0)
        self.inv = inv.double()
        self.rope = paged.Rope(inv.cuda())
        self.free = list(range(BLOCKS - 1, -1, -1))
        self.pages, self.keys, self.values = {}, {}, {}

    def start(self, name):
        self.pages[name] = []
        self.keys[name] = [torch.zeros((0, H, D))] * LAYERS
        self.values[name] = [torch.zeros((0, H, D))] * LAYERS

    def length(self, name):
        return self.keys[name][0].shape[0]

    def fork(self, name, other):
        """`other` shares all pages of `name` but the last, which is copied."""
        last, new = self.pages[name][-1], self.free.pop()
        pairs = torch.tensor([[last, new], [-1, -1]], dtype=torch.int32, device="cuda")
        assert paged.copy_blocks(self.caches, pairs) == Status.OK
        self.pages[other] = self.pages[name][:-1] + [new]
        self.keys[other], self.values[other] = list(self.keys[name]), list(self.values[name])

    def batch(self, names, new):
        """Host-side plan of a step: pages for the new tokens, slots, positions."""
        slots, positions = [], []
        for s, n in zip(names, new):
            for p in range(self.length(s), self.length(s) + n):
                if p // BS == len(self.pages[s]):
                    self.pages[s].append(self.free.pop())
                slots.append(self.pages[s][p // BS] * BS + p % BS)
                positions.append(p)
        table = torch.full((len(names), 4), -1, dtype=torch.int32)
        for i, s in enumerate(names):
            table[i, : len(self.pages[s])] = torch.tensor(self.pages[s], dtype=torch.int32)
        lens = torch.tensor([self.length(s) + n for s, n in zip(names, new)], dtype=torch.int32)
        ptr = torch.tensor([0] + list(new), dtype=torch.int32).cumsum(0).int()
        qkv = torch.randn((LAYERS, sum(new), H * (G + 2), D), generator=self.gen).to(DT[self.io])
        at = 0
        for s, n in zip(names, new):
            for l in range(LAYERS):
                k, v = qkv[l, at: at + n, H * G: H * G + H], qkv[l, at: at + n, H * G + H:]
                self.keys[s][l] = torch.cat([self.keys[s][l], k.float()])
                self.values[s][l] = torch.cat([self.values[s][l], v.float()])
            at += n
        return dict(slots=torch.tensor(slots), positions=torch.tensor(positions), table=table,
                    lens=lens, ptr=ptr, qkv=qkv)

    def layers(self, b, out, decode):
        """The step's kernels, on device tensors."""
        for l, cache in enumerate(self.caches):
            q, k, v = b["qkv"][l].split([H * G, H, H], 1)
            assert paged.rope_write_kv(cache, q, k, v, b["positions"], self.rope,
                                       b["slots"]) == Status.OK
            assert paged.attention(cache, q, out[l], b["table"], b["lens"],
                                   None if decode else b["ptr"]) == Status.OK

    def turned(self, x, first):
        a = torch.outer(torch.arange(first, first + x.shape[0]).double(), self.inv)
        c, s = a.cos()[:, None], a.sin()[:, None]
        x = x.double()
        x0, x1 = x[..., : D // 2], x[..., D // 2:]
        return torch.cat([x0 * c - x1 * s, x1 * c + x0 * s], -1)

    def check(self, names, new, b, out):
        torch.cuda.synchronize()
        u = HALF[self.io] if self.io != "f32" else 0.0
        scale = D ** -0.5
        for l in range(LAYERS):
            at = 0
            for s, n in zip(names, new):
                length = self.length(s)
                k, v = self.turned(self.keys[s][l], 0), self.values[s][l].double()
                q = self.turned(b["qkv"][l, at: at + n, : H * G], length - n)
                ref, _, tol, _ = attention_reference(
                    q, lambda _: (k, v, torch.ones(length, dtype=torch.bool)), [length], [n], G,
                    scale=scale, u_p=u)
                logit = 2 * (16 * U32 + u) * scale * q.norm(dim=-1) * k.norm(dim=-1).max()
                tol = tol + 2 * logit[..., None] * v.abs().max()
                tol = tol + HALF[self.io] * (ref.abs() + tol)
                got = out[l, at: at + n].cpu().double()
                assert ((got - ref).abs() <= tol).all(), (l, s)
                at += n


@pytest.mark.parametrize("io", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("layout", ["nhd", "packed_k", "vllm"])
@pytest.mark.parametrize("graph", [False, True])
def test_prefill_fork_and_decode(io, layout, graph):
    m = Server(io, layout)
    m.start("a")
    m.start("b")

    def device(b):
        return {k: v.cuda() for k, v in b.items()}

    names, new = ["a", "b"], [37, 20]
    b = m.batch(names, new)
    out = torch.full((LAYERS, 57, H * G, D), 7.0, dtype=DT[io], device="cuda")
    m.layers(device(b), out, decode=False)
    m.check(names, new, b, out)

    m.fork("a", "c")
    names, new = ["a", "b", "c"], [1, 1, 1]
    out = torch.full((LAYERS, 3, H * G, D), 7.0, dtype=DT[io], device="cuda")
    held = replay = None
    for step in range(13):  # b fills a page on the way, a and c theirs
        b = m.batch(names, new)
        if not graph:
            m.layers(device(b), out, decode=True)
        elif replay is None:
            held = device(b)
            m.layers(held, out, decode=True)  # eagerly first
            m.check(names, new, b, out)
            for t, x in b.items():
                held[t].copy_(x)  # rotated in place
            torch.cuda.synchronize()
            replay = torch.cuda.CUDAGraph()
            with torch.cuda.graph(replay):
                m.layers(held, out, decode=True)
            replay.replay()
        else:
            for t, x in b.items():
                held[t].copy_(x)
            out.fill_(7.0)
            replay.replay()
        m.check(names, new, b, out)
    # a chunk of one sequence beside decoding ones
    names, new = ["b", "a", "c"], [11, 1, 2]
    b = m.batch(names, new)
    out = torch.full((LAYERS, 14, H * G, D), 7.0, dtype=DT[io], device="cuda")
    m.layers(device(b), out, decode=False)
    m.check(names, new, b, out)
