"""Block copies in the caches of all layers (paged.copy_blocks): bit for bit,
and nothing else changed."""
import pytest
import torch

from kvx_amd import paged
from kvx_amd.abi import Status

from operator_helpers import DT, get_rows, make_cache, raw

pytestmark = pytest.mark.gpu


def fill(t, g):
    raw(t).copy_(torch.randint(0, 100, raw(t).shape, generator=g).to(raw(t).dtype))


def check(caches, pairs, **kw):
    before = [[get_rows(t, l).cpu().clone() for t, l in
               ((c.key_cache, c.k_layout), (c.value_cache, c.v_layout))] for c in caches]
    assert paged.copy_blocks(caches, pairs, **kw) == Status.OK
    torch.cuda.synchronize()
    for c, (k, v) in zip(caches, before):
        for want, t, l in ((k, c.key_cache, c.k_layout), (v, c.value_cache, c.v_layout)):
            src = raw(want).clone()
            for s, d in pairs.tolist():
                if 0 <= s < c.num_blocks and 0 <= d < c.num_blocks:
                    raw(want)[d] = src[s]
            assert torch.equal(raw(want), raw(get_rows(t, l).cpu()))


def some_pairs(nb, n, index, seed=0):
    ids = torch.randperm(nb, generator=torch.Generator().manual_seed(seed))[: 2 * n]
    return ids.view(-1, 2).to("cuda", index)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "packed", "packed_k", "vllm", "dim_outer",
                                    "block_inner"])
@pytest.mark.parametrize("dt", ["bf16", "f32", "e4m3"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_layouts_and_types(layout, dt, index):
    g = torch.Generator().manual_seed(1)
    caches = [make_cache(layout, 40, 16, 2, 64, dt, "cuda") for _ in range(3)]
    for c in caches:
        fill(c.key_cache, g)
        fill(c.value_cache, g)
    pairs = some_pairs(40, 9, index)
    pairs[3, 0] = -1
    pairs[4, 1] = -1
    pairs[5, 0] = 40
    pairs[6, 1] = 1000
    pairs[7, 1] = pairs[7, 0]
    check(caches, pairs)


@pytest.mark.parametrize("H,D,bs,dt", [(3, 17, 5, "bf16"), (1, 1, 1, "e4m3"), (1, 3, 2, "f16"),
                                       (5, 80, 24, "bf16"), (8, 128, 256, "f32"), (1, 2, 1, "f32")])
@pytest.mark.parametrize("layout", ["nhd", "hnd"])
def test_odd_block_sizes(H, D, bs, dt, layout):
    g = torch.Generator().manual_seed(2)
    c = make_cache(layout, 12, bs, H, D, dt, "cuda")
    fill(c.key_cache, g)
    fill(c.value_cache, g)
    check([c], some_pairs(12, 5, torch.int32))


@pytest.mark.parametrize("layers", [1, 47, 48, 49, 97])
def test_many_layers(layers):
    """More tensors than one launch takes, of one storage and of several."""
    g = torch.Generator().manual_seed(3)
    k = torch.empty((layers, 10, 8, 2, 16), dtype=torch.bfloat16, device="cuda")
    v = torch.empty_like(k)
    fill(k, g)
    fill(v, g)
    lay = paged.Layout.BLOCK_NHD
    caches = [paged.PagedCache(k[i], v[i], lay, lay, 10, 8, 2, 16) for i in range(layers)]
    check(caches, some_pairs(10, 4, torch.int64))


def test_caches_of_different_shapes():
    g = torch.Generator().manual_seed(4)
    caches = [make_cache("nhd", 20, 16, 2, 64, "bf16", "cuda"),
              make_cache("hnd", 9, 16, 4, 64, "bf16", "cuda"),  # fewer blocks: some pairs skip
              make_cache("block_inner", 20, 16, 2, 64, "bf16", "cuda"),
              make_cache("vllm", 20, 8, 1, 128, "e4m3", "cuda"),
              make_cache("nhd", 20, 16, 2, 64, "bf16", "cuda")]
    for c in caches:
        fill(c.key_cache, g)
        fill(c.value_cache, g)
    check(caches, some_pairs(20, 10, torch.int32))


def test_paired_pool_views_and_padded_blocks():
    """K and V as alternating blocks of one pool, and blocks with gaps."""
    g = torch.Generator().manual_seed(5)
    pool, kv = paged.alloc_block_pool(12, 16, 2, 64, torch.float16, "cuda")
    fill(pool.key_cache, g)
    check([kv], some_pairs(12, 5, torch.int64))
    check([pool], some_pairs(24, 8, torch.int64))
    k = torch.zeros((12, 16, 2, 70), dtype=torch.bfloat16, device="cuda")
    fill(k, g)
    v = k.clone()
    lay = paged.Layout.BLOCK_NHD
    c = paged.PagedCache(k[..., :64], v[..., :64], lay, lay, 12, 16, 2, 64)
    gaps = k[..., 64:].clone()
    check([c], some_pairs(12, 6, torch.int32))
    assert torch.equal(k[..., 64:], gaps)


def test_many_pairs_and_large_offsets():
    nb = 70_000  # 64 KiB blocks: 4.6 GB a tensor
    c = make_cache("nhd", nb, 32, 8, 128, "bf16", "cuda")
    ids = torch.randperm(nb, generator=torch.Generator().manual_seed(6))[:40].cuda()
    pairs = torch.stack([ids[:20], nb - 1 - torch.arange(20, device="cuda")], 1)
    ids = ids[:20]
    assert not set(ids.tolist()) & set(pairs[:, 1].tolist())
    c.key_cache[ids] = torch.randn((20, 32, 8, 128), device="cuda").bfloat16()
    c.value_cache[ids] = torch.randn((20, 32, 8, 128), device="cuda").bfloat16()
    assert paged.copy_blocks([c], pairs) == Status.OK
    torch.cuda.synchronize()
    for t in (c.key_cache, c.value_cache):
        assert torch.equal(t[pairs[:, 1]], t[ids])
    small = make_cache("nhd", 30_000, 1, 1, 8, "bf16", "cuda")
    fill(small.key_cache, torch.Generator().manual_seed(7))
    fill(small.value_cache, torch.Generator().manual_seed(8))
    check([small], some_pairs(30_000, 15_000, torch.int32))


def test_streams_graph_and_empty():
    g = torch.Generator().manual_seed(9)
    caches = [make_cache("nhd", 20, 16, 2, 64, "bf16", "cuda") for _ in range(2)]
    for c in caches:
        fill(c.key_cache, g)
        fill(c.value_cache, g)
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    check(caches, some_pairs(20, 4, torch.int64), stream=s)
    assert paged.copy_blocks(caches, torch.empty((0, 2), dtype=torch.int64,
                                                 device="cuda")) == Status.OK
    assert paged.copy_blocks([], some_pairs(20, 4, torch.int64)) == Status.OK
    pairs = some_pairs(20, 4, torch.int64)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert paged.copy_blocks(caches, pairs) == Status.OK
    for seed in (3, 4):
        pairs.copy_(some_pairs(20, 4, torch.int64, seed))
        want = [raw(c.key_cache).clone() for c in caches]
        graph.replay()
        torch.cuda.synchronize()
        for c, w in zip(caches, want):
            w[pairs[:, 1]] = w[pairs[:, 0]].clone()
            assert torch.equal(raw(c.key_cache), w)


def test_refusals_on_device():
    c = make_cache("nhd", 8, 16, 2, 64, "bf16", "cuda")
    with pytest.raises(ValueError):
        paged.copy_blocks([c], torch.zeros((2, 2), dtype=torch.int64))
    with pytest.raises(ValueError):
        paged.copy_blocks([c], torch.zeros((2, 3), dtype=torch.int64, device="cuda"))
    with pytest.raises(ValueError):
        paged.copy_blocks([c], torch.zeros((2, 2), dtype=torch.int16, device="cuda"))
    with pytest.raises(ValueError):
        paged.copy_blocks([c], torch.zeros((2, 4), dtype=torch.int64, device="cuda")[:, ::2])
