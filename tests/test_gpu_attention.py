"""Attention over a paged cache (paged.attention, kvx_launch_attention)
against its definition in 64 bits, at the sizes and masks where it can go
wrong.  Bounds: operator_helpers.attention_reference."""
import ctypes as C
import math

import pytest
import torch

from kvx_amd import abi, paged
from kvx_amd.abi import Status

from operator_helpers import AttentionCase, DT, set_rows

pytestmark = pytest.mark.gpu


def go(**kw):
    c = AttentionCase(**kw)
    assert c.run() == Status.OK
    c.check()
    return c


@pytest.mark.parametrize("layout", ["nhd", "hnd", "packed", "packed_k", "vllm", "dim_outer",
                                    "block_inner"])
@pytest.mark.parametrize("io,cache", [("bf16", None), ("f16", None), ("f32", None),
                                      ("bf16", "e4m3"), ("f16", "e4m3"), ("f32", "e4m3"),
                                      ("bf16", "e5m2"), ("f16", "e5m2")])
def test_decode_types_and_layouts(io, cache, layout):
    go(io=io, cache=cache, layout=layout, lens=[1, 15, 16, 17, 100, 333], H=2, G=4, D=64)


@pytest.mark.parametrize("layout", ["nhd", "hnd", "packed", "packed_k", "vllm", "dim_outer"])
@pytest.mark.parametrize("io,cache", [("bf16", None), ("f16", None), ("f32", None),
                                      ("bf16", "e4m3"), ("f16", "e5m2")])
def test_chunk_types_and_layouts(io, cache, layout):
    go(io=io, cache=cache, layout=layout, lens=[70, 1, 131, 200], new=[70, 1, 33, 5], H=2, G=3,
       D=64)


@pytest.mark.parametrize("table", ["packed", "ragged", "offsets"])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("new", [None, [3, 1, 60, 0, 2]])
def test_tables(table, index, new):
    go(table=table, index=index, lens=[50, 129, 64, 9, 300], new=new, D=128)


@pytest.mark.parametrize("bs", [1, 2, 4, 8, 16, 24, 32, 64, 128, 256])
@pytest.mark.parametrize("layout", ["nhd", "hnd", "vllm"])
def test_block_sizes(bs, layout):
    go(bs=bs, layout=layout, lens=[1, 77, 260], new=[1, 40, 2], D=64)
    go(bs=bs, layout=layout, lens=[90, 257], D=128, io="f16")


@pytest.mark.parametrize("D", [1, 8, 16, 17, 32, 40, 64, 72, 80, 96, 100, 112, 128, 192, 256, 264,
                               512])
@pytest.mark.parametrize("io,cache", [("bf16", None), ("f32", None), ("f16", "e4m3")])
def test_head_dims(D, io, cache):
    go(io=io, cache=cache, D=D, lens=[5, 130], H=2, G=2)
    go(io=io, cache=cache, D=D, lens=[90, 40], new=[50, 3], H=2, G=2)


@pytest.mark.parametrize("H,G", [(1, 1), (3, 1), (1, 2), (2, 5), (1, 7), (1, 8), (2, 16), (1, 17),
                                 (1, 32), (1, 71), (1, 130)])
@pytest.mark.parametrize("new", [None, [1, 6, 37]])
def test_head_groups(H, G, new):
    go(H=H, G=G, lens=[3, 66, 140], new=new, D=64)


@pytest.mark.parametrize("scales", ["tensor", "head", "block", "block_head"])
@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("new", [None, [80, 2]])
def test_scales(scales, io, new):
    go(io=io, cache="e4m3", scales=scales, lens=[100, 35], new=new, D=128, H=3)


@pytest.mark.parametrize("new", [None, [40, 3, 1, 30]])
@pytest.mark.parametrize("opts", [dict(causal=False), dict(window=1), dict(window=17),
                                  dict(window=64), dict(window=1000), dict(softcap=2.0),
                                  dict(softcap=30.0, window=50), dict(scale=0.0),
                                  dict(scale=-0.3), dict(causal=False, softcap=5.0)])
def test_masks_and_caps(new, opts):
    go(lens=[100, 64, 1, 290], new=new, D=64, **opts)
    go(lens=[100, 64, 1, 290], new=new, D=64, io="f32", **opts)


def test_long_sequences_split():
    """Contexts long enough that their tokens are split, with lengths from one
    token on beside them."""
    go(lens=[5000, 1, 2049, 640], H=1, G=4, D=128)
    go(lens=[5000, 1, 2049, 640], new=[4, 1, 2, 7], H=1, G=4, D=128, io="f16")
    go(lens=[3000], new=[20], H=1, G=2, D=64, io="f32", window=1500)


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_lengths_of_zero(io):
    """Empty sequences, sequences without new tokens, more new tokens than
    cached ones (their first rows attend to nothing), negative lengths."""
    c = go(io=io, lens=[0, 5, 3, 20, 0], new=[0, 0, 7, 2, 3], D=64)
    assert (c.lse[0:4].cpu() == -math.inf).all() and (c.out[0:4].cpu() == 0).all()
    go(io=io, lens=[0, 1, 0], D=64)
    go(io=io, lens=[-4, 9], D=64)


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_rows_behind_the_last_sequence(io):
    go(io=io, lens=[40, 30], new=[3, 20], extra_rows=9, D=64)


@pytest.mark.parametrize("io,cache", [("bf16", None), ("f16", "e4m3"), ("f32", None)])
@pytest.mark.parametrize("table", ["packed", "ragged", "offsets"])
def test_blocks_that_are_not_there(io, cache, table):
    """Negative and too large block ids: their tokens are not attended to,
    whole sequences of them give zero rows."""
    go(io=io, cache=cache, table=table, lens=[70, 33, 16, 200], D=64,
       holes=[(0, 1), (1, 2), (2, 0), (3, 0), (3, 5), (3, 12)])
    go(io=io, cache=cache, table=table, lens=[70, 33, 16, 200], new=[20, 2, 4, 90], D=64,
       holes=[(0, 1), (1, 2), (2, 0), (3, 0), (3, 5), (3, 12)])


@pytest.mark.parametrize("layout", ["nhd", "vllm"])
@pytest.mark.parametrize("io,cache,D", [("bf16", None, 128), ("f16", "e4m3", 64), ("f32", None, 64),
                                        ("f32", "e5m2", 80), ("bf16", None, 256)])
@pytest.mark.parametrize("share", [0.0, 0.1, 1.0])
def test_ragged_tables_whose_tokens_lie_apart(io, cache, D, layout, share):
    """A RAGGED table names each token's block: `share` of them are moved to
    other blocks, or to none, so that neighbours lie apart."""
    c = AttentionCase(io=io, cache=cache, layout=layout, table="ragged", lens=[70, 5, 200, 131],
                      new=[1, 2, 70, 40], D=D, H=2, G=2)
    ids = c.table.indices.cpu().clone()
    g = torch.Generator().manual_seed(5)
    moved = torch.rand(ids.shape, generator=g) < share
    ids[moved] = torch.randint(-1, c.nb + 1, ids.shape, generator=g).to(ids.dtype)[moved]
    c.table = paged.RaggedTable(ids.to("cuda"), c.table.indptr)
    ptr = c.table.indptr.tolist()

    def rows_of(s):
        b = ids[ptr[s]: ptr[s + 1]].long()
        o = torch.arange(b.numel()) % c.bs
        there = (b >= 0) & (b < c.nb)
        b = b.clamp(0, c.nb - 1)
        return c.exact[0][b, o], c.exact[1][b, o], there

    c.rows_of = rows_of
    assert c.run() == Status.OK
    c.check()


def test_lengths_past_the_table():
    """A length beyond what the table holds: the missing tokens are not
    attended to, positions count from the length."""
    c = AttentionCase(lens=[64, 48], new=[2, 2], D=64, window=40)
    c.lens_t += 10
    assert c.run() == Status.OK
    c2 = c.lens
    c.lens = [64, 48]

    def rows_of(s):
        n = [64, 64][s]
        b = c.tb[s].repeat_interleave(16)[:n]
        there = (b >= 0) & (b < c.nb)
        b = b.clamp(0, c.nb - 1)
        o = torch.arange(n) % 16
        return c.exact[0][b, o], c.exact[1][b, o], there

    c.rows_of = rows_of
    c.lens = [n + 10 for n in c2]
    c.check()


@pytest.mark.parametrize("stale", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("layout", ["nhd", "vllm", "packed"])
@pytest.mark.parametrize("io,cache", [("bf16", None), ("f32", None), ("f16", "e5m2")])
def test_stale_slots_do_not_matter(stale, layout, io, cache):
    """Slots behind a sequence's last token, and pages of nobody, hold NaN and
    infinities."""
    go(io=io, cache=cache, layout=layout, lens=[1, 17, 95], stale=stale, D=64)
    go(io=io, cache=cache, layout=layout, lens=[18, 17, 95], new=[18, 2, 50], stale=stale, D=64)


@pytest.mark.parametrize("io", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_masked_tokens_do_not_reach_rows(io, bad):
    """NaN or infinite keys and values of a token: rows that see it turn NaN
    or infinite, the others stay what they are."""
    c = AttentionCase(io=io, lens=[60, 90], new=[40, 6], D=64, window=30)
    spoiled = 50  # of sequence 0; rows at positions 50..59 see it
    b = int(c.tb[0, spoiled // 16])
    v = c.rows[1].clone()
    v[b, spoiled % 16] = bad
    set_rows(c.cache.value_cache, c.cache.v_layout, v)
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    out = c.out.cpu()
    first = spoiled - 20
    assert not torch.isfinite(out[first:40].double()).any()
    c.out[first:40] = c.reference()[0][first:40].to(DT[io]).cuda()
    c.check()
    # a key: every logit of it is NaN or infinite
    c = AttentionCase(io=io, lens=[60, 90], new=[40, 6], D=64, window=30)
    k = c.rows[0].clone()
    k[b, spoiled % 16] = float("nan")
    set_rows(c.cache.key_cache, c.cache.k_layout, k)
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    assert torch.isnan(c.out[first:40].double()).all() and torch.isnan(c.lse[first:40]).all()
    ref = c.reference()
    c.out[first:40] = ref[0][first:40].to(DT[io]).cuda()
    c.lse[first:40] = ref[1][first:40].float().cuda()
    c.check()


@pytest.mark.parametrize("io,cache", [("bf16", None), ("f16", None), ("f16", "e5m2"),
                                      ("bf16", "e4m3"), ("f32", None)])
@pytest.mark.parametrize("layout", ["nhd", "vllm"])
@pytest.mark.parametrize("new", [[40, 6], [5, 6]])
@pytest.mark.parametrize("long", [0, 3000])
def test_infinities_of_single_elements(io, cache, layout, new, long):
    """One element of a value infinite (or NaN): that element of the rows that
    see the token, and nothing else; also where tokens are split."""
    bad = float("inf") if cache != "e4m3" else float("nan")
    c = AttentionCase(io=io, cache=cache, layout=layout, lens=[60 + long, 90], new=new, D=64, H=2,
                      G=2)
    want, _, tol, _ = c.reference()
    for s, back, h, d, sign in ((0, 2, 1, 17, 1), (0, 3, 0, 40, -1), (1, 4, 1, 63, 1)):
        t = c.lens[s] - back
        v = c.rows[1][int(c.tb[s, t // 16]), t % 16, h]
        v[d] = sign * bad
        rows = range(sum(new[:s]) + new[s] - back, sum(new[: s + 1]))
        for r in rows:
            for j in range(h * c.G, h * c.G + c.G):
                want[r, j, d] = want[r, j, d] + sign * bad
    set_rows(c.cache.value_cache, c.cache.v_layout, c.rows[1])
    assert c.run() == Status.OK
    torch.cuda.synchronize()
    got = c.out.cpu().double()
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want))
    assert torch.equal(got[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)])
    half = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}[io]
    over = (got - want).abs()[fine] - (tol + half * (want.abs() + tol) + 2.0 ** -25)[fine]
    assert (over <= 0).all()


@pytest.mark.parametrize("io", ["bf16", "f32"])
@pytest.mark.parametrize("new", [None, [50, 3]])
def test_large_logits(io, new):
    """Logits in the thousands: the maximum is taken out before any exp."""
    go(io=io, lens=[80, 40], new=new, D=64, scale=40.0)


def test_strided_queries_and_outputs():
    """Views of one projection's output; outputs with padded heads and rows."""
    for new in (None, [30, 2]):
        for io in ("bf16", "f32"):
            c = AttentionCase(io=io, lens=[50, 77], new=new, D=64)
            Hq = c.H * c.G
            wide = torch.zeros((c.T, Hq + 4, c.D), dtype=DT[io], device="cuda")
            wide[:, 2: 2 + Hq] = c.q_dev
            out = torch.full((c.T, Hq + 1, c.D + 8), 5.0, dtype=DT[io], device="cuda")
            view = out[:, :Hq, : c.D]
            assert c.run(q=wide[:, 2: 2 + Hq], out=view) == Status.OK
            c.check(out=view)
            assert (out[:, Hq:] == 5.0).all() and (out[:, :, c.D:] == 5.0).all()
            # an odd offset: no 16-byte chunks
            odd = torch.zeros(c.q_dev.numel() + 1, dtype=DT[io], device="cuda")[1:].view(
                c.q_dev.shape)
            odd.copy_(c.q_dev)
            c.out.fill_(7.0)
            assert c.run(q=odd, lse=None) == Status.OK
            c.check(lse=False)


@pytest.mark.parametrize("io", ["bf16", "f32"])
def test_padded_and_odd_caches(io):
    """Cache tensors whose strides leave gaps, or whose base is not aligned."""
    for new in (None, [40, 2]):
        c = AttentionCase(io=io, lens=[50, 77], new=new, D=64)
        for pad in (8, 3):
            k = torch.empty((c.nb, 16, c.H, 64 + pad), dtype=DT[io], device="cuda")
            v = torch.empty((c.nb, 16, c.H, 64 + pad), dtype=DT[io], device="cuda")
            cache = paged.PagedCache(k[..., :64], v[..., :64], c.cache.k_layout, c.cache.v_layout,
                                     c.nb, 16, c.H, 64)
            cache.key_cache.copy_(c.rows[0])
            cache.value_cache.copy_(c.rows[1])
            kept, c.cache = c.cache, cache
            c.out.fill_(7.0)
            assert c.run() == Status.OK
            c.check()
            c.cache = kept


def test_offsets_past_32_bits():
    """Blocks beyond 4 GiB of a cache tensor."""
    nb, bs, H, D = 600_000, 16, 4, 64  # 4.9 GB each
    cache = paged.alloc_cache(nb, bs, H, D, torch.bfloat16, "cuda")
    for new in (None, [20, 1]):
        c = AttentionCase(lens=[100, 33], new=new, H=H, D=D)
        tb = torch.where(c.tb >= 0, nb - 1 - c.tb, c.tb)
        for i in range(c.nb):
            cache.key_cache[nb - 1 - i] = c.rows[0][i].cuda()
            cache.value_cache[nb - 1 - i] = c.rows[1][i].cuda()
        c.cache, c.table = cache, tb.to("cuda", torch.int32)
        assert c.run() == Status.OK
        c.check()


@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (64, 4), (1 << 20, 1 << 20)])
def test_hints_do_not_change_the_result(hints):
    c = AttentionCase(lens=[900, 20, 300], new=[130, 1, 9], D=128)
    assert c.run(max_seq_len=hints[0], max_query_len=hints[1]) == Status.OK
    c.check()


def test_same_call_twice_gives_the_same_bits():
    c = AttentionCase(lens=[3000, 700], new=[5, 1], D=128, H=1)
    c.run()
    first = c.out.clone(), c.lse.clone()
    c.out.fill_(7.0)
    c.lse.fill_(7.0)
    c.run()
    assert torch.equal(c.out, first[0]) and torch.equal(c.lse, first[1])


def test_streams_and_workspaces():
    """Two calls at once on streams of their own, each with its workspace, one
    of them allocated by the call."""
    a = AttentionCase(lens=[2500, 40], D=128, H=1, seed=1)
    b = AttentionCase(lens=[30, 3000], D=128, H=1, seed=2)
    size = paged.attention_workspace_size(a.cache, a.q_dev, a.table, a.lens_t, a.indptr,
                                          max_seq_len=2500, max_query_len=1)
    assert size > 0
    ws = torch.empty(size, dtype=torch.uint8, device="cuda")
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(5):
        assert a.run(stream=s1, workspace=ws) == Status.OK
        assert b.run(stream=s2.cuda_stream) == Status.OK
    a.check()
    b.check()
    assert a.run(workspace=ws[: size - 1]) == Status.INVALID_ARGUMENT
    assert a.run(workspace=ws[1:]) == Status.INVALID_ARGUMENT  # not aligned either


@pytest.mark.parametrize("new", [None, [60, 3]])
def test_graph(new):
    """Captured once, replayed with other lengths, queries and tables."""
    c = AttentionCase(lens=[2100, 300], new=new, D=128, H=1)
    c.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert c.run() == Status.OK
    for lens, seed in (([2100, 300], 0), ([700, 61], 5), ([1999, 64], 6)):
        d = AttentionCase(lens=lens, new=new, D=128, H=1, seed=seed, spare=3 + sum(
            -(-n // 16) for n in c.lens) - sum(-(-n // 16) for n in lens))
        assert d.nb == c.nb
        c.cache.key_cache.copy_(d.cache.key_cache)
        c.cache.value_cache.copy_(d.cache.value_cache)
        c.table.fill_(-1)
        c.table[:, : d.table.shape[1]] = d.table
        c.lens_t.copy_(d.lens_t)
        c.q_dev.copy_(d.q_dev)
        c.out.fill_(7.0)
        c.lse.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        d.check(out=c.out, lse=c.lse)
        graph.replay()  # and again after work of the program's own
        d.check(out=c.out, lse=c.lse)


@pytest.mark.parametrize("io,cache", [("bf16", None), ("f16", "e5m2"), ("f32", None)])
def test_graph_of_wide_heads(io, cache):
    """Heads of 256 elements, chunks and decoding sequences: the launch that
    needs the most LDS, captured before any eager call of its kind."""
    c = AttentionCase(io=io, cache=cache, lens=[300, 40, 2000], new=[90, 1, 3], D=256, H=1, G=4)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        assert c.run() == Status.OK
    for _ in range(3):
        c.out.fill_(7.0)
        c.lse.fill_(7.0)
        graph.replay()
        c.check()


@pytest.mark.parametrize("new", [None, [1, 30, 2]])
@pytest.mark.parametrize("share", [1.0, 0.5])
def test_pools_of_known_size(new, share):
    """KV_OFFSETS with `pool_blocks`: entries past a pool's blocks are not
    there."""
    c = AttentionCase(io="bf16", table="offsets", lens=[70, 33, 200], new=new, D=64)
    blocks = max(int(2 * c.nb * share) // 2 * 2, 2)

    def rows_of(s):
        n = c.lens[s]
        b = c.tb[s].repeat_interleave(c.bs)[:n]
        there = (b >= 0) & (2 * b + 1 < blocks)
        o = torch.arange(n) % c.bs
        b = b.clamp(0, c.nb - 1)
        return c.exact[0][b, o], c.exact[1][b, o], there

    c.rows_of = rows_of
    assert c.run(pool_blocks=(blocks, 0)) == Status.OK
    c.check()


@pytest.mark.parametrize("seqs", [1, 7, 9, 200])
@pytest.mark.parametrize("hint", [0, 1])
def test_narrow_heads_of_many_sequences(seqs, hint):
    """Heads that share lines run on one die: any number of sequences, with
    and without the query offsets."""
    lens = [1 + (37 * i) % 90 for i in range(seqs)]
    c = AttentionCase(io="bf16", cache="e4m3", lens=lens, H=3, G=2, D=48, bs=16,
                      new=[1] * seqs if hint else None)
    assert c.run(max_query_len=hint) == Status.OK
    c.check()
    c = AttentionCase(io="f16", lens=lens, H=3, G=2, D=24, new=[1] * seqs if hint else None)
    assert c.run(max_query_len=hint) == Status.OK
    c.check()


def test_more_sequences_than_one_scan():
    """Tiles are numbered over 256 sequences at a time: chunks far behind many
    short or empty ones."""
    new = [(1, 0, 3, 20)[i % 4] for i in range(700)]
    new[650] = 150
    c = AttentionCase(io="bf16", lens=[n + i % 5 for i, n in enumerate(new)], new=new, H=1, G=2,
                      D=64)
    assert c.run() == Status.OK
    c.check()


def test_two_graphs_do_not_share_memory():
    a = AttentionCase(lens=[2500], D=128, H=1, seed=1)
    b = AttentionCase(lens=[2600], D=128, H=1, seed=2)
    graphs = []
    for c in (a, b):
        c.run()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            assert c.run() == Status.OK
        graphs.append(g)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            graphs[0].replay()
        with torch.cuda.stream(s2):
            graphs[1].replay()
        torch.cuda.synchronize()
        a.check()
        b.check()


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("seqs", [255, 257, 1030])
@pytest.mark.parametrize("most", [1, 12])
def test_tiles_of_many_sequences(seqs, most, dtype):
    """However tiles are numbered, also with a hint that is too small."""
    new = [(i * 7 + i // 3) % (most + 1) for i in range(seqs)]
    for hint in (0, most, 1):
        c = AttentionCase(io="bf16", lens=[n + i % 4 for i, n in enumerate(new)], new=new, H=1,
                          G=4, D=32, index=dtype, indptr_dtype=dtype, extra_rows=3)
        assert c.run(max_query_len=hint) == Status.OK
        c.check()


@pytest.mark.parametrize("io,cache", [("bf16", None), ("f32", None), ("f16", "e4m3")])
@pytest.mark.parametrize("new", [None, [7, 1, 90]])
def test_output_in_place_of_the_query(io, cache, new):
    c = AttentionCase(io=io, cache=cache, lens=[3000, 200, 90], new=new, D=64, H=1)
    assert c.run(q=c.q_dev, out=c.q_dev) == Status.OK
    c.check(out=c.q_dev)


@pytest.mark.parametrize("new", [None, [1, 90]])
def test_workspace_size_holds_for_any_alignment(new):
    """The size is asked for with aligned tensors; the call's lie otherwise and
    take other kernels."""
    c = AttentionCase(lens=[5000, 900], new=new, D=128, H=1, G=2)
    size = paged.attention_workspace_size(c.cache, c.q_dev, c.table, c.lens_t, c.indptr,
                                          max_seq_len=5000, max_query_len=max(c.new))
    w = torch.empty(size, dtype=torch.uint8, device="cuda")
    flat = torch.full((c.out.numel() + 1,), 7.0, dtype=c.out.dtype, device="cuda")
    out = flat[1:].view(c.out.shape)
    assert c.run(out=out, workspace=w) == Status.OK
    c.check(out=out)


def test_refused_scales():
    c = AttentionCase(io="bf16", cache="e4m3", lens=[40, 30], D=64)
    good = torch.ones(1, device="cuda")
    for bad in (good.cpu(), good.half(), good.double()):
        for kw in (dict(k_scale=bad, v_scale=good), dict(k_scale=good, v_scale=bad)):
            with pytest.raises(ValueError):
                c.run(**kw)
            with pytest.raises(ValueError):
                x = c.q_dev[:, :2].contiguous()
                i = torch.zeros(2, dtype=torch.int64, device="cuda")
                paged.rope_write_kv(c.cache, None, x, x, i,
                                    paged.Rope(torch.ones(32, device="cuda")), i, **kw)
    assert (c.out == 7.0).all()


def test_refusals_on_device():
    c = AttentionCase(lens=[40, 30], D=64)
    with pytest.raises(ValueError):
        c.run(q=c.q)  # on the CPU
    with pytest.raises(ValueError):
        c.run(lse=c.lse[:, :3])
    with pytest.raises(ValueError):
        paged.attention(c.cache, c.q_dev, c.out, c.table.t(), c.lens_t)
    with pytest.raises(ValueError):
        paged.attention(c.cache, c.q_dev, c.out, c.table, c.lens_t[:1])
    with pytest.raises(ValueError):
        paged.attention(c.cache, c.q_dev, c.out, c.table, c.lens_t,
                        torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert c.run(q=c.q_dev[:, :7], lse=None) == Status.INVALID_ARGUMENT  # out has 8 heads
    assert c.run(q=c.q_dev.half(), out=c.out.half()) == Status.UNSUPPORTED
    assert c.run(out=c.out[:, :1].expand(-1, 8, -1)) == Status.UNSUPPORTED
    assert c.run(window=5, causal=False) == Status.INVALID_ARGUMENT
    assert c.run(softcap=-1.0) == Status.INVALID_ARGUMENT
    assert (c.out == 7.0).all()
    d = abi.AttentionDesc()
    assert abi.load().kvx_launch_attention(None, C.byref(d), None) == Status.INVALID_ARGUMENT
