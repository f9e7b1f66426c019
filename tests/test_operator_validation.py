"""Refusals of kvx_ext.h's operators, and the rotary frequencies (CPU only):
every malformed call returns its code before any HIP call is made."""
import ctypes as C
import math

import pytest
import torch

from kvx_amd import abi, paged
from kvx_amd.abi import DType, Layout, Memory, ScaleGranularity, Status, TableFormat

FAKE = 0x10000  # never dereferenced
DEV = Memory.DEVICE
OK, INV, UNS = Status.OK, Status.INVALID_ARGUMENT, Status.UNSUPPORTED


def cache(dt=DType.BF16, nb=8, bs=16, H=2, D=64, layout=Layout.BLOCK_NHD, mem=DEV):
    return abi.make_cache(layout, dt, mem, nb, bs, H, D, FAKE, FAKE)


def rows(dt, T, H, D, data=FAKE, stride=None, mem=DEV):
    t = abi.token_tensor(dt, mem, T, H, D, data)
    for i, s in enumerate(stride or ()):
        t.stride[i] = s
    return t


def attn(T=3, Hq=4, D=64, dt=DType.BF16, S=3, mbps=4, indptr=None, **kw):
    a = abi.AttentionDesc()
    a.size = C.sizeof(a)
    a.flags = abi.ATTENTION_CAUSAL
    a.query = rows(dt, T, Hq, D)
    a.out = rows(dt, T, Hq, D, FAKE + 4096)
    a.block_table = abi.make_block_table_packed(S, mbps, DType.S32, FAKE)
    a.seq_lens = abi.make_seq_lens(S, DType.S32, FAKE)
    a.scale = 0.125
    if indptr:
        a.query_indptr = FAKE
        a.query_indptr_dtype = indptr
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def A(lib, c, a):
    """Both entry points refuse alike; the launch without being reached when
    the arguments hold (a workspace of 0 bytes, or none, stops it)."""
    size = C.c_uint64(77)
    st = Status(lib.kvx_attention_workspace_size(abi.ref(c), abi.ref(a), C.byref(size)))
    if st != OK:
        assert Status(lib.kvx_launch_attention(abi.ref(c), abi.ref(a), None)) == st
    return st


def test_attention_arguments(kvx_lib):
    L = kvx_lib
    assert A(L, cache(), attn()) == OK
    assert A(L, None, attn()) == INV
    assert A(L, cache(), None) == INV
    assert L.kvx_attention_workspace_size(abi.ref(cache()), abi.ref(attn()), None) == INV
    for field, v in (("size", 8), ("flags", 6), ("softcap", -1.0), ("softcap", math.nan),
                     ("window", 0x80000000), ("max_seq_len", 0xFFFFFFFF)):
        assert A(L, cache(), attn(**{field: v})) == INV, field
    assert A(L, cache(), attn(flags=0, window=4)) == INV
    assert A(L, cache(), attn(flags=0)) == OK
    assert A(L, cache(), attn(window=4)) == OK
    # heads, dims, rows
    assert A(L, cache(), attn(Hq=5)) == INV
    assert A(L, cache(), attn(Hq=0)) == OK
    assert A(L, cache(), attn(D=32)) == INV
    assert A(L, cache(D=520), attn(D=520)) == UNS
    assert A(L, cache(D=512), attn(D=512)) == OK
    assert A(L, cache(), attn(T=4)) == INV               # no row numbers: one row each
    assert A(L, cache(), attn(T=4, indptr=DType.S64)) == OK
    assert A(L, cache(), attn(T=4, indptr=DType.F32)) == INV
    assert A(L, cache(), attn(T=0, S=0)) == OK
    # dtypes
    assert A(L, cache(), attn(dt=DType.F16)) == UNS
    assert A(L, cache(DType.S32), attn()) == UNS
    assert A(L, cache(DType.F8_E4M3), attn()) == INV      # no scales
    a = attn()
    a.out.dtype = DType.F16
    assert A(L, cache(), a) == UNS
    # host memory, tensor shapes and strides
    assert A(L, cache(mem=Memory.HOST), attn()) == INV
    assert A(L, cache(), attn(query=rows(DType.BF16, 3, 4, 64, mem=Memory.HOST))) == INV
    assert A(L, cache(), attn(out=rows(DType.BF16, 2, 4, 64))) == INV
    assert A(L, cache(), attn(query=rows(DType.BF16, 3, 4, 64, stride=(256, 64, 2)))) == UNS
    assert A(L, cache(), attn(query=rows(DType.BF16, 3, 4, 64, stride=(0, 0, 1)))) == OK
    assert A(L, cache(), attn(out=rows(DType.BF16, 3, 4, 64, stride=(256, 0, 1)))) == UNS
    assert A(L, cache(), attn(out=rows(DType.BF16, 3, 4, 64, stride=(64, 64, 1)))) == UNS
    assert A(L, cache(), attn(out=rows(DType.BF16, 3, 4, 64, stride=(64, 192, 1)))) == OK
    a = attn()
    a.query.ndim = 4
    assert A(L, cache(), a) == INV
    # cache
    c = cache()
    c.block_size = 0
    assert A(L, c, attn()) == INV
    c = cache()
    c.v.dtype = DType.F16
    assert A(L, c, attn()) == INV
    c = cache()
    c.k.layout = 9
    assert A(L, c, attn()) == UNS


def test_attention_softcap_is_finite(kvx_lib):
    assert A(kvx_lib, cache(), attn(softcap=math.inf)) == INV
    assert A(kvx_lib, cache(), attn(softcap=3e38)) == OK


def test_attention_tables(kvx_lib):
    L = kvx_lib
    a = attn()
    a.block_table.format = 9
    assert A(L, cache(), a) == UNS
    a = attn()
    a.block_table.size = 4
    assert A(L, cache(), a) == INV
    a = attn()
    a.seq_lens.seq_count = 2
    assert A(L, cache(), a) == INV
    a = attn()
    a.seq_lens.dtype = DType.S64
    assert A(L, cache(), a) == INV
    a = attn(mbps=1 << 28)
    assert A(L, cache(), a) == UNS                        # 2^32 tokens of one sequence
    # RAGGED
    def ragged(**kw):
        a = attn()
        t = a.block_table
        t.format, t.indptr, t.indptr_dtype = TableFormat.RAGGED, FAKE, DType.S32
        t.indptr_count, t.indices_count = 4, 100
        for k, v in kw.items():
            setattr(t, k, v)
        return a

    assert A(L, cache(), ragged()) == OK
    assert A(L, cache(), ragged(indptr_count=3)) == INV
    assert A(L, cache(), ragged(indptr_dtype=DType.F16)) == INV
    assert Status(L.kvx_launch_attention(abi.ref(cache()), abi.ref(ragged(indptr=None)),
                                         None)) == INV

    # KV_OFFSETS
    def offsets(c=None, **kw):
        c = c or cache()
        c.pool.size = C.sizeof(abi.PoolDesc)
        c.pool.bytes_per_block = 16 * 2 * 64 * 2
        c.pool.primary = FAKE
        a = attn()
        t = a.block_table
        t.format, t.flags, t.indices_count = TableFormat.KV_OFFSETS, 1, 3 * 2 * 4
        for k, v in kw.items():
            setattr(t, k, v)
        return c, a

    assert A(L, *offsets()) == OK
    assert A(L, *offsets(flags=0)) == INV
    assert A(L, *offsets(beam_width=0)) == INV
    assert A(L, *offsets(beam_width=2)) == UNS
    assert A(L, *offsets(indices_count=5)) == INV
    assert A(L, *offsets(index_dtype=DType.S64)) == INV
    assert A(L, *offsets(cache(bs=24))) == INV
    c, a = offsets()
    c.pool.bytes_per_block -= 2
    assert A(L, c, a) == INV
    c, a = offsets()
    pools = abi.PoolBlocks(C.sizeof(abi.PoolBlocks), 0, -1, 0)
    a.pool_blocks = C.pointer(pools)
    assert A(L, c, a) == INV
    pools.primary = 3
    assert A(L, c, a) == OK
    c, a = offsets(cache(DType.F8_E4M3))
    c.pool.bytes_per_block = 16 * 2 * 64
    a.k_scale = abi.scale_desc(FAKE, granularity=ScaleGranularity.PER_BLOCK, shape=(8,))
    a.v_scale = abi.scale_desc(FAKE)
    assert A(L, c, a) == UNS                              # no physical block ids
    a.k_scale = abi.scale_desc(FAKE, granularity=ScaleGranularity.PER_HEAD, shape=(2,))
    assert A(L, c, a) == OK
    a.k_scale.shape[0] = 3
    assert A(L, c, a) == INV


def test_attention_pointers_and_workspace(kvx_lib):
    L = kvx_lib
    launch = lambda c, a: Status(L.kvx_launch_attention(abi.ref(c), abi.ref(a), None))  # noqa: E731
    for null in ("query", "out"):
        a = attn()
        getattr(a, null).data = None
        assert launch(cache(), a) == INV
    a = attn()
    a.seq_lens.lengths = None
    assert launch(cache(), a) == INV
    a = attn()
    a.block_table.indices = None
    assert launch(cache(), a) == INV
    c = cache()
    c.k.data = None
    assert launch(c, attn()) == INV
    # a long sequence is split: the workspace has to be there, whole and aligned
    size = C.c_uint64()
    a = attn(mbps=4096)
    assert L.kvx_attention_workspace_size(abi.ref(cache()), abi.ref(a), C.byref(size)) == OK
    assert size.value > 0
    assert launch(cache(), a) == INV
    a.workspace, a.workspace_size = FAKE, size.value - 1
    assert launch(cache(), a) == INV
    a.workspace, a.workspace_size = FAKE + 4, size.value
    assert launch(cache(), a) == INV
    a.max_seq_len = 1
    assert L.kvx_attention_workspace_size(abi.ref(cache()), abi.ref(a), C.byref(size)) == OK
    assert size.value == 0
    # empty batches launch nothing
    for a in (attn(T=0, S=0), attn(Hq=0), attn(T=0, S=3, indptr=DType.S32)):
        assert launch(cache(), a) == OK


def rope(T=5, Hq=4, D=64, dt=DType.BF16, **kw):
    r = abi.RopeDesc()
    r.size = C.sizeof(r)
    r.rot_dim = D
    r.magnitude = 1.0
    r.position_dtype = DType.S64
    r.positions = FAKE
    r.inv_freq = FAKE
    r.query = rows(dt, T, Hq, D)
    r.query_out = rows(dt, T, Hq, D, FAKE + 8192)
    for k, v in kw.items():
        setattr(r, k, v)
    return r


def write(T=5, H=2, D=64, dt=DType.BF16):
    return abi.make_write(T, H, D, dt, DEV, FAKE, FAKE, DType.S64, FAKE)


def test_rope_arguments(kvx_lib):
    R = lambda c, w, r: Status(kvx_lib.kvx_launch_rope_write_kv(  # noqa: E731
        abi.ref(c), abi.ref(w), abi.ref(r), None))
    assert C.sizeof(abi.RopeDesc) == 264 and C.sizeof(abi.AttentionDesc) == 592
    assert R(cache(), write(0), rope(0)) == OK            # nothing to do
    for args in ((None, write(), rope()), (cache(), None, rope()), (cache(), write(), None)):
        assert R(*args) == INV
    for field, v in (("size", 8), ("style", 2), ("rot_dim", 3), ("rot_dim", 66),
                     ("position_dtype", DType.F32), ("positions", None), ("inv_freq", None)):
        assert R(cache(), write(), rope(**{field: v})) == INV, field
    big = 16384
    assert R(cache(D=big), write(D=big), rope(D=big)) == UNS
    assert R(cache(), write(4), rope()) == INV            # 4 keys, 5 queries
    assert R(cache(), write(), rope(dt=DType.F16)) == UNS
    assert R(cache(DType.F16), write(), rope()) == UNS
    assert R(cache(DType.F8_E4M3), write(), rope()) == INV  # no scale
    assert R(cache(mem=Memory.HOST), write(), rope()) == INV
    w = write()
    w.slots.token_count = 4
    assert R(cache(), w, rope()) == INV
    w = write()
    w.slots.dtype = DType.F32
    assert R(cache(), w, rope()) == INV
    w = write()
    w.slots.slots = None
    assert R(cache(), w, rope()) == INV
    w = write()
    w.io.key.data = None
    assert R(cache(), w, rope()) == INV
    w = write()
    w.io.value.stride[2] = 2
    assert R(cache(), w, rope()) == UNS
    r = rope()
    r.query_out.stride[1] = 0
    assert R(cache(), write(), r) == UNS                  # heads on top of each other
    r = rope()
    r.query_out.shape[1] = 3
    assert R(cache(), write(), r) == INV
    r = rope()
    r.query.data = None
    assert R(cache(), write(), r) == INV
    c = cache()
    c.block_size = 0
    assert R(c, write(), rope()) == INV


def test_copy_blocks_arguments(kvx_lib):
    def K(caches, pairs=FAKE, n=3, dt=DType.S64, count=None):
        arr = (C.POINTER(abi.CacheDesc) * max(1, len(caches)))(
            *[C.pointer(c) if c is not None else None for c in caches])
        return Status(kvx_lib.kvx_launch_copy_blocks(arr, len(caches) if count is None else count,
                                                     pairs, int(dt), n, None))

    assert K([cache()], n=0) == OK
    assert K([]) == OK
    assert Status(kvx_lib.kvx_launch_copy_blocks(None, 1, FAKE, int(DType.S32), 1, None)) == INV
    assert K([cache()], pairs=None) == INV
    assert K([cache()], dt=DType.F32) == INV
    assert K([cache()], n=0xFFFFFFFF) == INV
    assert K([cache(), None]) == INV
    assert K([cache(), cache(mem=Memory.HOST)]) == INV
    assert K([cache(DType.S32)]) == UNS
    c = cache()
    c.k.layout = 9
    assert K([c]) == UNS
    c = cache()
    c.v.data = None
    assert K([c]) == INV
    c = cache()
    c.block_size = 0
    assert K([c]) == INV
    c = cache()
    c.size = 4
    assert K([c]) == INV
    assert K([cache(nb=0)]) == OK


def test_paged_refuses_cpu_tensors():
    c = paged.alloc_cache(4, 16, 2, 64, torch.bfloat16, "cpu")
    q = torch.zeros((1, 4, 64), dtype=torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        paged.attention(c, q, q.clone(), one.view(1, 1), one)
    with pytest.raises(ValueError, match="GPU"):
        paged.rope_write_kv(c, q, q[:, :2], q[:, :2], one, paged.Rope(torch.ones(32)), one)
    with pytest.raises(ValueError, match="GPU"):
        paged.copy_blocks([c], torch.zeros((1, 2), dtype=torch.int32))


def test_workspace_size_of_torch_arguments():
    c = paged.alloc_cache(512, 16, 2, 64, torch.bfloat16, "meta")
    c = paged.PagedCache(torch.empty(8), torch.empty(8), c.k_layout, c.v_layout, 512, 16, 2, 64)
    with pytest.raises(ValueError, match="no attention"):
        paged.attention_workspace_size(c, torch.zeros((1, 4, 64), dtype=torch.bfloat16),
                                       torch.zeros((1, 32), dtype=torch.int32),
                                       torch.zeros(1, dtype=torch.int32))


# ---------------------------------------------------------------------------
# Rotary frequencies against their formulas, in Python floats.

def plain(r, base):
    return [base ** (-2 * i / r) for i in range(r // 2)]


def close(inv, want):
    """inv is want rounded to float32: half a step, and 2^-50 of the sums."""
    assert inv.dtype == torch.float32 and inv.shape == (len(want),)
    for a, b in zip(inv.tolist(), want):
        assert abs(a - b) <= (2.0 ** -24 + 2.0 ** -45) * b


@pytest.mark.parametrize("r,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (20, 100.0)])
def test_frequencies(r, base):
    inv, m = paged.rope_frequencies(r, base)
    close(inv, plain(r, base))
    assert m == 1.0
    inv, m = paged.rope_frequencies(r, base, scaling="linear", factor=4.0)
    close(inv, [f / 4 for f in plain(r, base)])
    if r > 2:
        inv, m = paged.rope_frequencies(r, base, scaling="ntk", factor=4.0)
        close(inv, plain(r, base * 4.0 ** (r / (r - 2))))
        # the slowest pair is slowed by the factor, the fastest kept
        assert inv[0] == 1.0
        assert abs(float(inv[-1]) * 4 / plain(r, base)[-1] - 1) < 1e-6


def test_llama3_frequencies():
    base, r, L = 500000.0, 128, 8192
    inv, m = paged.rope_frequencies(r, base, scaling="llama3", factor=8.0, original_length=L)
    want = []
    for f in plain(r, base):
        wave = 2 * math.pi / f
        if wave < L / 4.0:
            want.append(f)
        elif wave > L / 1.0:
            want.append(f / 8.0)
        else:
            s = (L / wave - 1.0) / (4.0 - 1.0)
            want.append((1 - s) * f / 8.0 + s * f)
    close(inv, want)
    assert m == 1.0 and want[0] == 1.0 and want[-1] == plain(r, base)[-1] / 8


def test_yarn_frequencies():
    base, r, L, factor = 10000.0, 64, 4096, 16.0
    inv, m = paged.rope_frequencies(r, base, scaling="yarn", factor=factor, original_length=L)
    at = lambda turns: r * math.log(L / (turns * 2 * math.pi)) / (2 * math.log(base))  # noqa: E731
    low, high = max(math.floor(at(32)), 0), min(math.ceil(at(1)), r - 1)
    want = []
    for i, f in enumerate(plain(r, base)):
        slow = min(max((i - low) / (high - low), 0.0), 1.0)
        want.append(slow * f / factor + (1 - slow) * f)
    close(inv, want)
    assert m == 0.1 * math.log(factor) + 1.0
    assert paged.rope_frequencies(r, base, scaling="yarn", factor=1.0, original_length=L)[1] == 1.0
    assert paged.rope_frequencies(r, base, scaling="yarn", factor=16.0, original_length=L,
                                  magnitude=1.25)[1] == 1.25


def test_frequency_refusals():
    for kw in (dict(rot_dim=3), dict(rot_dim=0), dict(rot_dim=8, base=1.0),
               dict(rot_dim=8, base=math.nan), dict(rot_dim=8, factor=0.0),
               dict(rot_dim=8, scaling="other"), dict(rot_dim=8, scaling="yarn", factor=2.0),
               dict(rot_dim=2, scaling="ntk", factor=2.0),
               dict(rot_dim=8, scaling="llama3", factor=2.0, original_length=8192,
                    high_freq_factor=1.0)):
        with pytest.raises(ValueError):
            paged.rope_frequencies(**kw)
