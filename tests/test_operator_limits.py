"""Sizes at the operators' limits (CPU only): refused before any arithmetic that
they would overflow."""
import ctypes as C

from kvx_amd import abi
from kvx_amd.abi import DType, Status

from test_operator_validation import attn, cache, rows

MOST = 0x7FFFFFFF


def size_of(lib, c, a):
    size = C.c_uint64(0)
    return Status(lib.kvx_attention_workspace_size(abi.ref(c), abi.ref(a), C.byref(size))), size.value


def test_tokens_and_sequences_together(kvx_lib):
    """With query offsets there are up to tokens + sequences tiles, which are
    32-bit numbers."""
    c = cache(H=1)
    for T, S in ((MOST, MOST), (MOST, 1), (1 << 30, (1 << 30) + 1)):
        st, _ = size_of(kvx_lib, c, attn(T=T, S=S, Hq=64, mbps=1, indptr=DType.S32))
        assert st == Status.UNSUPPORTED, (T, S)
        st = kvx_lib.kvx_launch_attention(abi.ref(c), abi.ref(
            attn(T=T, S=S, Hq=64, mbps=1, indptr=DType.S32)), None)
        assert Status(st) == Status.UNSUPPORTED
    st, _ = size_of(kvx_lib, c, attn(T=MOST - 1, S=1, Hq=64, mbps=1, indptr=DType.S32))
    assert st == Status.OK


def test_strides_that_no_memory_has(kvx_lib):
    """Spans past 2^56 elements are refused; strides of axes of one element may
    be anything."""
    for stride in (1 << 62, -(1 << 63), 1 << 56):
        a = attn()
        a.query.stride[0] = stride
        assert size_of(kvx_lib, cache(), a)[0] == Status.INVALID_ARGUMENT
        for axis in range(4):
            c = cache()
            c.v.stride[axis] = stride
            assert size_of(kvx_lib, c, attn())[0] == Status.INVALID_ARGUMENT
            ptrs = (C.POINTER(abi.CacheDesc) * 1)(C.pointer(c))
            assert Status(kvx_lib.kvx_launch_copy_blocks(
                ptrs, 1, 0x10000, int(DType.S32), 1, None)) == Status.INVALID_ARGUMENT
            w, r = rope_write()
            assert Status(kvx_lib.kvx_launch_rope_write_kv(
                abi.ref(c), abi.ref(w), abi.ref(r), None)) == Status.INVALID_ARGUMENT
        w, r = rope_write()
        w.io.key.stride[0] = stride
        assert Status(kvx_lib.kvx_launch_rope_write_kv(
            abi.ref(cache()), abi.ref(w), abi.ref(r), None)) == Status.INVALID_ARGUMENT
        a = attn(T=1, S=1)
        a.query.stride[0] = a.out.stride[0] = stride
        c = cache(nb=1)
        c.k.stride[0] = stride
        assert size_of(kvx_lib, c, a)[0] == Status.OK


def rope_write(T=3, H=2, D=64):
    w, r = abi.WriteDesc(), abi.RopeDesc()
    w.size, w.io.size, w.slots.size, r.size = (C.sizeof(x) for x in (w, w.io, w.slots, r))
    w.io.key, w.io.value = rows(DType.BF16, T, H, D), rows(DType.BF16, T, H, D)
    w.io.num_tokens, w.io.num_kv_heads, w.io.head_dim = T, H, D
    w.slots.dtype, w.slots.token_count, w.slots.slots = DType.S32, T, 0x10000
    r.rot_dim, r.magnitude, r.position_dtype = D, 1.0, DType.S32
    r.positions = r.inv_freq = 0x10000
    return w, r
