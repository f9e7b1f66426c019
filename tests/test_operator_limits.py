"""Sizes at the operators' limits (CPU only): refused before any arithmetic that
they would overflow."""
import ctypes as C

from kvx_amd import abi
from kvx_amd.abi import DType, Status

from test_operator_validation import cache, attn

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
