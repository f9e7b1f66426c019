"""Torch-facing host helpers over the KVX C ABI.

These build kvx_abi.h descriptors from torch tensors (shape, element strides,
data pointer, memory type) and call libkvx_amd.so; ``write_kv`` and
``gather_kv`` have them built natively where csrc/paged_host.cpp is built, and
through ctypes otherwise.  torch is only the source of device memory and
streams here; every byte is moved by the library's HIP kernels.  There is no
fallback for those: if libkvx_amd.so is missing, ``abi.load()`` raises.

The calls mirror the reference's launch API (kernels/kvx_paged_kv.h:11-21):
``write_kv`` -> kvx_launch_write_kv / kvx_launch_write_kv_prefill,
``gather_kv`` -> kvx_launch_gather_kv / kvx_launch_gather_kv_dequant, and
return the kvx_status_t as ``abi.Status``.
"""
from __future__ import annotations

import ctypes as C
import importlib.util
import math
import warnings
from dataclasses import dataclass
from pathlib import Path

import torch

from . import abi
from .abi import DType, Layout, Memory, Status

_HOST_PATH = Path(__file__).resolve().parent / "_paged_host.so"
_HOST = None  # the module, or False where it cannot be loaded
_STATUS = {int(s): s for s in Status}


def _host():
    """The native descriptor builder (csrc/paged_host.cpp), or False: it is
    built for one Python and torch, and where it is missing or made for
    others the ctypes helpers below build the descriptors."""
    global _HOST
    if _HOST is None:
        host = False
        if _HOST_PATH.exists():
            spec = importlib.util.spec_from_file_location("_paged_host", _HOST_PATH)
            try:
                host = importlib.util.module_from_spec(spec)
                spec.loader.exec_module(host)
            except ImportError as e:
                host = False
                warnings.warn(f"{_HOST_PATH.name} does not load ({e}); descriptors are built "
                              "through ctypes, which takes longer", RuntimeWarning, stacklevel=3)
        _HOST = host
    return _HOST


def _address(lib, name: str) -> int:
    """Address of an entry point of the loaded library."""
    known = lib.__dict__.setdefault("_kvx_addresses", {})
    if name not in known:
        known[name] = C.cast(getattr(lib, name), C.c_void_p).value
    return known[name]


_TORCH_DTYPE = {
    torch.float16: DType.F16,
    torch.bfloat16: DType.BF16,
    torch.float32: DType.F32,
    torch.float8_e4m3fn: DType.F8_E4M3,
    torch.float8_e5m2: DType.F8_E5M2,
    torch.int32: DType.S32,
    torch.int64: DType.S64,
}


def dtype_code(t: torch.Tensor | torch.dtype) -> DType:
    dt = t.dtype if isinstance(t, torch.Tensor) else t
    if dt not in _TORCH_DTYPE:
        raise ValueError(f"unsupported dtype {dt}")
    return _TORCH_DTYPE[dt]


def memory_of(t: torch.Tensor) -> Memory:
    return Memory.DEVICE if t.is_cuda else Memory.HOST


def tensor_desc(t: torch.Tensor, layout: Layout = Layout.BLOCK_CUSTOM,
                dtype: DType | None = None) -> abi.TensorDesc:
    """Descriptor of `t` as laid out in memory (its own shape and strides)."""
    d = abi.TensorDesc()
    d.size = C.sizeof(abi.TensorDesc)
    d.dtype = int(dtype if dtype is not None else dtype_code(t))
    d.layout = int(layout)
    d.memory = int(memory_of(t))
    d.ndim = t.dim()
    for i in range(t.dim()):
        d.shape[i] = t.shape[i]
        d.stride[i] = t.stride(i)
    d.data = t.data_ptr()
    return d


def cache_shape(layout: Layout, num_blocks: int, block_size: int, heads: int,
                head_dim: int, pack: int = 8) -> tuple:
    """Canonical shape of a cache tensor in `layout` (KVX_SPEC.md:50-56)."""
    layout = Layout(layout)
    if layout == Layout.BLOCK_NHD:
        return (num_blocks, block_size, heads, head_dim)
    if layout == Layout.BLOCK_HND:
        return (num_blocks, heads, block_size, head_dim)
    if layout == Layout.BLOCK_HND_PACKED:
        return (num_blocks, heads, head_dim // pack, block_size, pack)
    raise ValueError(layout)


@dataclass
class PagedCache:
    """K and V cache tensors and the kvx_cache_desc_t describing them."""

    key_cache: torch.Tensor
    value_cache: torch.Tensor
    k_layout: Layout
    v_layout: Layout
    num_blocks: int
    block_size: int
    heads: int
    head_dim: int

    def desc(self) -> abi.CacheDesc:
        k = tensor_desc(self.key_cache, self.k_layout)
        v = tensor_desc(self.value_cache, self.v_layout)
        return abi.cache_desc(self.num_blocks, self.block_size, self.heads,
                              self.head_dim, k, v)


def alloc_cache(num_blocks: int, block_size: int, heads: int, head_dim: int,
                dtype: torch.dtype, device, k_layout=Layout.BLOCK_NHD,
                v_layout=None, pack: int = 8) -> PagedCache:
    v_layout = k_layout if v_layout is None else v_layout
    k = torch.empty(cache_shape(k_layout, num_blocks, block_size, heads, head_dim, pack),
                    dtype=dtype, device=device)
    v = torch.empty(cache_shape(v_layout, num_blocks, block_size, heads, head_dim, pack),
                    dtype=dtype, device=device)
    return PagedCache(k, v, Layout(k_layout), Layout(v_layout), num_blocks, block_size,
                      heads, head_dim)


def custom_view(storage: torch.Tensor, order: str) -> torch.Tensor:
    """The logical CUSTOM view of a cache `storage` whose axes are named by
    `order`: a permutation of "bohd" (block, offset, head, dim) or "bohpx"
    (dim split as dim / x, x).  E.g. order "bhdo" is vLLM's value cache
    [num_blocks, H, D, block_size]."""
    logical = "bohpx" if len(order) == 5 else "bohd"
    if sorted(order) != sorted(logical):
        raise ValueError(f"order {order!r} is not a permutation of {logical!r}")
    return storage.permute([order.index(a) for a in logical])


def alloc_custom_cache(num_blocks: int, block_size: int, heads: int, head_dim: int,
                       dtype: torch.dtype, device, k_order: str = "bhdo",
                       v_order: str | None = None, x: int = 8) -> PagedCache:
    """K and V caches in KVX_LAYOUT_BLOCK_CUSTOM with storage axis orders
    k_order / v_order (see custom_view; 5-letter orders split dim by x)."""
    v_order = k_order if v_order is None else v_order

    def one(order):
        size = {"b": num_blocks, "o": block_size, "h": heads, "d": head_dim,
                "p": head_dim // x, "x": x}
        t = torch.empty([size[a] for a in order], dtype=dtype, device=device)
        return custom_view(t, order)

    return PagedCache(one(k_order), one(v_order), Layout.BLOCK_CUSTOM, Layout.BLOCK_CUSTOM,
                      num_blocks, block_size, heads, head_dim)


def alloc_block_pool(num_blocks: int, block_size: int, heads: int, head_dim: int,
                     dtype: torch.dtype, device, layout=Layout.BLOCK_NHD,
                     pack: int = 8) -> tuple[PagedCache, PagedCache]:
    """One pool of 2 * num_blocks single-tensor blocks in TensorRT-LLM's
    KVBlockArray pairing: the K block of logical block b is pool block 2b, its
    V block is 2b + 1.  Returns (pool, kv): `pool` describes all pool blocks
    (the cache for KV_OFFSETS gathers, whose OffsetsTable is
    ``pool_table``); `kv` views the same memory as K and V caches of
    num_blocks blocks for PACKED-table writes and gathers."""
    shape = cache_shape(layout, 2 * num_blocks, block_size, heads, head_dim, pack)
    mem = torch.empty(shape, dtype=dtype, device=device)
    layout = Layout(layout)
    pool = PagedCache(mem, mem, layout, layout, 2 * num_blocks, block_size, heads, head_dim)
    kv = PagedCache(mem[0::2], mem[1::2], layout, layout, num_blocks, block_size, heads,
                    head_dim)
    return pool, kv


def pool_table(pool: PagedCache, offsets: torch.Tensor,
               secondary: torch.Tensor | None = None) -> "OffsetsTable":
    """OffsetsTable over the memory of `pool` (see alloc_block_pool)."""
    mem = pool.key_cache
    return OffsetsTable(offsets, mem, secondary, mem.stride(0) * mem.element_size())


def _stream_handle(stream) -> int | None:
    if stream is None:
        return torch.cuda.current_stream().cuda_stream if torch.cuda.is_available() else None
    if isinstance(stream, torch.cuda.Stream):
        return stream.cuda_stream
    return int(stream)


@dataclass
class Scales:
    """FP8 scales of one tensor with a granularity: `values` is a float32
    device tensor of shape [1] (PER_TENSOR), [num_kv_heads] (PER_HEAD),
    [num_blocks] (PER_BLOCK, by physical block id) or [num_blocks,
    num_kv_heads] (PER_BLOCK_HEAD); its own strides are passed."""

    values: torch.Tensor
    granularity: abi.ScaleGranularity = abi.ScaleGranularity.PER_TENSOR


def scale_desc_of(scale) -> abi.ScaleDesc:
    """kvx_scale_desc_t for a one-element float32 tensor (per tensor) or a
    Scales."""
    if isinstance(scale, Scales):
        v = scale.values
        shape = tuple(v.shape) or (1,)
        stride = tuple(v.stride()) or (1,)
        return abi.scale_desc(v.data_ptr(), granularity=scale.granularity, shape=shape,
                              stride=stride)
    return abi.scale_desc(scale.data_ptr())


def _cache_args(cache: PagedCache) -> tuple:
    return (cache.key_cache, cache.value_cache, cache.k_layout, cache.v_layout, cache.num_blocks,
            cache.block_size, cache.heads, cache.head_dim)


def _scale_args(scale) -> tuple:
    """(tensor, granularity) of a scale; -1: a per-tensor tensor."""
    if isinstance(scale, Scales):
        return scale.values, int(scale.granularity)
    return scale, -1


def _table_args(table) -> tuple:
    """(table, indptr, primary, secondary, bytes_per_block) of a block table."""
    if isinstance(table, RaggedTable):
        return table.indices, table.indptr, None, None, 0
    if isinstance(table, OffsetsTable):
        return table.offsets, None, table.primary, table.secondary, table.bytes_per_block
    return table, None, None, None, 0


def build_write(cache: PagedCache, key: torch.Tensor, value: torch.Tensor,
                slot_mapping: torch.Tensor, k_scale=None, v_scale=None) -> abi.WriteDesc:
    """kvx_write_desc_t for [T, H, D] key/value rows and [T] slots.  FP8
    scales are one-element F32 device tensors, passed as PER_TENSOR scale
    descriptors."""
    T = key.shape[0]
    w = abi.WriteDesc()
    w.size = C.sizeof(abi.WriteDesc)
    w.io.size = C.sizeof(abi.KvIoDesc)
    w.io.key = tensor_desc(key)
    w.io.value = tensor_desc(value)
    w.io.num_tokens = T
    w.io.num_kv_heads = key.shape[1] if key.dim() == 3 else 0
    w.io.head_dim = key.shape[2] if key.dim() == 3 else 0
    w.slots.size = C.sizeof(abi.SlotMapping)
    w.slots.dtype = int(dtype_code(slot_mapping))
    w.slots.token_count = slot_mapping.numel()
    w.slots.invalid_slot = -1
    w.slots.slots = slot_mapping.data_ptr()
    if k_scale is not None:
        w.k_scale_desc = scale_desc_of(k_scale)
    if v_scale is not None:
        w.v_scale_desc = scale_desc_of(v_scale)
    return w


@dataclass
class RaggedTable:
    """RAGGED block table (KVX_SPEC.md:107-114): token t of sequence s is
    cached in block ``indices[indptr[s] + t]`` at offset ``t % block_size``,
    for t < indptr[s+1] - indptr[s]."""

    indices: torch.Tensor  # [total tokens] int32 / int64 block ids
    indptr: torch.Tensor   # [seq_count + 1] int32 / int64 prefix sums


@dataclass
class OffsetsTable:
    """KV_OFFSETS block table (KVX_SPEC.md:116-122, TensorRT-LLM's
    KVBlockArray): int32 ``offsets[s, 0, 0 (K) / 1 (V), j]`` are KVCacheIndex
    values; block j of sequence s lives at ``pool + (value & 0x7FFFFFFF) *
    bytes_per_block`` with bit 31 choosing the secondary pool.  The cache's K
    / V tensors give only the in-block layout."""

    offsets: torch.Tensor              # int32 [seq_count, 1, 2, max_blocks_per_seq]
    primary: torch.Tensor              # pool storage (its bytes)
    secondary: torch.Tensor | None
    bytes_per_block: int


def kv_cache_index(block: int, secondary: bool = False) -> int:
    """The int32 KVCacheIndex value for `block` in the primary or secondary
    pool (KV_CACHE_LAYOUTS.md:91-92)."""
    v = (int(block) & 0x7FFFFFFF) | (0x80000000 if secondary else 0)
    return v - (1 << 32) if v >= 0x80000000 else v


def _table_desc(table) -> abi.BlockTable:
    if isinstance(table, RaggedTable):
        t = abi.BlockTable()
        t.size = C.sizeof(abi.BlockTable)
        t.format = int(abi.TableFormat.RAGGED)
        t.index_dtype = int(dtype_code(table.indices))
        t.indptr_dtype = int(dtype_code(table.indptr))
        t.seq_count = table.indptr.numel() - 1
        t.beam_width = 1
        t.max_blocks_per_seq = 1  # not used by RAGGED; the ABI path requires > 0
        t.indices = table.indices.data_ptr()
        t.indptr = table.indptr.data_ptr()
        t.indices_count = table.indices.numel()
        t.indptr_count = table.indptr.numel()
        return t
    if isinstance(table, OffsetsTable):
        S, beam, two, mbps = table.offsets.shape
        if two != 2 or table.offsets.dtype != torch.int32:
            raise ValueError("KV_OFFSETS table is int32 [seq_count, beam, 2, max_blocks]")
        t = abi.BlockTable()
        t.size = C.sizeof(abi.BlockTable)
        t.format = int(abi.TableFormat.KV_OFFSETS)
        t.index_dtype = int(DType.S32)
        t.seq_count = S
        t.beam_width = beam
        t.max_blocks_per_seq = mbps
        t.indices = table.offsets.data_ptr()
        t.indices_count = table.offsets.numel()
        t.flags = abi.TABLE_FLAG_KVCACHEINDEX
        return t
    S, mbps = table.shape
    return abi.make_block_table_packed(S, mbps, dtype_code(table), table.data_ptr())


def gather_cache_desc(cache: PagedCache, block_table) -> abi.CacheDesc:
    """The cache descriptor of a gather; an OffsetsTable also fills its pool
    fields (kvx_pool_desc_t)."""
    cd = cache.desc()
    if isinstance(block_table, OffsetsTable):
        cd.pool.size = C.sizeof(abi.PoolDesc)
        cd.pool.memory = int(memory_of(block_table.primary))
        cd.pool.bytes_per_block = block_table.bytes_per_block
        cd.pool.primary = block_table.primary.data_ptr()
        cd.pool.secondary = (None if block_table.secondary is None
                             else block_table.secondary.data_ptr())
    return cd


def build_gather(key_out: torch.Tensor, value_out: torch.Tensor,
                 block_table, seq_lens: torch.Tensor,
                 max_seq_len: int) -> abi.GatherDesc:
    """kvx_gather_desc_t for [S, max_seq_len, H, D] outputs.  `block_table` is
    a [S, max_blocks_per_seq] tensor (PACKED), a RaggedTable or an
    OffsetsTable."""
    tb = _table_desc(block_table)
    S = tb.seq_count
    g = abi.GatherDesc()
    g.size = C.sizeof(abi.GatherDesc)
    g.io.size = C.sizeof(abi.KvIoDesc)
    g.io.key = tensor_desc(key_out)
    g.io.value = tensor_desc(value_out)
    g.io.num_tokens = S * max_seq_len
    g.io.num_kv_heads = key_out.shape[2]
    g.io.head_dim = key_out.shape[3]
    g.block_table = tb
    g.seq_lens = abi.make_seq_lens(seq_lens.numel(), dtype_code(seq_lens),
                                   seq_lens.data_ptr())
    g.max_seq_len = max_seq_len
    return g


def write_kv(cache: PagedCache, key: torch.Tensor, value: torch.Tensor,
             slot_mapping: torch.Tensor, *, tokens_per_seq: int | None = None,
             k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
             stream=None, entry: str = "launch") -> Status:
    """Scatter rows into the paged cache.  entry = "launch" (kvx_paged_kv.h)
    or "abi" (kvx_write_kv of kvx_abi.h)."""
    lib = abi.load()
    name = ("kvx_write_kv" if entry == "abi" else "kvx_launch_write_kv"
            if tokens_per_seq is None else "kvx_launch_write_kv_prefill")
    code = None
    host = _host()
    if host and type(cache) is PagedCache:
        code = host.write(
            _address(lib, name), None if entry == "abi" else tokens_per_seq,
            None if stream is None else _stream_handle(stream), *_cache_args(cache), key, value,
            slot_mapping, *_scale_args(k_scale), *_scale_args(v_scale))
    if code is not None:
        return _STATUS[code]
    # arguments that the native builder leaves to the descriptor helpers
    cd = cache.desc()
    wd = build_write(cache, key, value, slot_mapping, k_scale, v_scale)
    s = _stream_handle(stream)
    if entry == "abi":
        return Status(lib.kvx_write_kv(C.byref(cd), C.byref(wd), s))
    if tokens_per_seq is not None:
        return Status(lib.kvx_launch_write_kv_prefill(C.byref(cd), C.byref(wd),
                                                      tokens_per_seq, s))
    return Status(lib.kvx_launch_write_kv(C.byref(cd), C.byref(wd), s))


def gather_kv(cache: PagedCache, key_out: torch.Tensor, value_out: torch.Tensor,
              block_table, seq_lens: torch.Tensor, max_seq_len: int, *,
              k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
              stream=None, entry: str = "launch",
              pool_blocks: tuple[int, int] | None = None) -> Status:
    """Gather sequences into contiguous [S, max_seq_len, H, D] buffers.
    `block_table` is a PACKED [S, max_blocks_per_seq] tensor, a RaggedTable
    or an OffsetsTable (whose pool replaces the cache tensors' data).
    With k_scale/v_scale the FP8 cache is dequantized
    (kvx_launch_gather_kv_dequant).  pool_blocks = (primary, secondary)
    block counts go through kvx_launch_gather_kv_pools instead."""
    lib = abi.load()
    host = _host()
    if (host and type(cache) is PagedCache and pool_blocks is None
            and (entry != "abi" or k_scale is None)):
        table = _table_args(block_table)
        name = ("kvx_gather_kv" if entry == "abi" else "kvx_launch_gather_kv"
                if k_scale is None and v_scale is None else "kvx_launch_gather_kv_dequant")
        code = host.gather(
            _address(lib, name), None if stream is None else _stream_handle(stream),
            *_cache_args(cache), key_out, value_out, *table, seq_lens, max_seq_len,
            *_scale_args(k_scale), *_scale_args(v_scale))
        if code is not None:
            return _STATUS[code]
    # arguments that the native builder leaves to the descriptor helpers
    cd = gather_cache_desc(cache, block_table)
    gd = build_gather(key_out, value_out, block_table, seq_lens, max_seq_len)
    s = _stream_handle(stream)
    if entry == "abi":
        return Status(lib.kvx_gather_kv(C.byref(cd), C.byref(gd), s))
    if pool_blocks is not None:
        pb = abi.PoolBlocks(C.sizeof(abi.PoolBlocks), 0, pool_blocks[0], pool_blocks[1])
        ks = vs = None
        if k_scale is not None or v_scale is not None:
            ks, vs = C.byref(scale_desc_of(k_scale)), C.byref(scale_desc_of(v_scale))
        return Status(lib.kvx_launch_gather_kv_pools(C.byref(cd), C.byref(gd), C.byref(pb), ks,
                                                     vs, s))
    if k_scale is not None or v_scale is not None:
        ks = scale_desc_of(k_scale)
        vs = scale_desc_of(v_scale)
        return Status(lib.kvx_launch_gather_kv_dequant(C.byref(cd), C.byref(gd),
                                                       C.byref(ks), C.byref(vs), s))
    return Status(lib.kvx_launch_gather_kv(C.byref(cd), C.byref(gd), s))


# ---------------------------------------------------------------------------
# Operators of a serving step beside the write and the gather (kvx_ext.h; no
# reference counterparts).

@dataclass
class Rope:
    """Rotary positions: pair i of a head turns by position * inv_freq[i].
    `inv_freq` is a contiguous float32 device tensor [rot_dim / 2]
    (``rope_frequencies``); elements of a head from rot_dim on are not
    rotated.  `interleaved` pairs are (2 i, 2 i + 1), others (i, i + rot_dim /
    2); `magnitude` multiplies cosines and sines."""

    inv_freq: torch.Tensor
    interleaved: bool = False
    magnitude: float = 1.0


def rope_frequencies(rot_dim: int, base: float = 10000.0, *, scaling: str | None = None,
                     factor: float = 1.0, original_length: int | None = None,
                     low_freq_factor: float = 1.0, high_freq_factor: float = 4.0,
                     beta_fast: float = 32.0, beta_slow: float = 1.0,
                     magnitude: float | None = None, device=None) -> tuple[torch.Tensor, float]:
    """(inv_freq, magnitude) of a checkpoint's rotary settings, computed in 64
    bits: inv_freq[i] = base ** (-2 i / rot_dim) in float32, scaled for
    contexts `factor` times the trained `original_length`:

      None      as they are
      "linear"  all frequencies / factor
      "ntk"     base * factor ** (rot_dim / (rot_dim - 2))
      "llama3"  waves longer than original_length / low_freq_factor are
                slowed by factor, those shorter than original_length /
                high_freq_factor kept, those between blended by the number
                of turns in original_length
      "yarn"    pairs that turn fewer than beta_slow times in original_length
                are slowed by factor, those that turn more than beta_fast
                times kept, those between blended by their index; the
                magnitude is 0.1 ln(factor) + 1

    A given `magnitude` replaces the rule's."""
    if rot_dim <= 0 or rot_dim % 2:
        raise ValueError(f"rot_dim {rot_dim} is not a positive even number")
    if not base > 1.0 or not factor > 0.0:
        raise ValueError(f"base {base} or factor {factor} out of range")
    if scaling in ("llama3", "yarn") and not (original_length and original_length > 0):
        raise ValueError(f"scaling {scaling!r} needs original_length")
    i = torch.arange(rot_dim // 2, dtype=torch.float64)
    gain = 1.0
    if scaling == "ntk":
        if rot_dim == 2:
            raise ValueError("scaling 'ntk' needs rot_dim > 2")
        base = base * factor ** (rot_dim / (rot_dim - 2))
    inv = torch.pow(torch.tensor(base, dtype=torch.float64), -2.0 * i / rot_dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "llama3":
        if not high_freq_factor > low_freq_factor:
            raise ValueError("high_freq_factor must exceed low_freq_factor")
        turns = original_length * inv / (2 * math.pi)
        keep = ((turns - low_freq_factor) / (high_freq_factor - low_freq_factor)).clamp(0, 1)
        inv = inv * (keep + (1 - keep) / factor)
    elif scaling == "yarn":
        def pair_with(turns: float) -> float:
            return (rot_dim * math.log(original_length / (2 * math.pi * turns))
                    / (2 * math.log(base)))

        low = max(math.floor(pair_with(beta_fast)), 0)
        high = min(math.ceil(pair_with(beta_slow)), rot_dim - 1)
        slowed = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
        inv = inv * (1 - slowed + slowed / factor)
        gain = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"unknown scaling {scaling!r}")
    return inv.float().to(device or "cpu"), gain if magnitude is None else float(magnitude)


def _on_one_gpu(first: torch.Tensor, **tensors) -> torch.device:
    """The device of all tensors; ValueError names one that is elsewhere."""
    if not first.is_cuda:
        raise ValueError("the cache is not on a GPU")
    for name, t in tensors.items():
        if t is not None and t.device != first.device:
            raise ValueError(f"{name} is on {t.device}, the cache on {first.device}")
    return first.device


def _indices(name: str, t: torch.Tensor, shape: tuple | None = None) -> torch.Tensor:
    """`t`, an int32 / int64 tensor whose elements lie in order."""
    if t.dtype not in (torch.int32, torch.int64):
        raise ValueError(f"{name} is {t.dtype}, not int32 or int64")
    if not t.is_contiguous():
        raise ValueError(f"{name} is not contiguous")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {shape}")
    return t


def _check_scales(device: torch.device, **scales) -> None:
    for name, scale in scales.items():
        t = scale.values if isinstance(scale, Scales) else scale
        if t is None:
            continue
        if t.dtype != torch.float32:
            raise ValueError(f"{name} is {t.dtype}, not float32")
        if t.device != device:
            raise ValueError(f"{name} is on {t.device}, the cache on {device}")


def _row_tensor(name: str, t: torch.Tensor) -> torch.Tensor:
    if t.dim() != 3:
        raise ValueError(f"{name} is not [tokens, heads, head_dim]")
    return t


def build_rope(query: torch.Tensor | None, query_out: torch.Tensor | None,
               positions: torch.Tensor, rope: Rope) -> abi.RopeDesc:
    """kvx_rope_desc_t for [T, Hq, D] queries (or None) and [T] positions."""
    d = abi.RopeDesc()
    d.size = C.sizeof(abi.RopeDesc)
    d.style = int(abi.RopeStyle.INTERLEAVED if rope.interleaved else abi.RopeStyle.HALF)
    d.rot_dim = 2 * rope.inv_freq.numel()
    d.magnitude = rope.magnitude
    d.position_dtype = int(dtype_code(positions))
    d.positions = positions.data_ptr()
    d.inv_freq = rope.inv_freq.data_ptr()
    if query is not None:
        d.query = tensor_desc(query)
        d.query_out = tensor_desc(query_out)
    return d


def rope_write_kv(cache: PagedCache, query: torch.Tensor | None, key: torch.Tensor,
                  value: torch.Tensor, positions: torch.Tensor, rope: Rope,
                  slot_mapping: torch.Tensor, *, query_out: torch.Tensor | None = None,
                  k_scale=None, v_scale=None, stream=None) -> Status:
    """Rotates [T, Hq, D] queries into `query_out` (None: in place; else apart
    from the query) and [T, H, D] keys into the paged cache, and writes the
    values beside them:
    ``write_kv`` of the rotated keys, each element rounded once.  Tensors may
    have any token and head strides (views of one projection's output).  A
    slot of -1 skips a row's key and value; its query is rotated.  `query`
    None: keys and values alone.  kvx_launch_rope_write_kv."""
    lib = abi.load()
    if query is not None and query_out is None:
        query_out = query
    host = _host()
    if host and type(cache) is PagedCache:
        code = host.rope_write(
            _address(lib, "kvx_launch_rope_write_kv"),
            None if stream is None else _stream_handle(stream), *_cache_args(cache), query,
            query_out if query is not None else None, key, value, positions, rope.inv_freq,
            1 if rope.interleaved else 0, rope.magnitude, slot_mapping, *_scale_args(k_scale),
            *_scale_args(v_scale))
        if code is not None:
            return _STATUS[code]
    # what the native builder leaves to the descriptor helpers
    device = _on_one_gpu(cache.key_cache, value_cache=cache.value_cache, query=query, key=key,
                         value=value, positions=positions, inv_freq=rope.inv_freq,
                         slot_mapping=slot_mapping, query_out=query_out)
    _check_scales(device, k_scale=k_scale, v_scale=v_scale)
    T = _row_tensor("key", key).shape[0]
    _row_tensor("value", value)
    if query is not None:
        _row_tensor("query", query)
        _row_tensor("query_out", query_out)
    _indices("positions", positions, (T,))
    _indices("slot_mapping", slot_mapping, (T,))
    if rope.inv_freq.dtype != torch.float32 or not rope.inv_freq.is_contiguous():
        raise ValueError("inv_freq is not a contiguous float32 tensor")
    cd = cache.desc()
    wd = build_write(cache, key, value, slot_mapping, k_scale, v_scale)
    rd = build_rope(query, query_out, positions, rope)
    with torch.cuda.device(device):
        return Status(lib.kvx_launch_rope_write_kv(C.byref(cd), C.byref(wd), C.byref(rd),
                                                   _stream_handle(stream)))


def build_attention(query: torch.Tensor, out: torch.Tensor, block_table, seq_lens: torch.Tensor,
                    query_indptr: torch.Tensor | None = None, *, causal: bool = True,
                    scale: float | None = None, window: int = 0, softcap: float = 0.0,
                    lse: torch.Tensor | None = None, max_seq_len: int = 0,
                    max_query_len: int = 0, k_scale=None, v_scale=None) -> abi.AttentionDesc:
    """kvx_attention_desc_t, without workspace and pool counts."""
    d = abi.AttentionDesc()
    d.size = C.sizeof(abi.AttentionDesc)
    d.flags = abi.ATTENTION_CAUSAL if causal else 0
    d.query = tensor_desc(query)
    d.out = tensor_desc(out)
    d.lse = None if lse is None else lse.data_ptr()
    if query_indptr is not None:
        d.query_indptr = query_indptr.data_ptr()
        d.query_indptr_dtype = int(dtype_code(query_indptr))
    d.window = window
    d.scale = max(query.shape[-1], 1) ** -0.5 if scale is None else scale
    d.softcap = softcap
    d.max_seq_len = max_seq_len
    d.max_query_len = max_query_len
    d.block_table = _table_desc(block_table)
    d.seq_lens = abi.make_seq_lens(seq_lens.numel(), dtype_code(seq_lens), seq_lens.data_ptr())
    if k_scale is not None:
        d.k_scale = scale_desc_of(k_scale)
    if v_scale is not None:
        d.v_scale = scale_desc_of(v_scale)
    return d


def attention(cache: PagedCache, query: torch.Tensor, out: torch.Tensor, block_table,
              seq_lens: torch.Tensor, query_indptr: torch.Tensor | None = None, *,
              causal: bool = True, scale: float | None = None, window: int = 0,
              softcap: float = 0.0, lse: torch.Tensor | None = None, max_seq_len: int = 0,
              max_query_len: int = 0, k_scale=None, v_scale=None,
              pool_blocks: tuple[int, int] | None = None,
              workspace: torch.Tensor | None = None, stream=None) -> Status:
    """Attention of new tokens over the paged cache that holds them already.

    Sequence s has the rows query_indptr[s] .. query_indptr[s + 1] - 1 of
    `query` [T, Hq, D] (`query_indptr` None: the one row s, a decode step) and
    seq_lens[s] cached tokens, the new ones last.  A row at position p attends
    to the tokens up to p (`causal`; else to all), with a `window` only to the
    last `window` of them.  softmax(scale * q.k) v goes to `out` (like
    `query` and apart from it, or the query itself), the natural logarithm of the weights' sum to `lse` (float32 [T,
    Hq], or None); `scale` is 1 / sqrt(D) unless given; `softcap` > 0 turns a
    logit x into softcap * tanh(x / softcap).  Hq is a multiple of the cache's
    heads.  Rows that attend to nothing are 0 with lse -inf; rows behind the
    last sequence are left as they were.  `block_table`, `k_scale`, `v_scale`
    and `pool_blocks` as in ``gather_kv``.

    `max_seq_len` and `max_query_len`, the largest values in this batch, steer
    how the work is split (0: not known) and not the result.  `workspace` is a
    uint8 tensor of ``attention_workspace_size`` bytes, one for each call that
    may run at the same time; None allocates it.  kvx_launch_attention."""
    lib = abi.load()
    host = _host()
    if scale is None:
        scale = max(_row_tensor("query", query).shape[2], 1) ** -0.5
    if host and type(cache) is PagedCache and pool_blocks is None:
        code = host.attention(
            _address(lib, "kvx_launch_attention"),
            _address(lib, "kvx_attention_workspace_size"),
            None if stream is None else _stream_handle(stream), *_cache_args(cache), query, out,
            *_table_args(block_table), seq_lens, query_indptr, 1 if causal else 0,
            scale, window, softcap, lse, max_seq_len, max_query_len, *_scale_args(k_scale),
            *_scale_args(v_scale), workspace)
        if code is not None:
            return _STATUS[code]
    # what the native builder leaves to the descriptor helpers
    if isinstance(block_table, RaggedTable):
        table_tensors = {"indices": _indices("indices", block_table.indices),
                         "indptr": _indices("indptr", block_table.indptr)}
    elif isinstance(block_table, OffsetsTable):
        table_tensors = {"offsets": _indices("offsets", block_table.offsets),
                         "primary": block_table.primary, "secondary": block_table.secondary}
    else:
        table_tensors = {"block_table": _indices("block_table", block_table)}
        if block_table.dim() != 2:
            raise ValueError("block_table is not [sequences, blocks]")
    _row_tensor("query", query)
    device = _on_one_gpu(cache.key_cache, value_cache=cache.value_cache, query=query, out=out,
                         seq_lens=seq_lens, query_indptr=query_indptr, lse=lse,
                         workspace=workspace, **table_tensors)
    _check_scales(device, k_scale=k_scale, v_scale=v_scale)
    _row_tensor("out", out)
    cd = gather_cache_desc(cache, block_table)
    d = build_attention(query, out, block_table, seq_lens, query_indptr, causal=causal,
                        scale=scale, window=window, softcap=softcap, lse=lse,
                        max_seq_len=max_seq_len, max_query_len=max_query_len, k_scale=k_scale,
                        v_scale=v_scale)
    S = d.block_table.seq_count
    _indices("seq_lens", seq_lens, (S,))
    if query_indptr is not None:
        _indices("query_indptr", query_indptr, (S + 1,))
    if lse is not None and (lse.dtype != torch.float32 or not lse.is_contiguous()
                            or tuple(lse.shape) != tuple(query.shape[:2])):
        raise ValueError("lse is not a contiguous float32 [T, Hq] tensor")
    pools = None
    if pool_blocks is not None:
        pools = abi.PoolBlocks(C.sizeof(abi.PoolBlocks), 0, pool_blocks[0], pool_blocks[1])
        d.pool_blocks = C.pointer(pools)
    size = C.c_uint64()
    st = Status(lib.kvx_attention_workspace_size(C.byref(cd), C.byref(d), C.byref(size)))
    if st != Status.OK:
        return st
    with torch.cuda.device(device):
        if workspace is None and size.value:
            if isinstance(stream, int):
                stream = torch.cuda.ExternalStream(stream)
            # of the stream that uses it, so that it is not handed out before
            with torch.cuda.stream(stream):
                workspace = torch.empty(size.value, dtype=torch.uint8, device=device)
        if workspace is not None:
            if not workspace.is_contiguous():
                raise ValueError("workspace is not contiguous")
            d.workspace = workspace.data_ptr()
            d.workspace_size = workspace.numel() * workspace.element_size()
        return Status(lib.kvx_launch_attention(C.byref(cd), C.byref(d), _stream_handle(stream)))


def attention_workspace_size(cache: PagedCache, query: torch.Tensor, block_table,
                             seq_lens: torch.Tensor, query_indptr: torch.Tensor | None = None, *,
                             max_seq_len: int = 0, max_query_len: int = 0, k_scale=None,
                             v_scale=None) -> int:
    """Bytes of workspace that ``attention`` needs for such arguments."""
    cd = gather_cache_desc(cache, block_table)
    d = build_attention(query, query, block_table, seq_lens, query_indptr,
                        max_seq_len=max_seq_len, max_query_len=max_query_len, k_scale=k_scale,
                        v_scale=v_scale)
    size = C.c_uint64()
    st = Status(abi.load().kvx_attention_workspace_size(C.byref(cd), C.byref(d), C.byref(size)))
    if st != Status.OK:
        raise ValueError(f"no attention for these arguments: {st.name}")
    return size.value


def copy_blocks(caches, pairs: torch.Tensor, *, stream=None) -> Status:
    """Copies blocks inside the caches of a model's layers: for each row (src,
    dst) of `pairs` (int32 / int64 [n, 2]) block src of K and V to block dst,
    in every PagedCache of `caches`.  Rows with an id outside the pool (such
    as -1 padding) are skipped; no dst may be the src or dst of another row.
    Block-indexed FP8 scales are the caller's to copy with their blocks.
    kvx_launch_copy_blocks."""
    lib = abi.load()
    caches = caches if isinstance(caches, list) else list(caches)
    host = _host()
    if host:
        code = host.copy_blocks(_address(lib, "kvx_launch_copy_blocks"),
                                None if stream is None else _stream_handle(stream), PagedCache,
                                caches, pairs)
        if code is not None:
            return _STATUS[code]
    _indices("pairs", pairs)
    if pairs.dim() != 2 or pairs.shape[1] != 2:
        raise ValueError(f"pairs has shape {tuple(pairs.shape)}, not (n, 2)")
    if not caches:
        return Status.OK
    device = _on_one_gpu(caches[0].key_cache, pairs=pairs)
    for c in caches:
        _on_one_gpu(caches[0].key_cache, key_cache=c.key_cache, value_cache=c.value_cache)
    descs = [c.desc() for c in caches]
    ptrs = (C.POINTER(abi.CacheDesc) * len(descs))(*[C.pointer(d) for d in descs])
    with torch.cuda.device(device):
        return Status(lib.kvx_launch_copy_blocks(ptrs, len(descs), pairs.data_ptr(),
                                                 int(dtype_code(pairs)), pairs.shape[0],
                                                 _stream_handle(stream)))
