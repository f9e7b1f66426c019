"""Performance cases of the operators beside the paged write and gather.

Three operators of a serving step over a paged KV cache, each in the form a
user's program calls it (``own``) and in a plain form of elementary torch
operations:

``attention``      attention of each sequence's new tokens over its cached
                   ones: single-token decode steps, a few tokens at once
                   (verified drafts), prefill chunks and mixed batches.
``rope_write_kv``  rotary positions of query and key rows, the rotated keys
                   and the values written into the cache.
``copy_blocks``    pages copied inside the cache of every layer, as forks of
                   a sequence and a pool's compaction need.

Lengths depend on the case alone, so that its work does; values, block order
and scales depend on the seed.
"""
from __future__ import annotations

import math
import random

import torch

own = False

_DTYPE = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32,
          "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
_BYTES = {"f16": 2, "bf16": 2, "f32": 4, "e4m3": 1, "e5m2": 1}
_FP8_MAX = {"e4m3": 448.0, "e5m2": 57344.0}
_INDEX = {"s32": torch.int32, "s64": torch.int64}
_DEVICE = "cuda:0"


def _attention(name, io, cache, layout, table, block, heads, group, dim, seqs, lo, hi, **more):
    """`seqs` sequences of lo..hi cached tokens, the last new_lo..new_hi of
    them new; of `few` sequences in `few_of` only one token is new."""
    case = {"name": name, "op": "attention", "io": io, "cache": cache, "layout": layout,
            "table": table, "block": block, "heads": heads, "group": group, "dim": dim,
            "seqs": seqs, "lo": lo, "hi": hi, "new_lo": 1, "new_hi": 1, "few": 0, "few_of": 1,
            "window": 0, "softcap": 0.0, "scales": "tensor", "index": "s32", "lens_seed": 1}
    case.update(more)
    return case


def _rope(name, io, cache, layout, block, heads, group, dim, rot, style, seqs, lo, hi, **more):
    """The rows of `seqs` sequences with lo..hi new tokens each (1: decode),
    at positions up to `far`; `fused`: q, k and v are views of one
    projection's output."""
    case = {"name": name, "op": "rope_write", "io": io, "cache": cache, "layout": layout,
            "block": block, "heads": heads, "group": group, "dim": dim, "rot": rot,
            "style": style, "seqs": seqs, "lo": lo, "hi": hi, "far": 8192, "scaling": "none",
            "base": 10000.0, "fused": True, "padded": 0, "scales": "tensor", "index": "s64",
            "lens_seed": 1}
    case.update(more)
    return case


def _copy(name, cache, layout, block, heads, dim, layers, blocks, pairs, **more):
    """`pairs` pages copied in each of `layers` caches of `blocks` pages."""
    case = {"name": name, "op": "copy_blocks", "cache": cache, "layout": layout, "block": block,
            "heads": heads, "dim": dim, "layers": layers, "blocks": blocks, "pairs": pairs,
            "index": "s64"}
    case.update(more)
    return case


def listed():
    return [
        # The smallest attention call: one user's chat, a decode step over a
        # few hundred tokens of a small model.  Latency is all of it.
        _attention("decode_1_short", "f16", "f16", "nhd", "packed", 16, 4, 8, 64, 1, 301, 301),
        # One decode step in a layer of Llama-3-8B shape, 128 sequences of
        # 512 to 8192 tokens: the cache is read once.
        _attention("decode_128", "bf16", "bf16", "nhd", "packed", 16, 8, 4, 128, 128, 512, 8192),
        # The same from an FP8 cache with a scale for each head.
        _attention("decode_128_fp8", "bf16", "e4m3", "nhd", "packed", 16, 8, 4, 128, 128, 512,
                   8192, scales="head"),
        # Long contexts at a small batch, 70B shape: blocks of 32 tokens.
        _attention("decode_5_long", "bf16", "bf16", "hnd", "packed", 32, 8, 8, 128, 5, 16384,
                   32768, lens_seed=3),
        # Drafts of two to seven tokens verified at once, in vLLM's cache
        # layout (x-packed K, V with the token axis innermost), odd batch.
        _attention("verify_drafts_33", "f16", "f16", "vllm", "packed", 16, 8, 4, 128, 33, 700,
                   4100, new_lo=2, new_hi=7, index="s64"),
        # A prefill chunk of 2048 tokens in each of two sequences that hold
        # 4096 to 8192 tokens then: compute-bound.
        _attention("prefill_2048", "bf16", "bf16", "packed_k", "packed", 16, 8, 4, 128, 2, 4096,
                   8192, new_lo=2048, new_hi=2048),
        # A mixed step: chunks of 100 to 500 tokens beside sequences that
        # decode, of a model with a sliding window.
        _attention("mixed_window", "bf16", "bf16", "nhd", "ragged", 16, 4, 8, 64, 12, 300, 3000,
                   new_lo=100, new_hi=500, few=2, few_of=3, window=1024),
        # The rotation and write of a decode step of four sequences: latency.
        _rope("rope_decode_4", "bf16", "bf16", "nhd", 16, 8, 4, 128, 128, "half", 4, 1, 1,
              base=500000.0),
        # A padded decode batch far into long contexts, into an FP8 cache;
        # only the first half of each head rotates, in adjacent pairs.
        _rope("rope_decode_251_fp8", "bf16", "e4m3", "nhd", 16, 8, 4, 128, 64, "interleaved", 251,
              1, 1, far=1000000, scaling="yarn", padded=13),
        # Prefill of 16 chunks of 2048 tokens, x-packed K, row-major V.
        _rope("rope_prefill", "bf16", "bf16", "packed_k", 16, 8, 4, 128, 128, "half", 16, 2048,
              2048, scaling="llama3", base=500000.0, far=100000),
        # A fork of two sequences: their last pages copied in 32 layers.
        _copy("fork_2", "bf16", "nhd", 16, 8, 128, 32, 256, 2),
        # Compaction of a pool: 400 pages moved in 32 layers.
        _copy("compact_400", "bf16", "nhd", 16, 8, 128, 32, 1024, 400, index="s32"),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def _draw_attention(rng):
    io = rng.choice(["bf16", "bf16", "f16", "f16", "f32"])
    cache = rng.choice([io, io, "e4m3", "e5m2"])
    table = rng.choice(["packed", "packed", "ragged", "offsets"])
    layout = rng.choice(["nhd", "hnd", "packed"] if table == "offsets"
                        else ["nhd", "hnd", "packed", "packed_k", "vllm"])
    block = rng.choice([8, 16, 16, 32, 64, 128])
    heads = rng.choice([1, 2, 3, 4, 8])
    group = rng.choice([1, 2, 4, 5, 7, 8])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    kind = rng.choice(["decode", "decode", "drafts", "chunk", "mixed"])
    seed = rng.randrange(1 << 20)
    scales = rng.choice(["tensor", "head", "block"] if table != "offsets" else ["tensor", "head"])
    more = {"index": rng.choice(["s32", "s64"]), "lens_seed": seed, "scales": scales,
            "window": rng.choice([0, 0, 0, _log_uniform(rng, 16, 4096)]),
            "softcap": rng.choice([0.0, 0.0, 30.0])}
    if kind == "decode":
        hi = _log_uniform(rng, 1, 24000)
        seqs = _log_uniform(rng, 1, max(1, min(200, (1 << 28) // (hi * heads * dim))))
    elif kind == "drafts":
        hi = _log_uniform(rng, 8, 8000)
        seqs = _log_uniform(rng, 1, max(1, min(64, (1 << 27) // (hi * heads * dim))))
        more |= {"new_lo": rng.randint(1, 3), "new_hi": rng.randint(3, 8)}
    else:
        hi = _log_uniform(rng, 64, 6000)
        new = _log_uniform(rng, 17, min(hi, 2048))
        seqs = _log_uniform(rng, 1, max(1, min(24, (1 << 28) // (hi * heads * group * new),
                                               (1 << 27) // (hi * heads * dim))))
        more |= {"new_lo": max(1, new // 2), "new_hi": new}
        if kind == "mixed":
            more |= {"few": 1, "few_of": 2}
    lo = max(1, min(hi, _log_uniform(rng, max(1, hi // 8), hi)))
    return _attention("", io, cache, layout, table, block, heads, group, dim, seqs, lo, hi, **more)


def _draw_rope(rng):
    io = rng.choice(["bf16", "bf16", "f16", "f32"])
    cache = rng.choice([io, io, "e4m3", "e5m2"])
    dim = rng.choice([64, 80, 96, 128, 128, 256])
    rot = rng.choice([dim, dim, dim // 2, dim // 4])
    seqs = _log_uniform(rng, 1, 256)
    hi = rng.choice([1, _log_uniform(rng, 1, 4096)])
    heads = rng.choice([1, 2, 4, 8])
    group = rng.choice([1, 2, 4, 5, 8])
    seqs = max(1, min(seqs, (1 << 28) // (hi * heads * (group + 2) * dim * _BYTES[io])))
    return _rope("", io, cache, rng.choice(["nhd", "hnd", "packed", "packed_k", "vllm"]),
                 rng.choice([8, 16, 32, 64]), heads, group, dim, rot,
                 rng.choice(["half", "interleaved"]), seqs, max(1, hi // 2), hi,
                 far=_log_uniform(rng, 8192, 1 << 20), base=rng.choice([10000.0, 500000.0]),
                 scaling=rng.choice(["none", "linear", "ntk", "yarn", "llama3"]),
                 fused=rng.random() < 0.7, scales=rng.choice(["tensor", "head"]),
                 index=rng.choice(["s32", "s64"]), lens_seed=rng.randrange(1 << 20))


def _draw_copy(rng):
    cache = rng.choice(["bf16", "f16", "f32", "e4m3"])
    block = rng.choice([8, 16, 32, 64])
    heads = rng.choice([1, 2, 3, 4, 8])
    dim = rng.choice([64, 80, 96, 128, 256])
    layers = rng.choice([1, 16, 22, 32, 40])
    page = block * heads * dim * _BYTES[cache]
    most = max(2, min(8192, (1 << 30) // (page * layers)))
    pairs = _log_uniform(rng, 1, max(1, most * 2 // 5))
    return _copy("", cache, rng.choice(["nhd", "hnd", "packed", "packed_k", "vllm"]), block, heads,
                 dim, layers, max(2 * pairs, min(most, 4 * pairs)), pairs,
                 index=rng.choice(["s32", "s64"]))


def draw(rng):
    kind = rng.choice([_draw_attention, _draw_attention, _draw_attention, _draw_rope, _draw_rope,
                       _draw_copy])
    case = kind(rng)
    del case["name"]
    return case


# ---------------------------------------------------------------------------
# What a case has to do.  Lengths depend on the case alone.

def _lens(case):
    """(cached tokens, new tokens) of each sequence."""
    rng = random.Random(case["lens_seed"])
    if case["op"] == "rope_write":
        new = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
        return [n + rng.randrange(max(1, case["far"] - n)) for n in new], new
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["seqs"])]
    new = [min(n, rng.randint(case["new_lo"], case["new_hi"])) for n in lens]
    new = [1 if i % case["few_of"] < case["few"] else n for i, n in enumerate(new)]
    return lens, new


def _attended(case, n, m):
    """(attended pairs, distinct keys read) of m new tokens of n."""
    w = case["window"] or n
    pairs = sum(min(p + 1, w) for p in range(n - m, n))
    return pairs, n - max(0, n - m + 1 - w)


def work(case):
    item = _BYTES[case["cache"]]
    index = 4 if case["index"] == "s32" else 8
    if case["op"] == "copy_blocks":
        page = case["block"] * case["heads"] * case["dim"] * item
        pairs = case["pairs"]
        return {"bytes": 4 * page * pairs * case["layers"] + 2 * pairs * index, "flops": 0}
    lens, new = _lens(case)
    total = sum(new)
    io, h, g, d = _BYTES[case["io"]], case["heads"], case["group"], case["dim"]
    if case["op"] == "rope_write":
        kept = total - case["padded"]
        moved = total * 2 * h * g * d * io + kept * 2 * h * d * (io + item)
        return {"bytes": moved + total * 2 * index + case["rot"] * 2,
                "flops": 3 * case["rot"] * h * (g * total + kept)}
    each = [_attended(case, n, m) for n, m in zip(lens, new)]
    keys = sum(k for _, k in each)
    entries = {"packed": sum(-(-k // case["block"]) for _, k in each) * index,
               "ragged": keys * index, "offsets": sum(-(-k // case["block"]) for _, k in each) * 8}
    moved = keys * 2 * h * d * item + total * h * g * (2 * d * io + 4)
    return {"bytes": moved + entries[case["table"]] + len(lens) * (index + 4),
            "flops": 4 * d * h * g * sum(p for p, _ in each)}


# ---------------------------------------------------------------------------
# Inputs.

def _storage(case, shape_of, gen, lead=()):
    """K and V storages (axes in memory order) of a layout, filled with
    rows ~ N(0, 1) or, for FP8, the codes of such rows at their scale."""
    dt, top = _DTYPE[case["cache"]], _FP8_MAX.get(case["cache"])

    def one(order):
        t = torch.empty((*lead, *[shape_of[a] for a in order]), dtype=dt, device=_DEVICE)
        flat = t.view(-1)
        for part in flat.split(1 << 26):
            if top is None:
                part.normal_(generator=gen)
            else:
                x = torch.empty(part.shape, dtype=torch.float32, device=_DEVICE)
                part.copy_(x.normal_(generator=gen).mul_(top / 4.5).clamp_(-top, top))
        return t

    orders = _orders(case["layout"])
    return one(orders[0]), one(orders[1])


def _orders(layout):
    """Storage axes of K and V: b(lock), o(ffset), h(ead), d(im), or d split
    as p, x."""
    return {"nhd": ("bohd", "bohd"), "hnd": ("bhod", "bhod"), "packed": ("bhpox", "bhpox"),
            "packed_k": ("bhpox", "bohd"), "vllm": ("bhpox", "bhdo")}[layout]


def _shape_of(case, blocks):
    x = 16 // _BYTES[case["cache"]]
    return {"b": blocks, "o": case["block"], "h": case["heads"], "d": case["dim"],
            "p": case["dim"] // x, "x": x}


def _logical(t, order, lead=0):
    """The view [..., b, o, h, d] or [..., b, o, h, p, x] of a storage."""
    axes = "bohpx" if "p" in order else "bohd"
    return t.permute(list(range(lead)) + [lead + order.index(a) for a in axes])


def _paged_cache(case, k, v):
    """The framework's handle of a layer's cache."""
    from kvx_amd import paged
    from kvx_amd.abi import Layout

    kinds = {"bohd": Layout.BLOCK_NHD, "bhod": Layout.BLOCK_HND, "bhpox": Layout.BLOCK_HND_PACKED}
    ko, vo = _orders(case["layout"])
    blocks = k.shape[0]
    if vo in kinds:
        return paged.PagedCache(k, v, kinds[ko], kinds[vo], blocks, case["block"], case["heads"],
                                case["dim"])
    return paged.PagedCache(paged.custom_view(k, ko), paged.custom_view(v, vo),
                            Layout.BLOCK_CUSTOM, Layout.BLOCK_CUSTOM, blocks, case["block"],
                            case["heads"], case["dim"])


def _scale_values(case, gen, blocks):
    """K and V scales of an FP8 cache as a calibration gives them: the amax
    of N(0, 1) rows over the largest code; "block": one for each page and
    head."""
    if case["cache"] == case["io"]:
        return None, None
    n = {"tensor": (1,), "head": (case["heads"],), "block": (blocks, case["heads"])}[case["scales"]]
    u = torch.rand((2, *n), generator=gen, device=_DEVICE)
    s = (4.0 + u) / _FP8_MAX[case["cache"]]
    return s[0].contiguous(), s[1].contiguous()


def _scales(case, ks, vs):
    """The framework's arguments for them."""
    if ks is None:
        return None, None
    from kvx_amd import paged
    from kvx_amd.abi import ScaleGranularity

    g = {"tensor": ScaleGranularity.PER_TENSOR, "head": ScaleGranularity.PER_HEAD,
         "block": ScaleGranularity.PER_BLOCK_HEAD}[case["scales"]]
    return paged.Scales(ks, g), paged.Scales(vs, g)


def _block_table(case, lens, seed):
    """Random page ids for every cached token: [S, width] on the CPU, -1
    behind a sequence's last page, and the pool's size."""
    need = torch.tensor([-(-n // case["block"]) for n in lens])
    used = int(need.sum())
    pool = used + max(4, used // 8)
    ids = torch.randperm(pool, generator=torch.Generator().manual_seed(seed))[:used]
    table = torch.full((len(lens), int(need.max())), -1, dtype=torch.int64)
    table[torch.arange(table.shape[1])[None] < need[:, None]] = ids
    return table, pool


def prepare(case, seed):
    state = {"attention": _attention_inputs, "rope_write": _rope_inputs,
             "copy_blocks": _copy_inputs}[case["op"]](case, seed)
    if own:
        state.update(_handles(state))
    return state


def _handles(state):
    """What a user's program keeps beside the tensors: the caches, tables
    and rotary settings in the framework's types."""
    from kvx_amd import paged

    case = state["case"]
    if case["op"] == "copy_blocks":
        return {"caches": [_paged_cache(case, k, v) for k, v in zip(state["k"], state["v"])]}
    got = {"scales": _scales(case, state["ks"], state["vs"])}
    if case["op"] == "rope_write":
        got["rope"] = paged.Rope(state["inv_freq"], case["style"] == "interleaved",
                                 state["magnitude"])
    if case.get("table") == "offsets":
        got["cache"] = _paged_cache(case, state["pool"], state["pool"])
        got["table"] = paged.pool_table(got["cache"], state["indices"])
        return got
    got["cache"] = _paged_cache(case, state["k"], state["v"])
    if case["op"] == "attention":
        got["table"] = (paged.RaggedTable(state["indices"], state["ragged"])
                        if case["table"] == "ragged" else state["indices"])
    return got


def _copy_inputs(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    k, v = _storage(case, _shape_of(case, case["blocks"]), gen, (case["layers"],))
    ids = torch.randperm(case["blocks"], generator=torch.Generator().manual_seed(seed))
    pairs = ids[: 2 * case["pairs"]].reshape(-1, 2).to(_DEVICE, _INDEX[case["index"]])
    return {"case": case, "k": k, "v": v, "pairs": pairs}


def _attention_inputs(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    lens, new = _lens(case)
    table, blocks = _block_table(case, lens, seed)
    idx = _INDEX[case["index"]]
    dev = torch.device(_DEVICE)
    state = {"case": case, "max_len": max(lens), "max_new": max(new),
             "lens": torch.tensor(lens, dtype=idx, device=dev)}
    counts = torch.tensor(new)
    indptr = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(counts, 0)])
    state["indptr"] = None if max(new) == 1 else indptr.to(dev, torch.int32)
    shape = _shape_of(case, blocks)
    state["ks"], state["vs"] = _scale_values(case, gen, blocks)
    if case["table"] == "offsets":  # one pool, K of page b at 2b and V at 2b + 1
        state["pool"] = _storage(case, dict(shape, b=2 * blocks), gen)[0]
        state["k"], state["v"] = state["pool"][0::2], state["pool"][1::2]
        pair = torch.stack([2 * table, 2 * table + 1], dim=1)[:, None]
        pair[(table < 0)[:, None, None].expand_as(pair)] = 0x7FFFFFFF
        state["indices"] = pair.to(dev, torch.int32)
    else:
        state["k"], state["v"] = _storage(case, shape, gen)
        state["indices"] = table.to(dev, idx)
        if case["table"] == "ragged":
            n = torch.tensor(lens)
            seq = torch.repeat_interleave(torch.arange(len(lens)), n)
            at = torch.arange(int(n.sum())) - (torch.cumsum(n, 0) - n)[seq]
            ptr = torch.cat([torch.zeros(1, dtype=torch.int64), torch.cumsum(n, 0)])
            state["indices"] = table[seq, at // case["block"]].to(dev, idx)
            state["ragged"] = ptr.to(dev, torch.int32)
    state["ids"] = table.clamp(min=0).to(dev)
    total, hq = int(counts.sum()), case["heads"] * case["group"]
    # Trained heads are sharper than random ones: logits of about N(0, 2).
    q = torch.randn((total, hq, case["dim"]), generator=gen, device=dev) * math.sqrt(2.0)
    state["q"] = q.to(_DTYPE[case["io"]])
    state["out"] = torch.empty_like(state["q"])
    state["lse"] = torch.empty((total, hq), dtype=torch.float32, device=dev)
    state["seq"] = torch.repeat_interleave(torch.arange(len(new)), counts).to(dev)
    state["nth"] = (torch.arange(total) - indptr[:-1].repeat_interleave(counts)).to(dev)
    state["new"] = counts.to(dev)
    return state


def _frequencies(case):
    """Inverse frequencies, float32 [rot / 2], and the factor on cosines and
    sines, as the rotary settings of a checkpoint mean them."""
    r, base = case["rot"], case["base"]
    i = torch.arange(0, r, 2, dtype=torch.float64)
    kind, magnitude = case["scaling"], 1.0
    if kind == "ntk":
        base = base * 4.0 ** (r / (r - 2))
    f = base ** (-i / r)
    if kind == "linear":
        f = f / 4.0
    elif kind == "llama3":  # long waves slowed, short kept, between them blended
        turns = 8192.0 * f / (2 * math.pi)
        keep = ((turns - 1.0) / (4.0 - 1.0)).clamp(0, 1)
        f = keep * f + (1 - keep) * f / 8.0
    elif kind == "yarn":
        dim_at = lambda turns: (r * math.log(8192 / (turns * 2 * math.pi))  # noqa: E731
                                / (2 * math.log(base)))
        low, high = max(math.floor(dim_at(32.0)), 0), min(math.ceil(dim_at(1.0)), r - 1)
        high = high + 0.001 if high == low else high
        slow = ((i / 2 - low) / (high - low)).clamp(0, 1)
        f = slow * f / 8.0 + (1 - slow) * f
        magnitude = 0.1 * math.log(8.0) + 1.0
    return f.float(), magnitude


def _rope_inputs(case, seed):
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    dev = torch.device(_DEVICE)
    lens, new = _lens(case)
    counts = torch.tensor(new)
    total = int(counts.sum())
    seq = torch.repeat_interleave(torch.arange(len(new)), counts)
    nth = torch.arange(total) - (torch.cumsum(counts, 0) - counts)[seq]
    positions = (torch.tensor(lens) - counts)[seq] + nth
    # The pool holds each sequence's last pages, and as many others.
    bs = case["block"]
    first = (positions[nth == 0] // bs)
    table, _ = _block_table(case, [int(n) - int(f) * bs for n, f in zip(lens, first)], seed)
    blocks = 2 * int((table >= 0).sum())
    slots = table[seq, positions // bs - first[seq]] * bs + positions % bs
    pad = torch.randperm(total, generator=torch.Generator().manual_seed(case["lens_seed"]))
    slots[pad[: case["padded"]]] = -1
    idx = _INDEX[case["index"]]
    state = {"case": case, "slots": slots.to(dev, idx), "positions": positions.to(dev, idx)}
    state["k"], state["v"] = _storage(case, _shape_of(case, blocks), gen)
    state["ks"], state["vs"] = _scale_values(case, gen, blocks)
    h, g, d = case["heads"], case["group"], case["dim"]
    qkv = torch.randn((total, h * (g + 2), d), generator=gen, device=dev).to(_DTYPE[case["io"]])
    parts = qkv.split([h * g, h, h], dim=1)
    state["q"], state["key"], state["value"] = (
        parts if case["fused"] else [p.contiguous() for p in parts])
    state["q_out"] = torch.empty((total, h * g, d), dtype=qkv.dtype, device=dev)
    inv_freq, state["magnitude"] = _frequencies(case)
    state["inv_freq"] = inv_freq.to(dev)
    return state


# ---------------------------------------------------------------------------
# One pass.

def run(state):
    op = state["case"]["op"]
    if own:
        return {"attention": _own_attention, "rope_write": _own_rope,
                "copy_blocks": _own_copy}[op](state)
    return {"attention": _plain_attention, "rope_write": _plain_rope,
            "copy_blocks": _plain_copy}[op](state)


def _check(status):
    if status != 0:
        raise RuntimeError(f"kvx status {status}")


def _own_attention(state):
    from kvx_amd import paged

    case = state["case"]
    ks, vs = state["scales"]
    _check(paged.attention(state["cache"], state["q"], state["out"], state["table"],
                           state["lens"], state["indptr"], window=case["window"],
                           softcap=case["softcap"], lse=state["lse"],
                           max_seq_len=state["max_len"], max_query_len=state["max_new"],
                           k_scale=ks, v_scale=vs))
    return {"out": state["out"], "lse": state["lse"]}


def _own_rope(state):
    from kvx_amd import paged

    ks, vs = state["scales"]
    _check(paged.rope_write_kv(state["cache"], state["q"], state["key"], state["value"],
                               state["positions"], state["rope"], state["slots"],
                               query_out=state["q_out"], k_scale=ks, v_scale=vs))
    return {"q": state["q_out"], "k": state["k"], "v": state["v"]}


def _own_copy(state):
    from kvx_amd import paged

    _check(paged.copy_blocks(state["caches"], state["pairs"]))
    return {"k": state["k"], "v": state["v"]}


def _raw(t):
    """FP8 codes as bytes, which torch indexes; other types as they are."""
    return t.view(torch.uint8) if t.dtype.itemsize == 1 else t


def _cached_rows(t, order, ids, block, length, scale):
    """Rows 0..length of every sequence, in 32 bits: [S, length, H, D]."""
    at = torch.arange(length, device=ids.device)
    pages = ids[:, at // block]
    rows = _raw(_logical(t, order))[pages, (at % block)[None].expand_as(pages)]
    rows = rows.view(t.dtype).float().flatten(3)
    if scale is None:
        return rows
    s = scale[pages] if scale.dim() == 2 else scale
    return rows * s[..., None]


def _plain_attention(state):
    case = state["case"]
    ko, vo = _orders(case["layout"])
    h, g, d = case["heads"], case["group"], case["dim"]
    length, most = state["max_len"], state["max_new"]
    k = _cached_rows(state["k"], ko, state["ids"], case["block"], length, state["ks"])
    v = _cached_rows(state["v"], vo, state["ids"], case["block"], length, state["vs"])
    k = k.permute(0, 2, 3, 1).contiguous()
    v = v.permute(0, 2, 1, 3).contiguous()
    seqs = k.shape[0]
    q = torch.zeros((seqs, most, h * g, d), dtype=torch.float32, device=k.device)
    q[state["seq"], state["nth"]] = state["q"].float()
    q = q.view(seqs, most, h, g, d).permute(0, 2, 1, 3, 4).reshape(seqs, h, most * g, d)
    s = (q @ k) * (1.0 / math.sqrt(d))
    if case["softcap"]:
        s = case["softcap"] * torch.tanh(s / case["softcap"])
    t = torch.arange(length, device=k.device)
    pos = (state["lens"].long() - state["new"])[:, None] + torch.arange(most, device=k.device)
    seen = t <= pos[..., None]
    if case["window"]:
        seen &= t > pos[..., None] - case["window"]
    s = s.view(seqs, h, most, g, length).masked_fill_(~seen[:, None, :, None], -math.inf)
    top = s.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    p = s.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(seqs, h, most * g, length) @ v
    o = o.view(seqs, h, most, g, d) / total
    lse = (top + total.log())[..., 0]
    o = o.permute(0, 2, 1, 3, 4).reshape(seqs, most, h * g, d)
    lse = lse.permute(0, 2, 1, 3).reshape(seqs, most, h * g)
    at = state["seq"], state["nth"]
    return {"out": o[at].to(state["q"].dtype), "lse": lse[at]}


def _rotated(x, cos, sin, rot, interleaved):
    """x [T, H, D] in 32 bits, cos and sin [T, 1, rot / 2]."""
    r, rest = x[..., :rot], x[..., rot:]
    if interleaved:
        a, b = r[..., 0::2], r[..., 1::2]
        r = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = r[..., : rot // 2], r[..., rot // 2:]
        r = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([r, rest], dim=-1)


def _plain_write(case, t, order, rows, slots, scale):
    if scale is not None:
        top = _FP8_MAX[case["cache"]]
        rows = (rows / scale[:, None]).clamp(-top, top)
    rows = _raw(rows.to(t.dtype))
    view = _raw(_logical(t, order))
    view[slots // case["block"], slots % case["block"]] = rows.reshape(
        rows.shape[0], *view.shape[2:])


def _plain_rope(state):
    case = state["case"]
    angle = state["positions"].double()[:, None] * state["inv_freq"].double()
    cos = (angle.cos() * state["magnitude"]).float()[:, None]
    sin = (angle.sin() * state["magnitude"]).float()[:, None]
    turn = (cos, sin, case["rot"], case["style"] == "interleaved")
    q = _rotated(state["q"].float(), *turn).to(state["q"].dtype)
    key, value, slots = _rotated(state["key"].float(), *turn), state["value"].float(), state["slots"]
    if case["padded"]:
        kept = slots >= 0
        key, value, slots = key[kept], value[kept], slots[kept]
    ko, vo = _orders(case["layout"])
    slots = slots.long()
    _plain_write(case, state["k"], ko, key, slots, state["ks"])
    _plain_write(case, state["v"], vo, value, slots, state["vs"])
    return {"q": q, "k": state["k"], "v": state["v"]}


def _plain_copy(state):
    src, dst = state["pairs"][:, 0].long(), state["pairs"][:, 1].long()
    for t in (_raw(state["k"]), _raw(state["v"])):
        t[:, dst] = t[:, src]
    return {"k": state["k"], "v": state["v"]}


# ---------------------------------------------------------------------------
# The definitions in 64 bits.

def exact(case, seed):
    if case["op"] == "attention":
        return _exact_attention(prepare(case, seed))
    if case["op"] == "rope_write":
        return _exact_rope(prepare(case, seed))
    return None  # copies: no computed numbers


def _dequantized(t, order, pages, head, scale):
    """All rows of some pages of one head, in 64 bits: [rows, D]."""
    rows = _raw(_logical(t, order))[pages][:, :, head].view(t.dtype).double().flatten(2)
    if scale is not None:
        s = scale.double()
        rows = rows * (s[pages, head][:, None, None] if s.dim() == 2
                       else s[head if s.numel() > 1 else 0])
    return rows.flatten(0, 1)


def _exact_attention(state):
    """Sequence by sequence, head by head: each new token's softmax over the
    positions it sees."""
    case = state["case"]
    ko, vo = _orders(case["layout"])
    g, d = case["group"], case["dim"]
    lens, new = _lens(case)
    out = torch.empty(state["q"].shape, dtype=torch.float64, device=_DEVICE)
    lse = torch.empty(state["lse"].shape, dtype=torch.float64, device=_DEVICE)
    first = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        pages = state["ids"][s, : -(-n // case["block"])]
        place = torch.arange(n, device=_DEVICE)
        now = torch.arange(n - m, n, device=_DEVICE)[:, None]
        hidden = (place > now) | (place <= now - (case["window"] or n))
        for h in range(case["heads"]):
            k = _dequantized(state["k"], ko, pages, h, state["ks"])[:n]
            v = _dequantized(state["v"], vo, pages, h, state["vs"])[:n]
            for j in range(h * g, h * g + g):
                logits = state["q"][first: first + m, j].double() @ k.T.contiguous() / d ** 0.5
                if case["softcap"]:
                    logits = (logits / case["softcap"]).tanh() * case["softcap"]
                logits[hidden] = -math.inf
                each = torch.logsumexp(logits, dim=1)
                lse[first: first + m, j] = each
                out[first: first + m, j] = torch.exp(logits - each[:, None]) @ v
        first += m
    return {"out": out, "lse": lse}


def _exact_rope(state):
    """Each pair as a complex number, turned by exp(i * position * frequency)."""
    case = state["case"]
    r = case["rot"]
    angle = torch.outer(state["positions"].double(), state["inv_freq"].double())
    turn = torch.polar(torch.full_like(angle, state["magnitude"]), angle)[:, None]

    def rotate(x):
        x = x.double()
        if case["style"] == "interleaved":
            z = torch.view_as_complex(x[..., :r].unflatten(-1, (r // 2, 2)).contiguous()) * turn
            x[..., :r] = torch.view_as_real(z).flatten(-2)
        else:
            z = torch.complex(x[..., : r // 2].contiguous(), x[..., r // 2: r].contiguous()) * turn
            x[..., : r // 2], x[..., r // 2: r] = z.real, z.imag
        return x

    def written(t, order, rows, scale):
        full = t.double()
        at = _logical(full, order)
        if scale is not None:
            rows = (rows / scale.double()[:, None]).clamp(-_FP8_MAX[case["cache"]],
                                                          _FP8_MAX[case["cache"]])
        slots = state["slots"].long()
        kept = slots >= 0
        page, place = slots[kept] // case["block"], slots[kept] % case["block"]
        at[page, place] = rows[kept].reshape(-1, *at.shape[2:])
        return full

    ko, vo = _orders(case["layout"])
    q = rotate(state["q"].clone())
    k = written(state["k"], ko, rotate(state["key"].clone()), state["ks"])
    v = written(state["v"], vo, state["value"].double(), state["vs"])
    return {"q": q, "k": k, "v": v}
