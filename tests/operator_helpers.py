"""Shared by the tests of kvx_ext.h's operators: caches of every layout and
table format filled through torch, and the operators' definitions in 64 bits
on the CPU with bounds on how far 32-bit arithmetic may be from them."""
from __future__ import annotations

import math

import torch

from kvx_amd import paged
from kvx_amd.abi import Layout, ScaleGranularity

DT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32,
      "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
TOP = {"e4m3": 448.0, "e5m2": 57344.0}
# Half a rounding step relative to the value.
HALF = {k: torch.finfo(v).eps / 2 for k, v in DT.items()}
U32 = 2.0 ** -24

LAYOUTS = {"nhd": ("bohd", "bohd"), "hnd": ("bhod", "bhod"), "packed": ("bhpox", "bhpox"),
           "packed_k": ("bhpox", "bohd"), "vllm": ("bhpox", "bhdo"), "dim_outer": ("bdho", "bdho"),
           "block_inner": ("ohdb", "ohdb")}
_CODE = {"bohd": Layout.BLOCK_NHD, "bhod": Layout.BLOCK_HND, "bhpox": Layout.BLOCK_HND_PACKED}


def storage_of(order, nb, bs, H, D, dtype, device, x):
    size = {"b": nb, "o": bs, "h": H, "d": D, "p": D // x if x else 0, "x": x}
    return torch.empty([size[c] for c in order], dtype=dtype, device=device)


def make_cache(layout, nb, bs, H, D, dt, device, x=None):
    ko, vo = LAYOUTS[layout]
    x = x or 16 // DT[dt].itemsize
    k = storage_of(ko, nb, bs, H, D, DT[dt], device, x)
    v = storage_of(vo, nb, bs, H, D, DT[dt], device, x)
    if ko in _CODE and vo in _CODE:
        return paged.PagedCache(k, v, _CODE[ko], _CODE[vo], nb, bs, H, D)
    return paged.PagedCache(paged.custom_view(k, ko), paged.custom_view(v, vo),
                            Layout.BLOCK_CUSTOM, Layout.BLOCK_CUSTOM, nb, bs, H, D)


def logical(t, layout):
    """[nb, bs, H, D] or [nb, bs, H, D / x, x] view of a cache tensor."""
    if layout == Layout.BLOCK_HND:
        return t.permute(0, 2, 1, 3)
    if layout == Layout.BLOCK_HND_PACKED:
        return t.permute(0, 3, 1, 2, 4)
    return t


def raw(t):
    return t.view(torch.uint8) if t.dtype.itemsize == 1 else t


def set_rows(t, layout, rows):
    """Fills a whole cache tensor from rows [nb, bs, H, D] of its dtype."""
    view = raw(logical(t, layout))
    view.copy_(raw(rows.to(t.device)).reshape(view.shape))


def get_rows(t, layout):
    view = raw(logical(t, layout))
    return view.reshape(*view.shape[:3], -1).view(t.dtype)


def fp8(x, dt):
    return x.clamp(-TOP[dt], TOP[dt]).to(DT[dt])


def scale_arg(values, kind):
    g = {"tensor": ScaleGranularity.PER_TENSOR, "head": ScaleGranularity.PER_HEAD,
         "block": ScaleGranularity.PER_BLOCK, "block_head": ScaleGranularity.PER_BLOCK_HEAD}[kind]
    return paged.Scales(values, g)


def scale_rows(values, kind, nb, H):
    """[nb, H] float64 of a scale."""
    v = values.double().cpu()
    if kind == "head":
        v = v[None]
    elif kind == "block":
        v = v[:, None]
    elif kind == "tensor":
        v = v.reshape(1, 1)
    return v.expand(nb, H)


def attention_reference(q, rows_of, lens, new, G, *, causal=True, scale, window=0, softcap=0.0,
                        u_p=0.0, cap_rel=None):
    """out, lse in float64 and how far 32-bit kernels may be from them.

    rows_of(s) -> (k, v [n, H, D] float64, there [n] bool): the sequence's
    tokens that the table holds.  With c = (D + 8) 2^-24 times the sum of the
    absolute products, a logit is off by at most d = c (+ cap 2^-21 for the
    softcap's tanh; with `cap_rel` that part of the capped logit, and cap 2^-149
    where tanh's argument is subnormal), every weight by a relative 2 d + u_p (u_p: its rounding
    for the matrix cores), and sums over n weights by n 2^-24."""
    T, Hq, D = q.shape
    out = torch.zeros((T, Hq, D), dtype=torch.float64)
    lse = torch.full((T, Hq), -math.inf, dtype=torch.float64)
    tol_o = torch.zeros_like(out)
    tol_l = torch.zeros_like(lse)
    row = 0
    for s, (n, m) in enumerate(zip(lens, new)):
        k, v, there = rows_of(s)
        held = k.shape[0]
        for i in range(m):
            pos = n - m + i
            t = torch.arange(held)
            seen = there & (t < n)
            if causal:
                seen &= t <= pos
                if window:
                    seen &= t > pos - window
            if seen.any():
                kk, vv = k[seen], v[seen]
                qq = q[row].double().reshape(-1, G, D)
                x = torch.einsum("hgd,nhd->hgn", qq, kk) * scale
                size = torch.einsum("hgd,nhd->hgn", qq.abs(), kk.abs()) * abs(scale)
                d = (D + 8) * U32 * size.amax(-1)
                if softcap:
                    x = softcap * torch.tanh(x / softcap)
                    if cap_rel is None:
                        d = d + softcap * 2.0 ** -21
                    else:
                        d = d + cap_rel * x.abs().amax(-1) + softcap * 2.0 ** -149
                l = torch.logsumexp(x, -1)
                p = torch.exp(x - l[..., None])
                o = torch.einsum("hgn,nhd->hgd", p, vv)
                a = torch.einsum("hgn,nhd->hgd", p, vv.abs())
                cnt = int(seen.sum())
                out[row] = o.reshape(Hq, D)
                lse[row] = l.reshape(Hq)
                rel = 2 * d + u_p + (cnt + 16) * U32
                tol_o[row] = (rel[..., None] * a).reshape(Hq, D)
                tol_l[row] = (d + (cnt + 16) * U32 + 4 * U32 * l.abs()).reshape(Hq)
            row += 1
    return out, lse, tol_o, tol_l


class AttentionCase:
    """A batch for paged.attention: cache, table, queries, and its result in
    64 bits."""

    cap_rel = None  # see attention_reference

    def __init__(self, *, io="bf16", cache=None, layout="nhd", table="packed", bs=16, H=2, G=4,
                 D=64, lens=(37,), new=None, index=torch.int32, scales="tensor", seed=0,
                 causal=True, window=0, softcap=0.0, scale=None, extra_rows=0, indptr=None,
                 stale=None, holes=(), device="cuda", x=None, spare=3, indptr_dtype=torch.int32):
        g = torch.Generator().manual_seed(seed)
        self.io, self.cdt = io, cache or io
        self.lens = list(lens)
        self.new = [1] * len(self.lens) if new is None else list(new)
        self.H, self.G, self.D, self.bs = H, G, D, bs
        self.layout, self.tkind = layout, table
        self.args = dict(causal=causal, window=window, softcap=softcap)
        self.scale = D ** -0.5 if scale is None else scale
        S = len(self.lens)
        need = [-(-max(n, 0) // bs) for n in self.lens]
        width = max(need + [1])
        nb = sum(need) + spare
        ids = torch.randperm(nb, generator=g)
        tb = torch.full((S, width), -1, dtype=torch.int64)
        at = 0
        for s in range(S):
            tb[s, : need[s]] = ids[at: at + need[s]]
            at += need[s]
        for s, j in holes:  # block ids that the kernels must skip
            tb[s, j] = (-7, nb, nb + 5)[(s + j) % 3]
        self.tb, self.nb = tb, nb
        rows = []
        self.kv_scales = [None, None]
        scale_vals = [None, None]
        for which in range(2):
            r = torch.randn((nb, bs, H, D), generator=g)
            if which == 0:
                r = r * 1.5
            if self.cdt in TOP:
                shape = {"tensor": (1,), "head": (H,), "block": (nb,), "block_head": (nb, H)}[scales]
                sv = (0.5 + torch.rand(shape, generator=g)) * 4.0 / TOP[self.cdt]
                scale_vals[which] = scale_rows(sv, scales, nb, H)
                self.kv_scales[which] = scale_arg(sv.to(device), scales)
                r = fp8(r / scale_vals[which][:, None, :, None], self.cdt)
            else:
                r = r.to(DT[self.cdt])
            rows.append(r)
        exact = []
        for which in range(2):
            e = rows[which].double()
            if scale_vals[which] is not None:
                e = e * scale_vals[which][:, None, :, None]
            exact.append(e)
        if stale is not None:  # slots that hold no token of any sequence
            used = torch.zeros((nb, bs), dtype=torch.bool)
            for s in range(S):
                for t in range(max(self.lens[s], 0)):
                    b = int(tb[s, t // bs])
                    if 0 <= b < nb:
                        used[b, t % bs] = True
            for r in rows:
                raw(r)[~used] = raw(torch.full((1,), stale).to(r.dtype))[0]
        self.rows, self.exact = rows, exact
        if table == "offsets":
            pool, kv = paged.alloc_block_pool(nb, bs, H, D, DT[self.cdt], device,
                                              _CODE[LAYOUTS[layout][0]],
                                              x or 16 // DT[self.cdt].itemsize)
            set_rows(kv.key_cache, kv.k_layout, rows[0])
            set_rows(kv.value_cache, kv.v_layout, rows[1])
            pair = torch.stack([2 * tb, 2 * tb + 1], 1)[:, None]
            bad = ((tb < 0) | (tb >= nb))[:, None, None].expand_as(pair)
            pair[bad] = 0x7FFFFFFF
            self.cache = pool
            self.kv = kv
            self.table = paged.pool_table(pool, pair.to(device, torch.int32))
        else:
            self.cache = self.kv = make_cache(layout, nb, bs, H, D, self.cdt, device, x)
            set_rows(self.cache.key_cache, self.cache.k_layout, rows[0])
            set_rows(self.cache.value_cache, self.cache.v_layout, rows[1])
            if table == "ragged":
                flat = [tb[s, t // bs] for s in range(S) for t in range(max(self.lens[s], 0))]
                ptr = torch.tensor([0] + [max(n, 0) for n in self.lens]).cumsum(0)
                flat = torch.stack(flat) if flat else torch.zeros(1, dtype=torch.int64)
                self.table = paged.RaggedTable(flat.to(device, index), ptr.to(device, torch.int32))
            else:
                self.table = tb.to(device, index)
        self.lens_t = torch.tensor(self.lens, dtype=index, device=device)
        total = sum(self.new)
        ptr = torch.tensor([0] + self.new).cumsum(0)
        plain = new is None and extra_rows == 0
        self.indptr = None if plain else ptr.to(device, indptr_dtype)
        self.T = total + extra_rows
        self.total = total
        self.q = torch.randn((self.T, H * G, D), generator=g).to(DT[io])
        self.q_dev = self.q.to(device)
        self.out = torch.full((self.T, H * G, D), 7.0, dtype=DT[io], device=device)
        self.lse = torch.full((self.T, H * G), 7.0, dtype=torch.float32, device=device)

    def rows_of(self, s):
        n = max(self.lens[s], 0)
        b = self.tb[s].repeat_interleave(self.bs)[:n]
        o = torch.arange(n) % self.bs
        there = (b >= 0) & (b < self.nb)
        b = b.clamp(0, self.nb - 1)
        return self.exact[0][b, o], self.exact[1][b, o], there

    def reference(self):
        u_p = 0.0 if self.io == "f32" else HALF[self.io]
        return attention_reference(self.q[: self.total], self.rows_of, self.lens, self.new, self.G,
                                   scale=self.scale, u_p=u_p, cap_rel=self.cap_rel, **self.args)

    def run(self, **more):
        kw = dict(scale=self.scale, lse=self.lse, max_seq_len=max(self.lens + [0]),
                  max_query_len=max(self.new + [0]), k_scale=self.kv_scales[0],
                  v_scale=self.kv_scales[1], **self.args)
        kw.update(more)
        q, out = kw.pop("q", self.q_dev), kw.pop("out", self.out)
        return paged.attention(self.cache, q, out, self.table, self.lens_t, self.indptr, **kw)

    def check(self, out=None, lse=None):
        torch.cuda.synchronize()
        out = (self.out if out is None else out).cpu()
        ref, ref_l, tol, tol_l = self.reference()
        # the output's own rounding; f16 below its normal range: 2^-25
        tol = tol + HALF[self.io] * (ref.abs() + tol) + (2.0 ** -25 if self.io == "f16" else 1e-37)
        got = out[: self.total].double()
        assert torch.isfinite(got).all()
        over = (got - ref).abs() - tol
        assert (over <= 0).all(), f"out: {over.max().item()} over its bound"
        assert (out[self.total:] == 7.0).all(), "rows behind the last sequence changed"
        if lse is None:
            lse = self.lse
        if lse is not False:
            lse = lse.cpu()
            got = lse[: self.total].double()
            none = ref_l == -math.inf
            assert (got[none] == -math.inf).all()
            assert ((got - ref_l).abs() <= tol_l)[~none].all()
            assert (lse[self.total:] == 7.0).all()
