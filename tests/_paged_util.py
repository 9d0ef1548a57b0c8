"""Plain float64 forms of the paged cache's operators, and the error bounds of the kernels.

Bounds.  u is the unit roundoff of the 16-bit type (2^-8 bf16, 2^-11 f16).  A score is a
float32 sum of D products: its error, with the exponential's (2^-22) and that of its argument,
is below 2^-12 relative for the weights at the sizes tested (D 2^-24 sum |q k| scale, with
sum |q k| scale < 16 for unit normal q and k).  Weights are rounded to the 16-bit type for the
product with V, and the output once more:
    |out - ref| <= (u + 2^-12) sum_j w_j |v_j| + u |ref| (1 + u) + 2^-24
where the last term covers float16's subnormal results.  lse carries the score's error and
float32 rounding: 2^-12 + 2^-22 |lse|.  The rotation's sine and cosine are off by less than
2^-20 (hardware functions 2^-21, the rounded reduced angle 2^-22).
"""

from __future__ import annotations

import math

import torch

ROUND = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Case:
    """A cache whose unused rows hold NaN, a page table whose unused entries are no page, and
    the packed new tokens of ``news`` over sequences of ``lens`` positions."""

    def __init__(self, news, lens, *, dtype=torch.bfloat16, dim=128, hq=8, hkv=2, page=16,
                 seed=0, layout="nhd", window=None):
        from dsa_b200 import paged

        g = torch.Generator().manual_seed(seed)
        self.news, self.lens, self.window = list(news), list(lens), window
        self.dtype, self.dim, self.hq, self.hkv, self.page = dtype, dim, hq, hkv, page
        per = [-(-max(n, 0) // page) for n in lens]
        total, width = sum(per) + 2, max(max(per), 1) + 1
        order = torch.randperm(total, generator=g).tolist()
        table = torch.full((len(lens), width), 1 << 30, dtype=torch.int32)
        if layout == "nhd":
            shape, perm = (2, total, page, hkv, dim), (0, 1, 2, 3, 4)
        elif layout == "hnd":      # [pages, heads, page, dim] viewed as [pages, page, heads, dim]
            shape, perm = (2, total, hkv, page, dim), (0, 1, 3, 2, 4)
        else:                      # keys and values of a page next to each other
            shape, perm = (total, 2, page, hkv, dim), (1, 0, 2, 3, 4)
        store = torch.full(shape, math.nan, dtype=dtype).permute(perm)
        self.k, self.v = [], []
        at = 0
        for b, n in enumerate(lens):
            pages = order[at:at + per[b]]
            at += per[b]
            table[b, :per[b]] = torch.tensor(pages, dtype=torch.int32)
            k = torch.randn(max(n, 0), hkv, dim, generator=g).to(dtype)
            v = torch.randn(max(n, 0), hkv, dim, generator=g).to(dtype)
            for i, p in enumerate(pages):
                part = slice(i * page, min((i + 1) * page, n))
                store[0, p, :part.stop - part.start] = k[part]
                store[1, p, :part.stop - part.start] = v[part]
            self.k.append(k.double())
            self.v.append(v.double())
        self.tokens = sum(news)
        self.q = torch.randn(self.tokens, hq, dim, generator=g).to(dtype)
        starts = [0]
        for n in news:
            starts.append(starts[-1] + n)
        self.starts = starts
        self.table = table
        dev = torch.device("cuda")
        # permute(...).contiguous() order is kept by .to(device): rebuild the strided view
        inv = [perm.index(i) for i in range(5)]
        base = store.permute(inv).contiguous().to(dev)
        view = base.permute(perm)
        self.cache = paged.PagedKV(view[0], view[1])
        self.batch = paged.PagedBatch(table.to(dev), torch.tensor(starts, dtype=torch.int32,
                                                                  device=dev),
                                      torch.tensor(self.lens, dtype=torch.int32, device=dev),
                                      max_new=max(news))
        self.qd = self.q.to(dev)

    def reference(self, scale=None, indices=None):
        """(out, sum_j w_j |v_j|, lse) in float64 on the CPU."""
        scale = self.dim ** -0.5 if scale is None else scale
        g = self.hq // self.hkv
        out = torch.zeros(self.tokens, self.hq, self.dim, dtype=torch.float64)
        mag = torch.zeros_like(out)
        lse = torch.full((self.tokens, self.hq), -math.inf, dtype=torch.float64)
        for b, (n, length) in enumerate(zip(self.news, self.lens)):
            for i in range(n):
                t, pos = self.starts[b] + i, length - n + i
                if indices is not None:
                    sel = torch.as_tensor([j for j in indices[t].tolist() if 0 <= j < length],
                                          dtype=torch.long)
                else:
                    lo = 0 if self.window is None else max(0, pos - self.window + 1)
                    sel = torch.arange(lo, max(pos + 1, lo))
                if sel.numel() == 0:
                    continue
                for h in range(self.hkv):
                    heads = slice(h * g, h * g + g)
                    kk, vv = self.k[b][sel, h], self.v[b][sel, h]
                    z = self.q[t, heads].double() @ kk.T * scale
                    w = torch.softmax(z, -1)
                    out[t, heads] = w @ vv
                    mag[t, heads] = w @ vv.abs()
                    lse[t, heads] = torch.logsumexp(z, -1)
        return out, mag, lse


def assert_attention(got, lse, ref, dtype):
    out, mag, want_lse = ref
    u = ROUND[dtype]
    err = (got.double().cpu() - out).abs()
    lim = (u + 2.0 ** -12) * mag + u * (1 + u) * out.abs() + 2.0 ** -24
    bad = ~(err <= lim) & ~(torch.isnan(got.double().cpu()) & torch.isnan(out))
    assert not bad.any(), f"{int(bad.sum())} values off, first at {bad.nonzero()[0].tolist()}"
    if lse is not None:
        got_lse = lse.double().cpu()
        empty = want_lse == -math.inf
        assert torch.equal(got_lse == -math.inf, empty)
        e = (got_lse - want_lse)[~empty].abs()
        assert bool((e <= 2.0 ** -12 + 2.0 ** -22 * want_lse[~empty].abs()).all())


def rotate(x, pos, freq, interleaved):
    """R x in float64: x [T, H, D], pos [T]."""
    half = freq.shape[0]
    ang = pos.double()[:, None] * freq.double()
    c, s = ang.cos()[:, None], ang.sin()[:, None]
    x = x.double().clone()
    a = x[..., 0:2 * half:2].clone() if interleaved else x[..., :half].clone()
    b = x[..., 1:2 * half:2].clone() if interleaved else x[..., half:2 * half].clone()
    lo, hi = a * c - b * s, b * c + a * s
    if interleaved:
        x[..., 0:2 * half:2], x[..., 1:2 * half:2] = lo, hi
    else:
        x[..., :half], x[..., half:2 * half] = lo, hi
    return x
