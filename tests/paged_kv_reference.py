"""The paged cache operators from their definitions in 64 bits, and the bounds that the kernels' roundings allow."""
import math

import torch

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    """Largest relative error of one rounding to `dtype` (normal range)."""
    return torch.finfo(dtype).eps / 2


def tiny_step(dtype):
    """Largest absolute error of one rounding in the subnormal range of `dtype`."""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def make_cache(seqs, page, kv_heads, d, dtype, order, gen, dev, spare=3, fill=float("nan")):
    """Pages for `seqs`, a list of (new, keys), in random order; what no key lies in (page tails, spare pages) holds
    `fill`, unused table entries hold numbers that are no pages.  Returns k_pages, v_pages, table and the list of
    [keys, kv_heads, d] contents that the sequences see."""
    counts = [-(-k // page) for _, k in seqs]
    pages = sum(counts) + spare
    shape = (pages, kv_heads, page, d) if order == "heads" else (pages, page, kv_heads, d)
    pools = [torch.full(shape, fill, dtype=dtype, device=dev) for _ in range(2)]
    views = [p if order == "heads" else p.transpose(1, 2) for p in pools]
    perm = torch.randperm(pages, generator=gen)
    table = torch.full((len(seqs), max(max(counts), 1)), -7, dtype=torch.int32)
    table[:, 1::2] = 2 ** 30
    at, contents = 0, []
    for s, (_, keys) in enumerate(seqs):
        mine = perm[at:at + counts[s]]
        at += counts[s]
        table[s, :counts[s]] = mine.to(torch.int32)
        both = []
        for view in views:
            x = torch.randn(keys, kv_heads, d, generator=gen).to(dtype)
            where = torch.arange(keys)
            if keys:
                view[mine[where // page].to(dev), :, (where % page).to(dev)] = x.to(dev)
            both.append(x)
        contents.append(both)
    return views[0], views[1], table.to(dev), contents


def starts_of(seqs, dev):
    return torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).to(torch.int32).to(dev)


def lens_of(seqs, dev):
    return torch.tensor([k for _, k in seqs], dtype=torch.int32, device=dev)


def seen(n, keys, block, window):
    """[n, keys] truth values: which keys each new token sees."""
    p = (keys - n + torch.arange(n))[:, None]
    j = torch.arange(keys)[None, :]
    ok = (p >= 0) & (j >= 0)
    if block:
        end = (torch.div(p, block, rounding_mode="floor") + 1) * block
        ok = ok & (j < end)
        if window:
            ok = ok & (j >= end - window)
    return ok


def attention(q, k, v, mask, scale, dtype):
    """Output of one sequence and the largest error that its 16-bit and 32-bit roundings allow.
    q [n, heads, d], k and v [keys, kv_heads, d].

    The weights w and the output are each rounded once to `dtype`: half_step * (sum w |v| + |o|).  fp16 weights below the
    normal range lose an absolute tiny_step each, relative to a largest weight of one: tiny_step * sum |v| / l, l = sum of
    weights before the division.  A score is a sum of d products in fp32: off by at most (d + 4) 2^-23 of the sum of its
    absolute products, which moves a weight by that factor, numerator and denominator alike; the exponential, the sums and
    the joins add a few 2^-22 more: 2^-19 covers them for runs of up to thousands of additions of positive terms in
    partial sums of at most a few hundred."""
    n, heads, d = q.shape
    group = heads // k.shape[1]
    q, k, v = (t.double() for t in (q, k, v))
    kk, vv = k.repeat_interleave(group, 1), v.repeat_interleave(group, 1)
    s = torch.einsum("nhd,khd->hnk", q, kk) * scale
    sabs = torch.einsum("nhd,khd->hnk", q.abs(), kk.abs()) * scale
    s = s.masked_fill(~mask.to(s.device), -math.inf)
    top = s.amax(-1, keepdim=True) if s.shape[-1] else s.new_full((heads, n, 1), -math.inf)
    top = torch.where(top.isinf(), torch.zeros_like(top), top)
    e = (s - top).exp()
    l = e.sum(-1, keepdim=True)
    safe = torch.where(l > 0, l, torch.ones_like(l))
    w = e / safe
    o = torch.einsum("hnk,khd->nhd", w, vv)
    a = torch.einsum("hnk,khd->nhd", w, vv.abs())
    worst = (sabs * (w > 0)).amax(-1) if s.shape[-1] else sabs.new_zeros((heads, n))  # [h, n]
    delta = 2 * (d + 4) * 2.0 ** -23 * worst + 2.0 ** -19
    u = half_step(dtype)
    lost = tiny_step(dtype) * torch.einsum("hnk,khd->nhd", (w > 0).double(), vv.abs()) / safe.permute(1, 0, 2)
    bound = u * (a + o.abs()) * (1 + u) + delta.T[..., None] * a + lost + tiny_step(dtype)
    return o, bound


def append(x, norm_eps, weight, rope, cos, sin):
    """Normed and rotated heads x [n, heads, d] in 64 bits; cos, sin [n, d / 2].  Also the sum of the absolute terms of
    each element, to which fp32 errors are relative."""
    y = x.double()
    half = y.shape[-1] // 2
    if norm_eps is not None:
        y = y / (y.square().mean(-1, keepdim=True) + norm_eps).sqrt()
        if weight is not None:
            y = y * weight.double()
    if rope in (None, "none"):
        return y, y.abs()
    c, s = cos.double()[:, None], sin.double()[:, None]
    a, b = (y[..., :half], y[..., half:]) if rope == "halves" else (y[..., 0::2], y[..., 1::2])
    lo, hi = a * c - b * s, b * c + a * s
    lo_abs, hi_abs = (a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs()
    join = (lambda u, v: torch.stack((u, v), -1).flatten(-2)) if rope == "pairs" else (lambda u, v: torch.cat((u, v), -1))
    return join(lo, hi), join(lo_abs, hi_abs)
