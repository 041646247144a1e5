"""The 8-bit paged cache's operators, the residual norm and the choice of a
token from their definitions, in 64 bits, with the bound that each result's
arithmetic allows (derived here, per value)."""
import math

import numpy as np
import torch

from tests.paged_reference import TYPES, U32  # noqa: F401

# Half a step among the subnormal numbers, where a rounding is no longer relative: f16's begin at 2^-14 with
# steps of 2^-24; the others' lie under everything here.
TINY = {"f16": 2.0 ** -25, "bf16": 1e-30, "f32": 1e-30}


class Q8Pool:
    """An 8-bit paged cache on the GPU whose unused rows hold a NaN scale."""

    def __init__(self, pages, page_size, kv_heads, hd, seqs, table_stride, gap=0, scale_gap=0):
        from dianoia_b200 import _lib
        self.page_size, self.kv_heads, self.hd, self.pages = page_size, kv_heads, hd, pages
        block = kv_heads * page_size * hd
        self.page_stride, self.scale_stride = block + gap, kv_heads * page_size + scale_gap
        self.raw = [torch.randint(-127, 128, (pages * self.page_stride,), device="cuda", dtype=torch.int8) for _ in range(2)]
        self.raw_scales = [torch.full((pages * self.scale_stride,), float("nan"), device="cuda") for _ in range(2)]
        rows = lambda r: torch.as_strided(r, (pages, kv_heads, page_size, hd), (self.page_stride, page_size * hd, hd, 1))
        scales = lambda r: torch.as_strided(r, (pages, kv_heads, page_size), (self.scale_stride, page_size, 1))
        self.keys, self.values = map(rows, self.raw)
        self.key_scales, self.value_scales = map(scales, self.raw_scales)
        self.table = torch.full((seqs, table_stride), -1, dtype=torch.int32, device="cuda")
        self.c = _lib.PagedQ8Cache(self.raw[0].data_ptr(), self.raw[1].data_ptr(), self.raw_scales[0].data_ptr(),
                                   self.raw_scales[1].data_ptr(), self.table.data_ptr(), pages, page_size, kv_heads, hd, seqs,
                                   table_stride, self.page_stride, self.scale_stride)

    def where(self, seq, at):
        """Pages and slots of a sequence's positions `at` (page -1 where it has none)."""
        entry = at // self.page_size
        inside = (at >= 0) & (entry < self.table.shape[1])
        pages = torch.where(inside, self.table[seq].long()[entry.clamp(0, self.table.shape[1] - 1)], -1)
        return torch.where((pages >= 0) & (pages < self.pages), pages, -1), at % self.page_size

    def fill(self, seq, length, gen, spread=0.5):
        """Random rows, of sizes that differ, at a sequence's first positions (those it has pages for)."""
        page, slot = self.where(seq, torch.arange(length, device="cuda"))
        page, slot = page[page >= 0], slot[page >= 0]
        m = page.numel()
        for rows, scales in ((self.keys, self.key_scales), (self.values, self.value_scales)):
            rows[page, :, slot] = torch.randint(-127, 128, (m, self.kv_heads, self.hd), generator=gen, device="cuda", dtype=torch.int8)
            scales[page, :, slot] = torch.exp(spread * torch.randn((m, self.kv_heads), generator=gen, device="cuda")) / 60


def attention(pool, kind, q, q_start, lengths, scale, window, heads):
    """out [n, heads, hd] in f64 and the bound on each value's error.

    With p the softmax and A = sum p s |v|: rounding the result (u |out|); each
    weight p s in two or three bf16 parts, 2^-8 of what the parts before leave
    (A times 2^-16 or 2^-24); each score's f32 sum and scaling, at
    most (hd + 8) 2^-24 of scale sum |q| s |k|, which moves a probability by
    that much relatively, twice over through the normalization; and the f32
    sums over the keys with the exponential's, the products' and the joins'
    roundings, (keys + 64) 2^-24 A.
    """
    n, hd, group = q.shape[0], pool.hd, heads // pool.kv_heads
    u = TYPES[kind][2]
    parts = {"bf16": 2.0 ** -16, "f16": 2.0 ** -16, "f32": 2.0 ** -24}[kind]
    out = torch.zeros((n, heads, hd), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    for s in range(len(lengths)):
        for t in range(q_start[s], q_start[s + 1]):
            high = lengths[s] - (q_start[s + 1] - t)
            low = max(0, high - window + 1) if window else 0
            if high < low:
                continue
            page, slot = pool.where(s, torch.arange(low, high + 1, device="cuda"))
            page, slot = page[page >= 0], slot[page >= 0]
            if page.numel() == 0:
                continue
            k = (pool.keys[page, :, slot].double() * pool.key_scales[page, :, slot].double()[..., None]).repeat_interleave(group, 1)
            v = (pool.values[page, :, slot].double() * pool.value_scales[page, :, slot].double()[..., None]).repeat_interleave(group, 1)
            x = q[t].double()
            score = torch.einsum("hd,khd->hk", x, k) * scale
            mag = (torch.einsum("hd,khd->hk", x.abs(), k.abs()) * abs(scale)).amax(1)
            p = torch.softmax(score, 1)
            out[t] = torch.einsum("hk,khd->hd", p, v)
            a = torch.einsum("hk,khd->hd", p, v.abs())
            rel = parts + 2 * (hd + 8) * U32 * mag + (page.numel() + 64) * U32
            tol[t] = u * out[t].abs() + rel[:, None] * a * (1 + u) + TINY[kind]
    return out, tol


def rotated(x, w, table, rot, eps):
    """Heads [n, h, hd] in f64, normalized (w may be None) and turned, and the f32 arithmetic's error per value.

    The norm: a sum of hd squares over lanes and shuffles, each product and
    addition 2^-24 relatively, at most hd + 1 of them one behind another, of
    which the root keeps half; division, root, reciprocal and two products 5 more.
    The rotation: two products and their sum, 2 roundings of each term's size.
    """
    x = x.double()
    hd = x.shape[-1]
    err = torch.zeros_like(x)
    if w is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        err = x.abs() * ((hd + 1) / 2 + 5) * U32
    if rot:
        c, s = table[:, None, :rot // 2].double(), table[:, None, rot // 2:].double()
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        ea, eb = err[..., :rot // 2], err[..., rot // 2:rot]
        size = lambda f, g: (f * c).abs() + (g * s).abs()
        x = torch.cat([a * c - b * s, b * c + a * s, x[..., rot:]], -1)
        err = torch.cat([size(ea, eb) + 2 * U32 * size(a, b), size(eb, ea) + 2 * U32 * size(b, a), err[..., rot:]], -1)
    return x, err


def stepped_tol(x, err):
    """How far a row kept in 8 bits may read back from x: half a step of the row's scale, the value's own error,
    that of the scale (the largest value's) times up to 127 steps, and the roundings of scale, its reciprocal and
    the two products, 4 at 2^-24 of the row's largest."""
    top = x.abs().amax(-1, keepdim=True)
    top_err = err.amax(-1, keepdim=True)
    return (top + top_err) / 254 + err + top_err + 4 * U32 * top


def residual_norm(kind, x_kind, y, post, gate, scale, x, pre, eps):
    """x' and h in f64 with their bounds.

    A sum of squares adds up to cols / 128 terms a thread (at least 8 runs of
    8), five shuffles and up to 16 warps' sums twice over: at most D = cols / 32
    + 32 roundings one behind another, halved by the root; division, addition
    of eps, root and reciprocal 4 more. b has that, and a rounding for each of its three
    products and the scale; x' a rounding of itself on top. h takes x''s error,
    the change that it makes in the root mean square (rms of the error over rms of
    x'), the sum's own, and two products.
    """
    u, xu = TYPES[kind][2], TYPES[x_kind][2]
    y, x = y.double(), x.double()
    cols = y.shape[-1]
    depth = (cols / 32 + 32) / 2 + 4
    b, rel = y, 0.0
    if post is not None:
        b = post.double() * y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
        rel = (depth + 2) * U32
    if gate is not None:
        b, rel = b * gate.double(), rel + U32
    b, rel = b * scale, rel + 2 * U32
    out = x + b
    err = rel * b.abs() + U32 * out.abs()
    h = h_tol = None
    if pre is not None:
        rms = (out.square().mean(-1, keepdim=True) + eps).sqrt()
        h = pre.double() * out / rms
        moved = err.square().mean(-1, keepdim=True).sqrt() / rms
        h_err = (pre.double() / rms).abs() * err + h.abs() * (moved + (depth + 3) * U32)
        h_tol = h_err * (1 + u) + u * h.abs() + TINY[kind]
    return out, err * (1 + xu) + xu * out.abs() + TINY[x_kind], h, h_tol


def choose(logits, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, u=0.5):
    """(token, log-probability, tokens kept, margin) of one row, in 64 bits.

    `margin`: how far the nearest border is from a place that decides, over how
    far two right computations may lie apart there; the choice is determined
    where it is more than 1. In units of the largest weight: V weights in steps
    of 2^-44 are off by 2^-45 each, so that a sum, and the share of the whole
    that it is compared with, differ by V 2^-45 each, V 2^-44 together. A weight
    next to min_p is off by few f64 roundings, 2^-48 here.
    """
    x = np.asarray(logits, dtype=np.float64)
    x = np.where(np.isnan(x), -math.inf, x) + 0.0
    order = np.argsort(-x, kind="stable")
    order = order[:np.count_nonzero(x > -math.inf)]
    margin = math.inf
    off = len(x) * 2.0 ** -44
    if not len(order):
        return -1, -math.inf, 0, margin
    if not temperature > 0:
        return int(order[0]), 0.0, 1, margin
    top = x[order[0]]
    d = np.where(x[order] == top, 0.0, x[order] - top) if math.isfinite(top) else np.where(x[order] == top, 0.0, -math.inf)
    with np.errstate(invalid="ignore"):
        w = np.exp(np.where(d == 0, 0.0, d * (1.0 / float(temperature))))
    if top_k > 0:
        order, w = order[:top_k], w[:top_k]
    if top_p < 1:
        run = np.cumsum(w)
        at = float(top_p) * run[-1]
        m = min(len(w) - 1, int(np.searchsorted(run, at, side="left")))
        if top_p > 0:
            margin = min([abs(run[i] - at) / off for i in (m - 1, m) if 0 <= i < len(w)])
        order, w = order[:m + 1], w[:m + 1]
    if min_p > 0:
        margin = min(margin, float(np.min(np.abs(w - float(min_p)))) / 2.0 ** -48)
        m = max(1, np.count_nonzero(w >= float(min_p)))
        order, w = order[:m], w[:m]
    index = np.argsort(order)
    order, w = order[index], w[index]
    run = np.cumsum(w)
    at = min(max(float(u), 0.0), 1.0) * run[-1]
    last = int(np.nonzero(w > 2.0 ** -45)[0][-1])
    i = min(last, int(np.searchsorted(run, at, side="right")))
    if i < last:
        margin = min(margin, abs(run[i] - at) / off)
    if i > 0:
        margin = min(margin, abs(run[i] - w[i] - at) / off)
    return int(order[i]), math.log(w[i] / run[-1]), len(order), margin
