"""The batched step's operators from their definitions, in 64 bits, with the
error bound that each result's arithmetic allows (derived here, per value)."""
import torch

TYPES = {"f32": (torch.float32, 0, 2.0 ** -24), "f16": (torch.float16, 1, 2.0 ** -11),
         "bf16": (torch.bfloat16, 2, 2.0 ** -8)}  # torch type, DN_* code, unit roundoff
U32 = 2.0 ** -24


class Pool:
    """A paged cache on the GPU: pools of keys and values, a table, and its descriptor."""

    def __init__(self, kind, pages, page_size, kv_heads, hd, seqs, table_stride, fill=float("nan"), gap=0, offset=0):
        from dianoia_b200 import _lib
        self.dt, code, self.u = TYPES[kind]
        self.page_size, self.kv_heads, self.hd, self.pages = page_size, kv_heads, hd, pages
        block = kv_heads * page_size * hd
        self.page_stride = block + gap
        size = pages * self.page_stride + offset
        self.raw = [torch.full((size,), fill, device="cuda", dtype=self.dt) for _ in range(2)]
        self.keys, self.values = (r[offset:].view(pages, self.page_stride)[:, :block].view(pages, kv_heads, page_size, hd)
                                  if gap == 0 else torch.as_strided(r, (pages, kv_heads, page_size, hd),
                                                                    (self.page_stride, page_size * hd, hd, 1), offset)
                                  for r in self.raw)
        self.table = torch.full((seqs, table_stride), -1, dtype=torch.int32, device="cuda")
        self.c = _lib.PagedCache(self.keys.data_ptr(), self.values.data_ptr(), self.table.data_ptr(), code, pages, page_size,
                                 kv_heads, hd, seqs, table_stride, self.page_stride)

    def where(self, seq, length):
        """Pages and slots of a sequence's first `length` positions (page -1 where it has none)."""
        at = torch.arange(length, device="cuda")
        entry = at // self.page_size
        inside = entry < self.table.shape[1]
        pages = torch.where(inside, self.table[seq].long()[entry.clamp(max=self.table.shape[1] - 1)], -1)
        return torch.where((pages >= 0) & (pages < self.pages), pages, -1), at % self.page_size


def attention(pool, q, q_start, lengths, prefix_pages, prefix, scale, window, heads):
    """out [n, heads, hd] in f64 and the bound on each value's error.

    With p the softmax and A = sum p |v|: rounding the result (u |out|), the
    probabilities of 16-bit types (u A), each score's f32 sum and scaling,
    (hd + 8) 2^-24 scale sum |q||k| at most, which moves a probability by that
    much relatively, twice over through the normalization, and the f32 sums
    over the keys with the exponential's and the joins' roundings,
    (keys + 64) 2^-24 A.
    """
    n, hd, group = q.shape[0], pool.hd, heads // pool.kv_heads
    out = torch.zeros((n, heads, hd), dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    p_round = pool.u if pool.dt != torch.float32 else 0.0
    for s in range(len(lengths)):
        for t in range(q_start[s], q_start[s + 1]):
            high = lengths[s] - (q_start[s + 1] - t)
            low = max(0, high - window + 1) if window else 0
            if high < low:
                continue
            page, slot = pool.where(s, high + 1)
            pre = min(prefix, high + 1)
            if pre:
                at = torch.arange(pre, device="cuda")
                page[:pre] = prefix_pages.long()[at // pool.page_size]
                page = torch.where((page >= 0) & (page < pool.pages), page, -1)
            ok = page >= 0
            ok[:low] = False
            page, slot = page[ok], slot[ok]
            if page.numel() == 0:
                continue
            k = pool.keys[page, :, slot].double().repeat_interleave(group, 1)  # [keys, heads, hd]
            v = pool.values[page, :, slot].double().repeat_interleave(group, 1)
            x = q[t].double()
            score = torch.einsum("hd,khd->hk", x, k) * scale
            mag = (torch.einsum("hd,khd->hk", x.abs(), k.abs()) * abs(scale)).amax(1)
            p = torch.softmax(score, 1)
            out[t] = torch.einsum("hk,khd->hd", p, v)
            a = torch.einsum("hk,khd->hd", p, v.abs())
            rel = p_round + 2 * (hd + 8) * U32 * mag + (page.numel() + 64) * U32
            tol[t] = pool.u * out[t].abs() + rel[:, None] * a * (1 + pool.u) + 1e-30
    return out, tol


def rotated(x, w, eps, cos, sin, rot):
    """[n, heads, hd] in f64, normed by w (or not) and rotated, and the bound
    of its f32 arithmetic: four roundings of the two products, and for the
    norm (hd + 16) more of the mean, the root and the products."""
    y = x.double()
    k = 4
    if w is not None:
        y = y * w.double() / (y.square().mean(-1, keepdim=True) + eps).sqrt()
        k += x.shape[-1] + 16
    a, b = y[..., :rot // 2], y[..., rot // 2:rot]
    c, s = cos.double()[:, None], sin.double()[:, None]
    out = torch.cat([a * c - b * s, b * c + a * s, y[..., rot:]], -1)
    mag = torch.cat([(a * c).abs() + (b * s).abs(), (b * c).abs() + (a * s).abs(), y[..., rot:].abs()], -1)
    return out, k * U32 * mag


def logits(x, rules, vocab):
    """Row by row in f64, and the bound of the f32 arithmetic: six roundings of the terms."""
    n = x.shape[0]
    out = torch.empty((n, vocab), dtype=torch.float64, device="cuda")
    mag = torch.empty_like(out)
    ids = torch.arange(vocab, device="cuda")
    for r in range(n):
        y = x[r, :vocab].double()
        m = y.abs()
        if rules.get("history") is not None:
            a, b = rules["history"][r].item(), rules["history"][r + 1].item()
            toks = rules["tokens"][a:b].long()
            made = toks[len(toks) - (rules["generated"][r].item() if rules.get("generated") is not None else len(toks)):]
            toks, made = (z[(z >= 0) & (z < vocab)] for z in (toks, made))
            seen, count = torch.bincount(toks, minlength=vocab) > 0, torch.bincount(made, minlength=vocab).double()
            if rules.get("repetition") is not None:
                p = rules["repetition"][r].double()
                y = torch.where(seen, torch.where(y > 0, y / p, y * p), y)
                m = torch.where(seen, torch.maximum(m, y.abs()), m)
            for name, by in (("frequency", count), ("presence", (count > 0).double())):
                if rules.get(name) is not None:
                    d = rules[name][r].double() * by
                    y, m = torch.where(by > 0, y - d, y), m + d.abs()
        if rules.get("bias_start") is not None:
            a, b = rules["bias_start"][r].item(), rules["bias_start"][r + 1].item()
            for i in range(a, b):
                t = rules["bias_tokens"][i].item()
                if 0 <= t < vocab:
                    y[t] += rules["bias"][i].double()
                    m[t] += rules["bias"][i].double().abs()
        if rules.get("mask") is not None:
            row = r if rules.get("mask_row") is None else rules["mask_row"][r].item()
            if 0 <= row < rules["mask"].shape[0]:
                word = rules["mask"][row].long()[ids // 32]
                y = torch.where((word >> (ids % 32)) & 1 != 0, y, -torch.inf)
        out[r], mag[r] = y, m
    return out, 6 * U32 * mag


def check(got, want, tol, u, what=""):
    """Every value within its bound plus the rounding to its type (u of the value, and below f16's normal
    numbers half their spacing, 2^-25); infinities and NaN in the same places."""
    tol = tol + (2.0 ** -25 if got.dtype == torch.float16 else 0.0)
    got = got.double()
    fin = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what + ": NaN elsewhere"
    assert torch.equal(got[~fin & ~torch.isnan(want)], want[~fin & ~torch.isnan(want)]), what + ": infinities differ"
    bad = (got - want).abs()[fin] > (tol + u * want.abs())[fin]
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} out of bounds, worst " \
                          f"{((got - want).abs() / (tol + u * want.abs() + 1e-300))[fin].max().item():.3g} times the bound"
