"""dn_paged_q8_append, dn_paged_q8_read and dn_paged_q8_attention against their
definitions in 64 bits (tests/paged_q8_reference.py derives each value's bound):
types, head layouts, page sizes, strides, ragged and empty sequences, windows,
rows that nobody sees, offsets past 32 bits, graphs, and refusals."""
import random

import pytest

from tests import paged_q8_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from dianoia_b200 import _lib  # noqa: E402

TYPES = ref.TYPES


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------- append and read


class Tokens:
    """Tokens of a few sequences in a pool, in no order, some of them skipped for each reason there is."""

    def __init__(self, n, heads, kv_heads, hd, page, seed=0, gap=0, scale_gap=0, skip=True):
        rng = random.Random(seed)
        self.n, self.heads, seqs = n, heads, 3
        width = -(-n // page) + 1
        self.pool = ref.Q8Pool(seqs * width, page, kv_heads, hd, seqs, width, gap, scale_gap)
        order = list(range(seqs * width))
        rng.shuffle(order)
        self.pool.table.copy_(ints(order).view(seqs, width))
        self.pool.table[2, 0] = -1
        at = [0] * seqs
        self.seq, self.pos = [], []
        for _ in range(n):
            s = rng.randrange(seqs)
            self.seq.append(s)
            self.pos.append(at[s])
            at[s] += 1
        self.rope_rows = max(self.pos) + 1
        if skip and n > 6:
            self.seq[1], self.seq[2], self.pos[3], self.pos[4] = -1, seqs, -1, width * page
            self.pos[5] = 1 << 30
        live = [0 <= s < seqs and 0 <= p < width * page and not (s == 2 and p < page) for s, p in zip(self.seq, self.pos)]
        self.live = torch.tensor(live, device="cuda")
        self.freeze()

    def freeze(self):
        """The lists as the tensors that calls read, which live as long as this."""
        self.seq_t, self.pos_t = ints(self.seq), ints(self.pos)


def append(L, t, kind, out_kind, qkv, rope, rot, q_norm, k_norm, eps=1e-6, q_out=None, flags=0):
    hd, kvh = t.pool.hd, t.pool.kv_heads
    q_out = torch.full((t.n, t.heads, hd), 7.0, device="cuda", dtype=TYPES[out_kind][0]) if q_out is None else q_out
    q = qkv.data_ptr()
    k = q + t.heads * hd * qkv.element_size()
    v = k + kvh * hd * qkv.element_size()
    ptr = lambda x: None if x is None else x.data_ptr()
    rc = L.dn_paged_q8_append(t.pool.c, TYPES[kind][1], q, qkv.stride(0), k, qkv.stride(0), v, qkv.stride(0),
                              t.seq_t.data_ptr(), t.pos_t.data_ptr(), ptr(rope), rope.shape[0] if rope is not None else 0,
                              rot, ptr(q_norm), ptr(k_norm), eps, TYPES[out_kind][1], q_out.data_ptr(), q_out.stride(0), t.heads,
                              t.n, flags, stream())
    assert rc == 0
    return q_out


def read(L, t, kind, k_out=None, v_out=None):
    rows = (t.n, t.pool.kv_heads * t.pool.hd)
    k_out, v_out = (torch.full(rows, 7.0, device="cuda", dtype=TYPES[kind][0]) if o is None else o for o in (k_out, v_out))
    assert L.dn_paged_q8_read(t.pool.c, TYPES[kind][1], t.seq_t.data_ptr(), t.pos_t.data_ptr(), k_out.data_ptr(),
                              k_out.stride(0), v_out.data_ptr(), v_out.stride(0), t.n, 0, stream()) == 0
    return k_out, v_out


def stored(pool):
    return [x.clone() for x in (*pool.raw, *pool.raw_scales)]


@pytest.mark.parametrize("kind,out_kind", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f32"),
                                           ("bf16", "f16")])
@pytest.mark.parametrize("heads,kv_heads,hd,page,rot,norm,n", [
    (16, 8, 128, 16, 128, True, 37), (12, 4, 96, 32, 48, False, 33), (8, 8, 64, 7, 64, True, 40), (3, 1, 16, 1, 16, True, 9),
    (8, 2, 256, 24, 256, True, 21), (4, 2, 80, 16, 36, True, 25), (0, 2, 32, 16, 0, False, 11), (5, 5, 48, 16, 6, False, 1),
    (2, 1, 240, 3, 240, True, 300)])
def test_append(cuda_lib, kind, out_kind, heads, kv_heads, hd, page, rot, norm, n):
    t, g = Tokens(n, heads, kv_heads, hd, page, seed=n, gap=32, scale_gap=3), gen(n)
    qkv = (torch.randn((n, (heads + 2 * kv_heads) * hd + 8), generator=g, device="cuda") * 2).to(TYPES[kind][0])
    angle = torch.rand((t.rope_rows, max(rot // 2, 1)), generator=g, device="cuda") * 7
    rope = torch.cat([angle.cos(), angle.sin()], 1) if rot else None
    w = [1 + 0.2 * torch.randn(hd, generator=g, device="cuda") if norm else None for _ in range(2)]
    before = stored(t.pool)
    q_out = append(cuda_lib, t, kind, out_kind, qkv, rope, rot, *w)
    torch.cuda.synchronize()
    live = t.live.clone()
    if rot:
        live &= ints(t.pos) < t.rope_rows
    at = ints(t.pos).long().clamp(0, t.rope_rows - 1)
    x = qkv[:, :(heads + 2 * kv_heads) * hd].reshape(n, heads + 2 * kv_heads, hd)
    table = rope[at] if rot else None
    u = TYPES[out_kind][2]
    if heads:
        want, err = ref.rotated(x[:, :heads], w[0], table, rot, 1e-6)
        assert (q_out[~live] == 0).all()
        off = (q_out.double() - want).abs()
        assert (off <= err * (1 + u) + u * want.abs() + ref.TINY[out_kind])[live].all()
    for part, wk, turn, rows, scales in ((x[:, heads:heads + kv_heads], w[1], rot, t.pool.keys, t.pool.key_scales),
                                         (x[:, heads + kv_heads:], None, 0, t.pool.values, t.pool.value_scales)):
        want, err = ref.rotated(part, wk, table, turn, 1e-6)
        tol = ref.stepped_tol(want, err)
        for i in live.nonzero()[:, 0].tolist():
            page_i = t.pool.table[t.seq[i], t.pos[i] // page].item()
            slot = t.pos[i] % page
            got = rows[page_i, :, slot].double() * scales[page_i, :, slot].double()[:, None]
            assert ((got - want[i]).abs() <= tol[i]).all(), i
            assert (rows[page_i, :, slot].abs().amax(-1) == 127).all()
    # Nothing else has changed, gaps included.
    for i in live.nonzero()[:, 0].tolist():
        page_i, slot = t.pool.table[t.seq[i], t.pos[i] // page].item(), t.pos[i] % page
        for old, raw, size, stride in ((before[0], t.pool.raw[0], hd, t.pool.page_stride), (before[1], t.pool.raw[1], hd, t.pool.page_stride),
                                       (before[2], t.pool.raw_scales[0], 1, t.pool.scale_stride),
                                       (before[3], t.pool.raw_scales[1], 1, t.pool.scale_stride)):
            for h in range(kv_heads):
                a = page_i * stride + (h * page + slot) * size
                old[a:a + size] = raw[a:a + size]
    for old, new in zip(before, stored(t.pool)):
        assert torch.equal(old.view(torch.uint8), new.view(torch.uint8))


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("hd,page,offset", [(128, 16, 0), (64, 5, 0), (96, 16, 1), (256, 32, 0), (16, 1, 3)])
def test_moved_rows_are_exact(cuda_lib, kind, hd, page, offset):
    """Without norm and rotation a row is quantized from its own values: bit for bit what lab_quantize_q8's steps give
    it, and read back bit for bit as int8 times scale, at any alignment of the rows."""
    n, kvh = 61, 3
    t, g = Tokens(n, 0, kvh, hd, page, seed=hd, skip=True), gen(hd)
    dt = TYPES[kind][0]
    raw = torch.zeros(n * (2 * kvh * hd + 5) + offset, device="cuda", dtype=dt)
    qkv = raw[offset:].view(n, 2 * kvh * hd + 5)
    qkv[:, :2 * kvh * hd] = torch.randn((n, 2 * kvh * hd), generator=g, device="cuda") * torch.exp(
        3 * torch.randn((n, 1), generator=g, device="cuda")).clamp(max=100)
    qkv[7] = 0
    append(cuda_lib, t, kind, "f32", qkv, None, 0, None, None)
    # On the CPU, where a division by a number is one.
    x = qkv[:, :2 * kvh * hd].float().reshape(n, 2, kvh, hd).cpu()
    scale = x.abs().amax(-1) / torch.full((n, 2, kvh), 127.0)
    q = x * torch.where(scale > 0, 1 / scale, 0.0)[..., None]
    q, scale = torch.where(q < 0, q - 0.5, q + 0.5).trunc().clamp(-127, 127).cuda(), scale.cuda()
    for i in t.live.nonzero()[:, 0].tolist():
        p, slot = t.pool.table[t.seq[i], t.pos[i] // page].item(), t.pos[i] % page
        for j, (rows, scales) in enumerate(((t.pool.keys, t.pool.key_scales), (t.pool.values, t.pool.value_scales))):
            assert torch.equal(rows[p, :, slot].float(), q[i, j]) and torch.equal(scales[p, :, slot], scale[i, j])
    for out_kind in TYPES:
        odt = TYPES[out_kind][0]
        buf = [torch.full((n * (kvh * hd + 3) + offset,), 7.0, device="cuda", dtype=odt) for _ in range(2)]
        outs = [b[offset:].view(n, kvh * hd + 3) for b in buf]
        read(cuda_lib, t, out_kind, *outs)
        for j, o in enumerate(outs):
            want = (q[:, j] * scale[:, j][..., None]).to(odt).view(n, -1)
            want[~t.live] = 0
            assert torch.equal(o[:, :kvh * hd], want)
            assert (o[:, kvh * hd:] == 7).all() and (buf[j][:offset] == 7).all()


def test_read_one_side(cuda_lib):
    t = Tokens(50, 0, 2, 64, 16, skip=True)
    for s in range(3):
        t.pool.fill(s, 50, gen(s))
    k, v = read(cuda_lib, t, "f32")
    for side in (0, 1):
        out = torch.full_like(k, 5.0)
        args = [None, 0, None, 0]
        args[2 * side], args[2 * side + 1] = out.data_ptr(), out.stride(0)
        assert cuda_lib.dn_paged_q8_read(t.pool.c, 0, t.seq_t.data_ptr(), t.pos_t.data_ptr(), *args, t.n, 0, stream()) == 0
        assert torch.equal(out.view(torch.int32), (k, v)[side].view(torch.int32))


def test_rows_that_are_not_finite_or_tiny(cuda_lib):
    n, kvh, hd = 8, 2, 64
    t = Tokens(n, 0, kvh, hd, 16, skip=False)
    t.pool.table[2, 0] = t.pool.pages - 1 if t.pool.pages - 1 not in t.pool.table.tolist()[2] else t.pool.table[2, 1]
    t.seq, t.pos = [0] * n, list(range(n))
    t.freeze()
    x = torch.ones((n, 2 * kvh * hd), device="cuda")
    x[0, 3], x[1, 5], x[2, 70], x[3, :64] = float("nan"), float("inf"), float("-inf"), 1e-37
    x[4, :64], x[5, 130], x[6, 2], x[7, :64] = 2.0 ** -119.2, float("nan"), 3.4e38, 2.0 ** -118.9
    append(cuda_lib, t, "f32", "f32", x, None, 0, None, None)
    k, v = (o.view(n, kvh, hd) for o in read(cuda_lib, t, "f32"))
    for out, row, head in ((k, 0, 0), (k, 1, 0), (k, 2, 1), (v, 5, 0)):
        assert out[row, head].isnan().all()
    assert k[0, 1].eq(1).all() and k[5].eq(1).all() and v[5, 1].eq(1).all()
    # 127 is 2^6.989: scales of 2^-126.19 and less are under the least normal number, one of 2^-125.89 is not.
    assert k[3, 0].eq(0).all() and k[4, 0].eq(0).all()
    step = 2.0 ** -118.9 / 127
    assert ((k[7, 0].double() - x[7, 0].double()).abs() <= step).all() and (k[7, 0] > 0).all()
    assert k[6, 0, 2] > 3.3e38 and k[6, 0, :2].eq(0).all()


def test_append_in_place_and_far_offsets(cuda_lib):
    """Queries rotated where they lie; pages past 2^31 bytes; a stream of its own."""
    kvh, hd, page, n, heads = 8, 256, 64, 6, 2
    g = gen(1)
    pages = 20000  # 2.6 GB a pool
    pool = ref.Q8Pool.__new__(ref.Q8Pool)
    pool.page_size, pool.kv_heads, pool.hd, pool.pages = page, kvh, hd, pages
    keys, values = (torch.zeros((pages, kvh, page, hd), dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros((pages, kvh, page), device="cuda") for _ in range(2))
    table = torch.tensor([[pages - 1, 17]], dtype=torch.int32, device="cuda")
    cache = _lib.PagedQ8Cache(keys.data_ptr(), values.data_ptr(), ks.data_ptr(), vs.data_ptr(), table.data_ptr(), pages, page, kvh,
                              hd, 1, 2, kvh * page * hd, kvh * page)
    qkv = torch.randn((n, (heads + 2 * kvh) * hd), generator=g, device="cuda")
    keep = qkv.clone()
    seq, pos = ints([0] * n), ints([0, 63, 64, 65, 30, 127])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    k = qkv.data_ptr() + heads * hd * 4
    row = qkv.shape[1]
    angle = torch.rand((128, hd // 2), generator=g, device="cuda")
    rope = torch.cat([angle.cos(), angle.sin()], 1)
    s.wait_stream(torch.cuda.current_stream())
    assert cuda_lib.dn_paged_q8_append(cache, 0, qkv.data_ptr(), row, k, row, k + kvh * hd * 4, row, seq.data_ptr(), pos.data_ptr(),
                                       rope.data_ptr(), 128, hd, None, None, 1e-6, 0, qkv.data_ptr(), row, heads, n, 0,
                                       s.cuda_stream) == 0
    out = [torch.empty((n, kvh * hd), device="cuda") for _ in range(2)]
    s.wait_stream(torch.cuda.current_stream())
    assert cuda_lib.dn_paged_q8_read(cache, 0, seq.data_ptr(), pos.data_ptr(), out[0].data_ptr(), kvh * hd, out[1].data_ptr(),
                                     kvh * hd, n, 0, s.cuda_stream) == 0
    s.synchronize()
    x = keep.view(n, heads + 2 * kvh, hd)
    want, err = ref.rotated(x[:, :heads], None, rope[pos.long()], hd, 0)
    assert ((qkv.view(n, -1, hd)[:, :heads].double() - want).abs() <= err + 1e-30 + ref.U32 * want.abs()).all()
    assert torch.equal(qkv.view(n, -1, hd)[:, heads:], x[:, heads:])
    for o, part, turn in ((out[0], x[:, heads:heads + kvh], hd), (out[1], x[:, heads + kvh:], 0)):
        want, err = ref.rotated(part, None, rope[pos.long()], turn, 0)
        assert ((o.view(n, kvh, hd).double() - want).abs() <= ref.stepped_tol(want, err) + ref.U32 * want.abs()).all()
    assert (ks != 0).sum() == n * kvh


# ------------------------------------------------------------------- attention


class Batch:
    def __init__(self, kind, heads, kv_heads, hd, page, lengths, q_lens, seed=0, gap=0, scale_gap=0, holes=0, spread=0.5, wide=0):
        rng, g = random.Random(seed), gen(seed)
        self.kind, self.heads, self.lengths = kind, heads, lengths
        width = max(1, -(-max(lengths) // page)) + wide
        need = [-(-n // page) for n in lengths]
        pages = sum(need) + 2
        order = list(range(pages))
        rng.shuffle(order)
        self.pool = ref.Q8Pool(pages, page, kv_heads, hd, len(lengths), width, gap, scale_gap)
        at, table = 0, []
        for k in need:
            table.append(order[at:at + k] + [-1] * (width - k))
            at += k
        self.pool.table.copy_(ints(table))
        for s, n in enumerate(lengths):
            if n > 0:
                self.pool.fill(s, n, g, spread)
        for _ in range(holes):  # freed pages
            self.pool.table[rng.randrange(len(lengths)), rng.randrange(width)] = rng.choice([-1, pages, 1 << 30])
        self.starts = [0]
        for q in q_lens:
            self.starts.append(self.starts[-1] + q)
        self.n = self.starts[-1]
        self.q = (torch.randn((self.n, heads, hd), generator=g, device="cuda") * 2).to(TYPES[kind][0])

    def run(self, L, window=0, scale=None, q_start=True, q=None, out=None, max_length=None, flags=0, ws=None):
        scale = self.pool.hd ** -0.5 if scale is None else scale
        q = self.q if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        most = max(self.lengths) if max_length is None else max_length
        starts, lens = ints(self.starts), ints(self.lengths)
        need = L.dn_paged_q8_attention_workspace(self.pool.c, self.heads, self.n, most)
        assert need > 0
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda") if ws is None else ws  # NaN
        assert L.dn_paged_q8_attention(self.pool.c, TYPES[self.kind][1], q.data_ptr(), q.stride(0),
                                       starts.data_ptr() if q_start else None, lens.data_ptr(), most, scale, window, out.data_ptr(),
                                       out.stride(0), self.heads, self.n, ws.data_ptr(), need, flags, stream()) == 0
        torch.cuda.synchronize()
        return out

    def check(self, L, window=0, scale=None, **kw):
        out = self.run(L, window, scale, **kw)
        want, tol = ref.attention(self.pool, self.kind, self.q, self.starts, self.lengths,
                                  self.pool.hd ** -0.5 if scale is None else scale, window, self.heads)
        off = (out[:self.n].double() - want).abs()
        assert (off <= tol).all(), float((off / tol.clamp(min=1e-38)).max())
        assert (out[:self.n].double()[tol == 0] == 0).all()
        return out


LAYOUTS = [(16, 8, 128), (12, 4, 96), (28, 4, 128), (8, 8, 64), (8, 2, 256), (9, 3, 64), (16, 1, 128), (3, 3, 16), (40, 1, 80),
           (4, 2, 240), (64, 1, 32)]


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("heads,kv_heads,hd", LAYOUTS)
def test_single_tokens(cuda_lib, kind, heads, kv_heads, hd):
    """One token a sequence: lengths of 0, 1 and around tiles, ragged."""
    lengths = [1, 0, 2, 15, 16, 17, 31, 33, 64, 100, 257, 515]
    b = Batch(kind, heads, kv_heads, hd, 16, lengths, [1] * len(lengths), seed=hd)
    first = b.check(cuda_lib, q_start=False)
    assert torch.equal(b.run(cuda_lib), first)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("page", [1, 3, 8, 16, 24, 64, 100])
def test_pages(cuda_lib, kind, page):
    b = Batch(kind, 8, 2, 64, page, [page, 7 * page + 1, 300, 99], [1, 2, 1, 3], seed=page, gap=48, scale_gap=5)
    b.check(cuda_lib)


@pytest.mark.parametrize("kind,heads,kv_heads,hd", [("bf16", 16, 8, 128), ("f16", 12, 4, 96), ("f32", 9, 3, 64), ("bf16", 8, 2, 256),
                                                    ("f32", 16, 1, 256), ("f16", 40, 1, 128)])
def test_drafts_and_prompts(cuda_lib, kind, heads, kv_heads, hd):
    """Ragged queries, sequences with none, a whole prompt."""
    b = Batch(kind, heads, kv_heads, hd, 16, [40, 5, 130, 77, 333, 0], [2, 5, 130, 0, 9, 0], seed=3)
    b.check(cuda_lib)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("window", [1, 2, 16, 50, 1000])
def test_windows_and_holes(cuda_lib, kind, window):
    b = Batch(kind, 8, 4, 64, 16, [200, 16, 1, 130, 470], [1, 3, 1, 17, 2], seed=window, holes=14)
    b.check(cuda_lib, window=window)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_long(cuda_lib, kind):
    """Lengths that are split, with every hint of the longest."""
    b = Batch(kind, 8, 2, 128, 64, [9000, 1, 5000], [1, 1, 2], seed=5)
    for hint in (None, 0, 1, 100000, 1 << 30):
        b.check(cuda_lib, max_length=hint)
    b.check(cuda_lib, window=3001)


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
def test_sizes(cuda_lib, kind):
    """Rows and scores of every size: large scores, one key that takes all, scales far apart, zeros."""
    b = Batch(kind, 8, 4, 128, 16, [300, 40], [1, 2], seed=9, spread=4.0)
    b.check(cuda_lib)
    b.check(cuda_lib, scale=3.0)
    b.check(cuda_lib, scale=-1.0)
    out = b.check(cuda_lib, scale=0.0)
    assert out.isfinite().all()
    b.pool.value_scales[:] = torch.where(b.pool.value_scales.isnan(), b.pool.value_scales, b.pool.value_scales * 1e30)
    if kind != "f16":  # beyond its range
        b.check(cuda_lib)
    b.pool.value_scales[:] = torch.where(b.pool.value_scales.isnan(), b.pool.value_scales, b.pool.value_scales * 1e-60)
    b.check(cuda_lib)
    b.pool.key_scales[:] = torch.where(b.pool.key_scales.isnan(), b.pool.key_scales, 0.0)
    b.check(cuda_lib)


def test_unseen_rows_do_not_count(cuda_lib):
    """Rows past a length, before a window or behind no page hold NaN scales: nothing of them comes out. A seen row's NaN does."""
    for kind in TYPES:
        b = Batch(kind, 8, 4, 64, 16, [37, 90, 200], [1, 4, 2], seed=2, wide=3)
        want = b.check(cuda_lib, window=30)
        spare = b.pool.where(2, torch.arange(0, 160, device="cuda"))  # before the window of every token of sequence 2
        for scales in (b.pool.key_scales, b.pool.value_scales):
            scales[spare[0], :, spare[1]] = float("inf")
        assert torch.equal(b.run(cuda_lib, window=30), want)
        page, slot = b.pool.where(1, torch.tensor([88], device="cuda"))
        old = b.pool.value_scales[page, 1, slot].clone()
        b.pool.value_scales[page, 1, slot] = float("nan")  # the third of sequence 1's four tokens is at 88
        out = b.run(cuda_lib, window=30)
        bad = torch.zeros_like(out, dtype=torch.bool)
        bad[3:5, 2:4] = True
        assert out[bad].isnan().all() and torch.equal(out[~bad], want[~bad])
        b.pool.value_scales[page, 1, slot] = old
        b.pool.key_scales[page, 1, slot] = float("nan")
        out = b.run(cuda_lib, window=30)
        assert out[bad].isnan().all() and torch.equal(out[~bad], want[~bad])


def test_tokens_behind_the_last_sequence_stay(cuda_lib):
    b = Batch("bf16", 8, 4, 64, 16, [20, 300], [1, 2], seed=4)
    q = torch.cat([b.q, b.q])
    out = torch.full_like(q, 7.0)
    n, b.n = b.n, q.shape[0]
    b.run(cuda_lib, q=q, out=out)
    b.n = n
    assert (out[n:] == 7).all()
    assert torch.equal(out[:n], b.check(cuda_lib))


def test_strides_in_place_and_alignment(cuda_lib):
    for kind in TYPES:
        b = Batch(kind, 8, 4, 64, 16, [20, 300, 41], [1, 2, 5], seed=6)
        want = b.check(cuda_lib)
        wide = torch.full((b.n, 3 * 512 + 1), 7.0, device="cuda", dtype=b.q.dtype)
        q = wide[:, 513:513 + 512]
        q.copy_(b.q.view(b.n, 512))
        out = torch.full((b.n, 517), 7.0, device="cuda", dtype=b.q.dtype)[:, 1:513]
        b.run(cuda_lib, q=q, out=out)
        assert torch.equal(out.reshape_as(want), want)
        b.run(cuda_lib, q=q, out=q)
        assert torch.equal(q.reshape_as(want), want) and (wide[:, :513] == 7).all() and (wide[:, 1025:] == 7).all()


def test_graphs_streams_and_two_at_once(cuda_lib):
    """Captured calls replayed beside eager ones on another stream, each with a workspace of its own; equal every time."""
    b = Batch("bf16", 16, 8, 128, 16, [700, 2100, 3, 0, 5000], [1, 1, 2, 1, 1], seed=8)
    c = Batch("f32", 9, 3, 64, 24, [900, 1200], [1, 4], seed=9)
    want_b, want_c = b.check(cuda_lib), c.check(cuda_lib)
    args = []
    for x in (b, c):
        need = cuda_lib.dn_paged_q8_attention_workspace(x.pool.c, x.heads, x.n, max(x.lengths))
        ws, out = torch.empty(need, dtype=torch.uint8, device="cuda"), torch.zeros_like(x.q)
        keep = (ints(x.starts), ints(x.lengths), ws, out)
        args.append((keep, lambda s, x=x, k=keep: cuda_lib.dn_paged_q8_attention(
            x.pool.c, TYPES[x.kind][1], x.q.data_ptr(), x.q.stride(0), k[0].data_ptr(), k[1].data_ptr(), max(x.lengths),
            x.pool.hd ** -0.5, 0, k[3].data_ptr(), k[3].stride(0), x.heads, x.n, k[2].data_ptr(), k[2].numel(), _lib.DN_FLAG_PDL, s)))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(2):
            assert args[0][1](stream()) == 0
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for _ in range(20):
        graph.replay()
        assert args[1][1](other.cuda_stream) == 0
    torch.cuda.synchronize()
    assert torch.equal(args[0][0][3], want_b) and torch.equal(args[1][0][3], want_c)


def test_shared_pages_and_far_offsets(cuda_lib):
    """Sequences that name the same pages; pages past 2^31 bytes."""
    kvh, hd, page, heads = 8, 256, 64, 16
    g, pages = gen(1), 18000
    pool = ref.Q8Pool.__new__(ref.Q8Pool)
    pool.page_size, pool.kv_heads, pool.hd, pool.pages = page, kvh, hd, pages
    pool.keys, pool.values = (torch.zeros((pages, kvh, page, hd), dtype=torch.int8, device="cuda") for _ in range(2))
    pool.key_scales, pool.value_scales = (torch.full((pages, kvh, page), float("nan"), device="cuda") for _ in range(2))
    pool.table = ints([[pages - 1, 17, pages - 2], [pages - 1, 17, 5]])
    pool.c = _lib.PagedQ8Cache(pool.keys.data_ptr(), pool.values.data_ptr(), pool.key_scales.data_ptr(), pool.value_scales.data_ptr(),
                               pool.table.data_ptr(), pages, page, kvh, hd, 2, 3, kvh * page * hd, kvh * page)
    b = Batch.__new__(Batch)
    b.kind, b.heads, b.lengths, b.pool, b.starts, b.n = "bf16", heads, [150, 190], pool, [0, 1, 3], 3
    pool.fill(0, 150, g)
    pool.fill(1, 190, g)
    b.q = torch.randn((3, heads, hd), generator=g, device="cuda").bfloat16()
    b.check(cuda_lib)


def test_table_that_ends_before_the_length(cuda_lib):
    """Positions past the table do not exist."""
    b = Batch("bf16", 4, 2, 64, 16, [112, 64], [1, 2], seed=1)  # whole pages
    b.lengths = [150, 64]
    b.check(cuda_lib)
