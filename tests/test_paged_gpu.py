"""dn_paged_append and dn_paged_attention against their definitions in 64
bits (tests/paged_reference.py derives each value's bound): types, head
layouts, page sizes, strides, ragged and empty sequences, windows, what lies in
slots that nobody sees, offsets past 32 bits, and refusals."""
import ctypes
import random

import pytest

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


class Batch:
    """Sequences behind a shared prefix in a pool whose other slots hold NaN."""

    def __init__(self, kind, heads, kv_heads, hd, page, prefix, own, q_lens, seed=0, gap=0, offset=0, holes=0):
        rng, g = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
        self.heads, self.prefix, self.q_lens = heads, prefix, q_lens
        self.lengths = [prefix + k if k is not None else 0 for k in own]
        seqs = len(own)
        first = prefix // page  # entries before this one are only read through prefix_pages
        width = max(1, -(-max(self.lengths + [prefix]) // page))
        need = [max(0, -(-n // page) - first) for n in self.lengths]
        shared = -(-prefix // page)
        pages = shared + sum(need) + 2
        order = list(range(pages))
        rng.shuffle(order)
        self.pool = ref.Pool(kind, pages, page, kv_heads, hd, seqs, width, gap=gap, offset=offset)
        self.prefix_pages = ints(order[:max(1, shared)])
        at = shared
        table = []
        for k in need:
            row = [-1] * first + order[at:at + k]
            table.append((row + [-1] * width)[:width])
            at += k
        self.pool.table.copy_(ints(table))
        u = lambda *s: torch.randn(s, generator=g, device="cuda").to(self.pool.dt)
        for p in range(prefix):
            pg, slot = order[p // page], p % page
            self.pool.keys[pg, :, slot], self.pool.values[pg, :, slot] = u(kv_heads, hd), u(kv_heads, hd)
        for s, n in enumerate(self.lengths):
            m = max(0, n - prefix)
            if m:
                pg, slot = self.pool.where(s, n)
                self.pool.keys[pg[prefix:], :, slot[prefix:]] = u(m, kv_heads, hd)
                self.pool.values[pg[prefix:], :, slot[prefix:]] = u(m, kv_heads, hd)
        for _ in range(holes):  # freed pages
            self.pool.table[rng.randrange(seqs), rng.randrange(first, width)] = rng.choice([-1, pages, 1 << 30])
        self.starts = [0]
        for q in q_lens:
            self.starts.append(self.starts[-1] + q)
        self.n = self.starts[-1]
        self.q = u(self.n, heads, hd) * 2

    def run(self, L, window=0, scale=None, q_start=True, q=None, out=None, max_length=None, flags=0):
        hd = self.pool.hd
        scale = hd ** -0.5 if scale is None else scale
        q = self.q if q is None else q
        out = torch.full_like(q, 7.0) if out is None else out
        most = max(self.lengths) if max_length is None else max_length
        starts, lens = ints(self.starts), ints(self.lengths)
        need = L.dn_paged_attention_workspace(self.pool.c, self.heads, self.n, self.prefix, most)
        assert need > 0
        ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")  # NaN
        rc = L.dn_paged_attention(self.pool.c, q.data_ptr(), q.stride(0), starts.data_ptr() if q_start else None,
                                  lens.data_ptr(), self.prefix_pages.data_ptr(), self.prefix, most, scale, window,
                                  out.data_ptr(), out.stride(0), self.heads, self.n, ws.data_ptr(), need, flags, stream())
        assert rc == 0
        torch.cuda.synchronize()
        return out

    def check(self, L, window=0, scale=None, **kw):
        out = self.run(L, window, scale, **kw)
        want, tol = ref.attention(self.pool, self.q, self.starts, self.lengths, self.prefix_pages, self.prefix,
                                  self.pool.hd ** -0.5 if scale is None else scale, window, self.heads)
        ref.check(out.view(self.n, self.heads, self.pool.hd), want, tol, 0.0, "attention")
        return out


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,hd,page", [(16, 8, 128, 16), (8, 2, 64, 7), (9, 3, 96, 32), (4, 4, 256, 16),
                                                    (20, 1, 128, 64), (3, 3, 72, 16), (6, 2, 80, 1), (2, 1, 33, 5), (4, 2, 20, 16)])
def test_decode_batch(cuda_lib, kind, heads, kv_heads, hd, page):
    """One query a sequence: own parts of 1 to 300 keys, an empty slot, and no own key but its own."""
    own = [1, 17, 300, None, 64, 65, 2]
    Batch(kind, heads, kv_heads, hd, page, 2 * 32 * 7, own, [1] * 7, seed=hd).check(cuda_lib)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 333, 1500])
def test_prefix_lengths(cuda_lib, kind, prefix):
    """No prefix, and prefixes that end inside a page and a tile."""
    Batch(kind, 8, 2, 64, 16, prefix, [5, 40, 1, None, 130], [1] * 5, seed=prefix).check(cuda_lib, q_start=False)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("window", [0, 1, 50, 400])
def test_ragged_queries(cuda_lib, kind, window):
    """Several queries a sequence (causal), sequences with none, a chunk longer than a tile, windows."""
    q_lens = [3, 0, 1, 90, 0, 2, 7]
    own = [3, 9, 200, 90, None, 33, 150]
    Batch(kind, 6, 2, 64, 16, 64, own, q_lens, seed=window).check(cuda_lib, window=window)


@pytest.mark.parametrize("group", [1, 3, 7, 16, 17, 40])
def test_groups(cuda_lib, group):
    Batch("bf16", group * 2, 2, 64, 16, 96, [30, 1, 77], [2, 1, 5], seed=group).check(cuda_lib)


@pytest.mark.parametrize("seqs,group", [(70, 2), (130, 4), (200, 8)])
def test_many_rows_share_the_prefix(cuda_lib, seqs, group):
    rng = random.Random(seqs)
    own = [rng.choice([1, 5, 60, None]) for _ in range(seqs)]
    Batch("bf16", group * 2, 2, 128, 32, 700, own, [1] * seqs, seed=seqs).check(cuda_lib)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd,kv_heads", [(64, 2), (128, 1), (256, 1)])
def test_many_rows_with_a_window(cuda_lib, kind, hd, kv_heads):
    """Rows of one tile that see different parts of the prefix: windows, and lengths inside it."""
    rng = random.Random(hd)
    own = [rng.choice([1, 9, 80]) for _ in range(90)]
    b = Batch(kind, 3 * kv_heads, kv_heads, hd, 16, 400, own, [1] * 90, seed=hd)
    b.lengths[5], b.lengths[40], b.lengths[41] = 100, 1, 399  # shorter than the prefix
    b.check(cuda_lib, window=0)
    b.check(cuda_lib, window=130)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_long_own_sequences_are_split(cuda_lib, kind):
    """Few long sequences, and the same with a max_length that says nothing useful."""
    b = Batch(kind, 4, 1, 128, 16, 16, [5000, 1, 2777], [1, 1, 1])
    b.check(cuda_lib)
    b.check(cuda_lib, max_length=0)
    b.check(cuda_lib, max_length=1 << 20)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_pages_that_are_not_there(cuda_lib, kind):
    """Table entries outside the pool hide their positions; a table shorter than the length ends it."""
    b = Batch(kind, 4, 2, 64, 16, 32, [100, 200, 64, 90], [1, 2, 1, 1], holes=6, seed=3)
    b.check(cuda_lib)
    b.prefix_pages[1] = -1
    b.check(cuda_lib)
    b.lengths[1] = 5000  # past the table: the queries' own positions too
    b.check(cuda_lib)


@pytest.mark.parametrize("kind", ["f32", "bf16"])
def test_unseen_infinities_stay_out(cuda_lib, kind):
    """Later tokens of a chunk and keys before a window hold infinities and NaN: the rows that do not see them are exact."""
    q = 40
    b = Batch(kind, 4, 2, 128, 16, 48, [q + 30, q + 3], [q, q], seed=11)
    b.check(cuda_lib, window=25)
    want, tol = ref.attention(b.pool, b.q, b.starts, b.lengths, b.prefix_pages, b.prefix, 128 ** -0.5, 25, 4)
    pg, slot = b.pool.where(0, b.lengths[0])
    bad = b.lengths[0] - 5  # seen by the last five queries of sequence 0 only
    b.pool.values[pg[bad], :, slot[bad]] = float("nan")
    b.pool.keys[pg[bad], :, slot[bad]] = float("inf")
    out = b.run(cuda_lib, window=25)
    keep = torch.ones(2 * q, dtype=torch.bool, device="cuda")
    keep[q - 5:q] = False
    ref.check(out[keep], want[keep], tol[keep], 0.0, "rows that do not see the bad key")
    assert torch.isnan(out[~keep]).all()
    mid = b.lengths[1] - q - 5  # in the prefix; seen by the first 20 queries of sequence 1
    assert 0 <= mid < b.prefix
    b.pool.values[b.prefix_pages[mid // 16], :, mid % 16] = float("inf")
    out = b.run(cuda_lib, window=25)
    keep[q:q + 20] = False
    ref.check(out[keep], want[keep], tol[keep], 0.0, "rows that do not see the infinite value")
    assert not torch.isfinite(out[q:q + 20]).any()


def test_extreme_scores(cuda_lib):
    """Scores of hundreds (a softmax that is one key), and scale 0 (the mean)."""
    b = Batch("bf16", 4, 2, 64, 16, 64, [50, 3], [1, 1], seed=5)
    b.check(cuda_lib, scale=30.0)
    b.check(cuda_lib, scale=0.0)
    b.check(cuda_lib, scale=-0.5)


def test_strides_alignment_in_place_and_streams(cuda_lib):
    """Rows inside wider ones, a pool with gaps and an unaligned start, out over q, another stream."""
    for kind, gap, offset in (("bf16", 64, 0), ("bf16", 3, 1), ("f32", 4, 0), ("f16", 0, 3)):
        b = Batch(kind, 4, 2, 64, 16, 40, [70, 1, 9], [1, 4, 1], gap=gap, offset=offset, seed=gap)
        plain = b.check(cuda_lib)
        wide = torch.full((b.n, 4 * 64 + 13), 3.0, device="cuda", dtype=b.pool.dt)
        wide[:, 5:5 + 256] = b.q.view(b.n, 256)
        got = wide[:, 5:5 + 256]
        b.run(cuda_lib, q=got, out=got)
        assert torch.equal(got.reshape(plain.shape), plain)
        assert (wide[:, :5] == 3).all() and (wide[:, 261:] == 3).all()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            assert torch.equal(b.run(cuda_lib), plain)
            assert torch.equal(b.run(cuda_lib, flags=1), plain)


def test_same_result_twice_and_in_a_graph(cuda_lib):
    b = Batch("bf16", 16, 8, 128, 16, 512, [100, 5, 300, 41], [1, 1, 1, 1])
    first = b.run(cuda_lib).clone()
    assert torch.equal(b.run(cuda_lib), first)
    L, out = cuda_lib, torch.zeros_like(b.q)
    starts, lens = ints(b.starts), ints(b.lengths)
    need = L.dn_paged_attention_workspace(b.pool.c, 16, 4, 512, max(b.lengths))
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        assert L.dn_paged_attention(b.pool.c, b.q.data_ptr(), b.q.stride(0), starts.data_ptr(), lens.data_ptr(),
                                    b.prefix_pages.data_ptr(), 512, max(b.lengths), 128 ** -0.5, 0, out.data_ptr(),
                                    out.stride(0), 16, 4, ws.data_ptr(), need, 0, stream()) == 0
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    lens[2] = b.lengths[2] = 250  # lengths are read when the graph runs
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, b.run(cuda_lib))


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_offsets_past_32_bits(cuda_lib, kind):
    """Pages whose elements start past 2^32: append and attention at the end of a long pool."""
    L = cuda_lib
    dt, code, u = ref.TYPES[kind]
    from dianoia_b200 import _lib
    hd, page, pages = 64, 16, 8
    stride = ((1 << 32) // (pages - 3) + 4095) // 4096 * 4096  # the last pages start past 2^32 elements
    pool = torch.empty(pages * stride, dtype=dt, device="cuda")
    view = torch.as_strided(pool, (pages, 2, page, hd), (stride, page * hd, hd, 1))
    view.fill_(float("nan"))
    table = ints([[7, 6, 5], [3, 7, 6]])
    c = _lib.PagedCache(pool.data_ptr(), pool.data_ptr(), table.data_ptr(), code, pages, page, 1, hd, 1, 3, stride)
    # Keys in kv head 0's block, values in the block after it.
    c.values = pool.data_ptr() + page * hd * pool.element_size()
    n = 45
    k, v, q = (torch.randn((n, hd), device="cuda").to(dt) for _ in range(3))
    seq, pos = ints([0] * n), torch.arange(n, device="cuda", dtype=torch.int32)
    qo = torch.zeros_like(q)
    assert L.dn_paged_append(c, code, q.data_ptr(), hd, k.data_ptr(), hd, v.data_ptr(), hd, seq.data_ptr(), pos.data_ptr(),
                             None, 0, 0, None, None, 0.0, qo.data_ptr(), hd, 1, n, 0, stream()) == 0
    torch.cuda.synchronize()
    where = table[0].long()[torch.arange(n, device="cuda") // page], torch.arange(n, device="cuda") % page
    assert torch.equal(view[where[0], 0, where[1]], k) and torch.equal(view[where[0], 1, where[1]], v)
    assert torch.equal(qo, q)
    need = L.dn_paged_attention_workspace(c, 1, n, 0, n)
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    out = torch.zeros_like(q)
    assert L.dn_paged_attention(c, q.data_ptr(), hd, ints([0, n]).data_ptr(), ints([n]).data_ptr(), None, 0, n, 0.125, 0,
                                out.data_ptr(), hd, 1, n, ws.data_ptr(), need, 0, stream()) == 0
    torch.cuda.synchronize()
    s = (q.double() @ k.double().T) * 0.125
    s = s.masked_fill(torch.arange(n, device="cuda")[None] > torch.arange(n, device="cuda")[:, None], -torch.inf)
    p = torch.softmax(s, 1)
    want, a = p @ v.double(), p @ v.double().abs()
    mag = (q.double().abs() @ k.double().abs().T).amax(1, keepdim=True) * 0.125
    tol = (u * (kind != "f32") + 2 * (hd + 8) * ref.U32 * mag + (n + 64) * ref.U32) * a * (1 + u)
    ref.check(out, want, tol, u, "attention past 2^32")


def test_tokens_after_the_last_sequence_are_left_alone(cuda_lib):
    b = Batch("bf16", 4, 2, 64, 16, 32, [20, 30], [1, 2])
    out = torch.full((8, 4, 64), 7.0, device="cuda", dtype=b.pool.dt)
    q = torch.zeros_like(out)
    q[:3] = b.q
    n, b.n = b.n, 8
    b.run(cuda_lib, q=q, out=out)
    b.n = n
    assert torch.equal(out[:3], b.check(cuda_lib)) and (out[3:] == 7).all()


# ---------------------------------------------------------------------- append


def append(L, pool, kind, q, k, v, seq, pos, rope, rot, qn, kn, q_out, heads, eps=1e-6, flags=0):
    code = ref.TYPES[kind][1]
    return L.dn_paged_append(pool.c, code, q.data_ptr() if heads else None, q.stride(0) if heads else 0, k.data_ptr(),
                             k.stride(0), v.data_ptr(), v.stride(0), seq.data_ptr(), pos.data_ptr(),
                             rope.data_ptr() if rot else None, rope.shape[0], rot, qn.data_ptr() if qn is not None else None,
                             kn.data_ptr() if kn is not None else None, eps, q_out.data_ptr() if heads else None,
                             q_out.stride(0) if heads else 0, heads, seq.numel(), flags, stream())


def tables(rows, rot):
    at = torch.arange(rows, dtype=torch.float64, device="cuda")[:, None]
    ang = at * 1e4 ** (-torch.arange(rot // 2, dtype=torch.float64, device="cuda") * 2 / max(rot, 1))
    return torch.cat([ang.cos(), ang.sin()], 1).float()


@pytest.mark.parametrize("kind,cache", [("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16"),
                                        ("bf16", "f32"), ("f16", "bf16")])
@pytest.mark.parametrize("heads,kv_heads,hd,rot,page", [(16, 8, 128, 128, 16), (3, 1, 64, 32, 7), (0, 2, 256, 256, 32), (4, 2, 96, 48, 16),
                                                        (2, 2, 33, 10, 1), (5, 1, 80, 0, 16), (1, 1, 2, 2, 3), (4, 4, 128, 6, 16)])
@pytest.mark.parametrize("norm", [False, True])
def test_append(cuda_lib, kind, cache, heads, kv_heads, hd, rot, page, norm):
    """Three parts of one fused row, ragged sequences, padding and homeless tokens; nothing else of the pool changes."""
    L = cuda_lib
    dt, _, _ = ref.TYPES[kind]
    g = torch.Generator(device="cuda").manual_seed(hd + rot)
    rng = random.Random(hd)
    pool = ref.Pool(cache, 40, page, kv_heads, hd, 5, 6, fill=3.0)
    order = rng.sample(range(40), 30)
    pool.table.copy_(ints([order[6 * i:6 * i + 6] for i in range(5)]))
    pool.table[2, 1], pool.table[3, 0] = -1, 40
    tokens = [(s, p) for s in range(5) for p in rng.sample(range(6 * page), min(5, 6 * page))]
    tokens += [(-1, 0), (5, 0), (0, -1), (1, 6 * page), (1 << 30, 2), (2, page), (3, 0), (4, 6 * page - 1)]
    tokens = list(dict.fromkeys(tokens))
    n = len(tokens)
    rope_rows = 6 * page - 1  # the last position is past the rotation's table
    seq, pos = ints([s for s, _ in tokens]), ints([p for _, p in tokens])
    row = (heads + 2 * kv_heads) * hd
    fused = torch.randn((n, row + (5 if hd % 2 else 8)), generator=g, device="cuda").to(dt)
    q, k, v = fused[:, :heads * hd], fused[:, heads * hd:(heads + kv_heads) * hd], fused[:, (heads + kv_heads) * hd:row]
    rope = tables(rope_rows, rot)
    qn, kn = ((1 + 0.3 * torch.randn(hd, generator=g, device="cuda") for _ in range(2)) if norm else (None, None))
    q_out = torch.full((n, heads * hd), 9.0, device="cuda", dtype=pool.dt)
    before = [r.clone() for r in pool.raw]
    assert append(L, pool, kind, q, k, v, seq, pos, rope, rot, qn, kn, q_out, heads) == 0
    torch.cuda.synchronize()
    held = torch.zeros(n, dtype=torch.bool)
    for i, (s, p) in enumerate(tokens):
        if 0 <= s < 5 and 0 <= p < 6 * page and (rot == 0 or p < rope_rows):
            held[i] = 0 <= pool.table[s, p // page].item() < 40
    held = held.cuda()
    table = rope[pos.long().clamp(0, rope_rows - 1)]
    cos, sin = table[:, :rot // 2], table[:, rot // 2:]
    page_id = torch.where(held, pool.table[seq.long().clamp(0, 4), (pos.long() // page).clamp(0, 5)].long(), 0)
    slot = pos.long().clamp(min=0) % page
    want_k, tol_k = ref.rotated(k.reshape(n, kv_heads, hd), kn, 1e-6, cos, sin, rot)
    ref.check(pool.keys[page_id, :, slot][held], want_k[held], tol_k[held], pool.u, "keys")
    assert torch.equal(pool.values[page_id, :, slot][held], v.reshape(n, kv_heads, hd).float().to(pool.dt)[held])
    if heads:
        want_q, tol_q = ref.rotated(q.reshape(n, heads, hd), qn, 1e-6, cos, sin, rot)
        got = q_out.view(n, heads, hd)
        ref.check(got[held], want_q[held], tol_q[held], pool.u, "queries")
        assert (got[~held] == 0).all()
    # Nothing else of the pools changed.
    for r, b, name in zip(pool.raw, before, ("keys", "values")):
        view = getattr(pool, name)
        view[page_id[held], :, slot[held]] = 3.0
        assert torch.equal(r, b)


def test_append_in_place_and_unaligned(cuda_lib):
    """q rotated where it lies, and rows that start at odd addresses: the same bits as the aligned call."""
    L = cuda_lib
    pool = ref.Pool("bf16", 8, 16, 2, 64, 2, 4, fill=0.0)
    pool.table.copy_(ints([[0, 1, 2, 3], [4, 5, 6, 7]]))
    n = 50
    seq, pos = ints([i % 2 for i in range(n)]), ints([i // 2 for i in range(n)])
    fused = torch.randn((n, 6 * 64), device="cuda").to(torch.bfloat16)
    rope, w = tables(64, 64), torch.rand(64, device="cuda")
    out = torch.zeros((n, 2 * 64), device="cuda", dtype=torch.bfloat16)
    parts = lambda f: (f[:, :128], f[:, 128:256], f[:, 256:384])
    q, k, v = parts(fused)
    assert append(L, pool, "bf16", q, k, v, seq, pos, rope, 64, w, w, out, 2) == 0
    torch.cuda.synchronize()
    keys, values = pool.keys.clone(), pool.values.clone()
    odd = torch.zeros(n * 389 + 1, device="cuda", dtype=torch.bfloat16)[1:].view(n, 389)
    odd[:, :384] = fused
    q, k, v = parts(odd)
    pool.keys.zero_(), pool.values.zero_()
    assert append(L, pool, "bf16", q, k, v, seq, pos, rope, 64, w, w, q, 2, flags=1) == 0
    torch.cuda.synchronize()
    # The norm's sum runs in another order over unaligned rows: a last bit may differ.
    assert (q.float() - out.float()).abs().max() <= 2.0 ** -7 * out.float().abs().max()
    assert torch.equal(pool.values, values)
    assert (pool.keys.float() - keys.float()).abs().max() <= 2.0 ** -7 * keys.float().abs().max()
    assert torch.equal(odd[:, 128:384], fused[:, 128:]) and (odd[:, 384:] == 0).all()


def test_append_nothing(cuda_lib):
    pool = ref.Pool("bf16", 2, 16, 2, 64, 1, 2, fill=1.0)
    x = torch.zeros((1, 128), device="cuda", dtype=torch.bfloat16)
    assert append(cuda_lib, pool, "bf16", x, x, x, ints([]), ints([]), tables(4, 64), 64, None, None, x, 2) == 0


# -------------------------------------------------------------------- refusals


def changed(c, **kw):
    from dianoia_b200 import _lib
    d = _lib.PagedCache()
    ctypes.memmove(ctypes.byref(d), ctypes.byref(c), ctypes.sizeof(c))
    for k, v in kw.items():
        setattr(d, k, v)
    return d


BAD_CACHES = [(dict(type=3), -1), (dict(type=-1), -1), (dict(hd=0), -1), (dict(hd=257), -5), (dict(page_size=0), -1),
              (dict(kv_heads=0), -1), (dict(pages=-1), -1), (dict(page_stride=5), -1), (dict(sequences=-1), -1),
              (dict(table_stride=-1), -1), (dict(keys=None), -1), (dict(values=None), -1), (dict(table=None), -1),
              (dict(page_size=1 << 21), -5), (dict(table_stride=1 << 28), -5)]


def test_append_refusals(cuda_lib):
    L = cuda_lib
    pool = ref.Pool("bf16", 2, 16, 2, 64, 1, 2, fill=1.0)
    x = torch.zeros((4, 512), device="cuda")
    i, p, st = ints([0]).data_ptr(), x.data_ptr(), stream()
    base = dict(cache=pool.c, type=0, q=p, qs=128, k=p + 512, ks=128, v=p + 1024, vs=128, seq=i, pos=i, rope=p, rows=4, rot=64,
                qn=None, kn=None, eps=1e-6, qo=p + 4096, qos=128, heads=2, n=1, flags=0, st=st)
    call = lambda **kw: L.dn_paged_append(*{**base, **kw}.values())
    for kw, rc in BAD_CACHES:
        assert call(cache=changed(pool.c, **kw)) == rc, kw
    for kw, rc in [(dict(type=5), -1), (dict(n=-1), -1), (dict(heads=-1), -1), (dict(rot=3), -1), (dict(rot=66), -1), (dict(rot=-2), -1),
                   (dict(qs=127), -1), (dict(ks=64), -1), (dict(vs=64), -1), (dict(qos=100), -1), (dict(q=None), -1),
                   (dict(k=None), -1), (dict(v=None), -1), (dict(seq=None), -1), (dict(pos=None), -1), (dict(rope=None), -1),
                   (dict(q=p + 2), -1), (dict(k=p + 1), -1), (dict(qo=p + 4097), -1), (dict(qo=p), -1), (dict(qo=p + 256), -1),
                   (dict(cache=None), -1), (dict(rope=p + 2), -1), (dict(n=1 << 30), -5), (dict(ks=1 << 40), -5), (dict(rows=-1), -1)]:
        assert call(**kw) == rc, kw
    torch.cuda.synchronize()
    assert (pool.keys == 1).all()


def test_attention_refusals(cuda_lib):
    L = cuda_lib
    pool = ref.Pool("bf16", 2, 16, 2, 64, 2, 2, fill=1.0)
    x = torch.zeros((8, 512), device="cuda", dtype=torch.bfloat16)
    i, p, st = ints([0, 1, 2, 0]).data_ptr(), x.data_ptr(), stream()
    need = L.dn_paged_attention_workspace(pool.c, 4, 2, 16, 32)
    ws = torch.zeros(need + 16, dtype=torch.uint8, device="cuda")
    base = dict(cache=pool.c, q=p, qs=256, start=i, lens=i, pages=i, prefix=16, most=32, scale=1.0, window=0, out=p + 4096,
                os=256, heads=4, n=2, ws=ws.data_ptr(), bytes=need, flags=0, st=st)
    call = lambda **kw: L.dn_paged_attention(*{**base, **kw}.values())
    for kw, rc in BAD_CACHES:
        assert call(cache=changed(pool.c, **kw)) == rc, kw
        assert L.dn_paged_attention_workspace(changed(pool.c, **kw), 4, 2, 16, 32) == rc, kw
    for kw, rc in [(dict(heads=3), -1), (dict(heads=0), -1), (dict(n=-1), -1), (dict(prefix=-1), -1), (dict(window=-1), -1),
                   (dict(qs=255), -1), (dict(os=255), -1), (dict(q=None), -1), (dict(out=None), -1), (dict(lens=None), -1),
                   (dict(ws=None), -1), (dict(bytes=need - 1), -1), (dict(bytes=0), -1), (dict(pages=None), -1), (dict(q=p + 1), -1),
                   (dict(ws=ws.data_ptr() + 8), -1), (dict(out=p + 2), -1), (dict(start=None, n=3), -1), (dict(most=-1), -1),
                   (dict(window=1 << 33), -1), (dict(n=1 << 29), -5), (dict(qs=1 << 40), -5), (dict(cache=None), -1),
                   (dict(lens=i + 1), -1)]:
        assert call(**kw) == rc, kw
    for args in [(3, 2, 16, 32), (4, -1, 16, 32), (4, 2, -1, 32), (4, 2, 16, -1)]:
        assert L.dn_paged_attention_workspace(pool.c, *args) == -1, args
    assert call(n=0) == 0


@pytest.mark.parametrize("own", [1, 120])
def test_both_kernels_at_once_repeat_and_replay(cuda_lib, own):
    """Many rows on the prefix beside each sequence's own: the same bits every time, back to back, with programmatic launch and in a graph."""
    L = cuda_lib
    seqs, heads = 100, 8
    b = Batch("bf16", heads, 2, 128, 16, 1200, [1 + (own * (i % 7)) // 6 for i in range(seqs)], [1] * seqs, seed=own)
    first = b.check(L).clone()
    starts, lens = ints(b.starts), ints(b.lengths)
    most = max(b.lengths)
    need = L.dn_paged_attention_workspace(b.pool.c, heads, b.n, b.prefix, most)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    outs = [torch.zeros_like(b.q) for _ in range(8)]

    def call(out, flags):
        assert L.dn_paged_attention(b.pool.c, b.q.data_ptr(), b.q.stride(0), starts.data_ptr(), lens.data_ptr(),
                                    b.prefix_pages.data_ptr(), b.prefix, most, 128 ** -0.5, 0, out.data_ptr(), out.stride(0), heads,
                                    b.n, ws.data_ptr(), need, flags, stream()) == 0

    for flags in (0, 1):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for out in outs:
            call(out, flags)
        torch.cuda.synchronize()
        assert all(torch.equal(out, first) for out in outs)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for i, out in enumerate(outs):
            call(out, i % 2)
    for _ in range(3):
        for out in outs:
            out.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, first) for out in outs)
    assert L.dn_device_status(1) == 0


# ---- heads between two panel counts, after other heads have used the same shared memory


def spoil(L, kind, hd, wide, value):
    """A pass over keys and values of `value` that fills the kernel's shared memory on every SM."""
    seqs, q = (40, 40) if wide else (500, 1)
    b = Batch(kind, 4, 2, hd, 16, 0, [64] * seqs, [q] * seqs, seed=1)
    b.pool.keys.fill_(value), b.pool.values.fill_(value)
    b.run(L)


@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [136, 160, 192, 200])
@pytest.mark.parametrize("page", [16, 7])
@pytest.mark.parametrize("group,q", [(2, 1), (12, 1), (2, 40)])
def test_heads_whose_last_panel_is_not_copied(cuda_lib, kind, hd, page, group, q):
    """Heads of 129 to 192 elements fill three of the four panels of their kernel: what another call left in the
    fourth, NaN and large values, does not reach a score. Thin blocks of 8 and of 16 rows, and wide ones."""
    own = [70, 45, 130, 64]
    b = Batch(kind, group * 2, 2, hd, page, 48, [max(k, q) for k in own], [q] * 4, seed=hd + q)
    for value in (float("nan"), 6e4, 1.0):
        spoil(cuda_lib, kind, 256, q > 1, value)
        b.check(cuda_lib, max_length=4096)
        spoil(cuda_lib, kind, 256, q > 1, value)
        b.check(cuda_lib)



@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("page", [32, 64, 96])
@pytest.mark.parametrize("prefix", [16, 48, 96, 208])
@pytest.mark.parametrize("shape", ["queries", "heads"])
def test_short_sequences_of_many_rows_behind_a_prefix_inside_a_page(cuda_lib, kind, page, prefix, shape):
    """Short sequences that read the prefix themselves, with rows enough for the wide kernel: keys after the prefix's
    end come from the sequence's own page, also where one page's worth of copies spans the end."""
    if shape == "queries":
        b = Batch(kind, 4, 2, 64, page, prefix, [112, 60, 45], [40] * 3, seed=prefix)
    else:
        b = Batch(kind, 40, 1, 128, page, prefix, [30, 1], [1, 1], seed=prefix)
    assert max(b.lengths) <= 512 and len(b.lengths) * prefix <= 8192
    b.check(cuda_lib)
    b.check(cuda_lib, window=70)
    b.check(cuda_lib, max_length=5000)



@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("hd", [136, 160, 192])
def test_result_does_not_depend_on_what_ran_before(cuda_lib, kind, hd):
    """Many rows with a window (tiles whose values are looked at): the same bits after any other call."""
    b = Batch(kind, 4, 2, hd, 16, 0, [300, 211], [90, 90], seed=hd)
    outs = []
    for value in (0.0, float("nan"), 6e4, float("inf"), 0.0):
        spoil(cuda_lib, kind, 256, True, value)
        outs.append(b.check(cuda_lib, window=50).clone())
    assert all(torch.equal(o, outs[0]) for o in outs)



@pytest.mark.parametrize("kind,hd", [("f32", 64), ("bf16", 64), ("f16", 33)])
@pytest.mark.parametrize("prefix", [0, 32])
@pytest.mark.parametrize("n", [1, 3, 100])
def test_tokens_without_sequences_are_left_alone(cuda_lib, kind, hd, prefix, n):
    """A batch of no sequences: every token lies past q_start[0]."""
    from dianoia_b200 import _lib
    L = cuda_lib
    dt, code, _ = ref.TYPES[kind]
    pool = ref.Pool(kind, 4, 16, 2, hd, 1, 2, fill=1.0)
    c = changed(pool.c, sequences=0)
    q, out = torch.ones((n, 4, hd), device="cuda", dtype=dt), torch.full((n, 4, hd), 7.0, device="cuda", dtype=dt)
    starts, lens, pages = ints([0]), ints([0]), ints([0, 1])
    need = L.dn_paged_attention_workspace(c, 4, n, prefix, 64)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    assert L.dn_paged_attention(c, q.data_ptr(), 4 * hd, starts.data_ptr(), lens.data_ptr(), pages.data_ptr(), prefix, 64, 0.125, 0,
                                out.data_ptr(), 4 * hd, 4, n, ws.data_ptr(), need, 0, stream()) == _lib.DN_OK
    torch.cuda.synchronize()
    assert (out == 7).all()



@pytest.mark.parametrize("kind,page", [("f32", 16), ("bf16", 16), ("bf16", 7), ("f16", 64)])
@pytest.mark.parametrize("q", [1, 40])
def test_prefix_needs_no_table(cuda_lib, kind, page, q):
    """Sequences that lie in the prefix altogether, behind tables that end before it: the prefix is read through its
    own pages, whatever length the batch is said to have."""
    prefix = 128
    b = Batch(kind, 4, 2, 64, page, prefix, [0, 0, 0], [q] * 3, seed=q)
    b.lengths = [128, 100, 40]
    b.pool.table = b.pool.table[:, :1].contiguous()
    b.pool.c.table, b.pool.c.table_stride = b.pool.table.data_ptr(), 1
    b.check(cuda_lib)
    b.check(cuda_lib, max_length=5000)
    b.check(cuda_lib, window=30)
    b.lengths[0] = 140  # its last positions have no page
    b.check(cuda_lib)



@pytest.mark.parametrize("kind,hd", [("f32", 64), ("f16", 64), ("bf16", 128), ("bf16", 20)])
@pytest.mark.parametrize("q", [6, 40])
def test_seen_infinities_count_however_small_their_weight(cuda_lib, kind, hd, q):
    """A value that is not finite, at a key that a query sees with a weight below every type's least: the query's output
    is not finite, whether the rows beside it see the same keys or not."""
    b = Batch(kind, 4, 2, hd, 16, 0, [90, 90], [q, q], seed=hd)
    b.q.fill_(1.0)
    b.pool.keys[torch.isfinite(b.pool.keys)] = 0.0
    for at, value in ((3, float("inf")), (90 - 4, float("nan"))):  # seen by all, by the last four queries
        pg, slot = b.pool.where(0, 90)
        b.pool.keys[pg[at], :, slot[at]] = -60.0  # a score of -60 hd
        b.pool.values[pg[at], :, slot[at]] = value
    out = b.run(cuda_lib, scale=1.0)
    assert not torch.isfinite(out[:q]).any()
    assert torch.isfinite(out[q:]).all()
    out = b.run(cuda_lib, scale=1.0, window=40)  # now position 3 is behind every window
    assert torch.isfinite(out[:q - 4]).all() and not torch.isfinite(out[q - 4:q]).any()



@pytest.mark.parametrize("kind", ["f16", "bf16"])
@pytest.mark.parametrize("shared", [False, True])
def test_many_small_probabilities_beside_a_large_one(cuda_lib, kind, shared):
    """One key of weight near 1 and value 0 (where attention goes that has nowhere to go), and 131071 of weight e^-18
    and value 1 behind it: their sum reaches the output. Batches large enough that no slice is short."""
    L = cuda_lib
    dt, code, u = ref.TYPES[kind]
    from dianoia_b200 import _lib
    keys, page, hd = 1 << 17, 64, 64
    seqs, heads = (75, 128) if shared else (600, 4)
    pages = keys // page
    pool = ref.Pool(kind, pages, page, 1, hd, seqs, pages + 1, fill=0.0)
    pool.table[:, :pages] = torch.arange(pages, device="cuda", dtype=torch.int32)  # one sequence's pages for all
    pool.values.fill_(1.0)
    pool.keys[0, 0, 3, 0], pool.values[0, 0, 3] = 4.0, 0.0
    q = torch.zeros((seqs, heads, hd), device="cuda", dtype=dt)
    q[:, :, 0] = 4.5
    out = torch.full_like(q, 7.0)
    prefix = keys if shared else 0
    lens = ints([keys] * seqs)
    need = L.dn_paged_attention_workspace(pool.c, heads, seqs, prefix, keys)
    ws = torch.full((need,), 255, dtype=torch.uint8, device="cuda")
    assert L.dn_paged_attention(pool.c, q.data_ptr(), heads * hd, None, lens.data_ptr(), pool.table[0].data_ptr(), prefix, keys, 1.0, 0,
                                out.data_ptr(), heads * hd, heads, seqs, ws.data_ptr(), need, 0, stream()) == 0
    torch.cuda.synchronize()
    import math
    tail = (keys - 1) * math.exp(-18.0)
    want = torch.full_like(out, tail / (1 + tail), dtype=torch.float64)
    # The probabilities' rounding: u of each, and in f16, whose numbers end at 2^-24, half of that for each key against
    # a largest probability of 2^7 at least; scores and sums in f32 as in the reference's bound (mag 18).
    a = want[0, 0, 0].item()
    small = keys * 2.0 ** -25 * 2.0 ** -7 if kind == "f16" else 0.0
    tol = small + a * (u + 2 * (hd + 8) * ref.U32 * 18 + (keys + 64) * ref.U32) * (1 + u)
    ref.check(out, want, torch.full_like(want, tol), u, "small probabilities")


def test_waits_that_run_out_leave_nothing_in_flight(cuda_lib):
    """With a wait limit far shorter than a copy takes, calls come back (their outputs may be incomplete, and the status
    word says so with the bits of a copy or of a product alone) and the next ones with the usual limit are right."""
    L = cuda_lib
    batches = [Batch("bf16", 4, 2, 64, 16, 48, [300, 64, 77], [1, 1, 1], seed=1),  # copied by tiles
               Batch("f16", 4, 2, 96, 7, 0, [300, 64, 77], [1, 9, 1], seed=2),  # by the lanes
               Batch("bf16", 8, 2, 128, 16, 1200, [40] * 60, [1] * 60, seed=3),  # wide blocks beside thin ones
               Batch("f16", 4, 1, 192, 32, 0, [500, 90], [90, 90], seed=4)]
    firsts = [b.check(L).clone() for b in batches]
    assert L.dn_device_status(1) == 0
    torch.cuda.synchronize()
    assert L.dn_set_wait_limit_ns(1) == 0
    try:
        for b in batches:
            for _ in range(3):
                b.run(L)
    finally:
        torch.cuda.synchronize()
        assert L.dn_set_wait_limit_ns(0) == 0
    assert L.dn_device_status(1) & ~(1 | 4) == 0
    for b, first in zip(batches, firsts):
        assert torch.equal(b.run(L), first)
    assert L.dn_device_status(1) == 0
