"""dn_logits_apply against its definition in 64 bits (tests/paged_reference.py
derives the bound): every rule alone and together, vocabularies and strides of
any alignment, duplicates, ids outside the vocabulary, masks that leave nothing,
infinities and NaN, and refusals."""
import random

import pytest

from tests import paged_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def stream():
    return torch.cuda.current_stream().cuda_stream


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def make_rules(n, vocab, names, seed=0, history=200, biases=20):
    rng, g = random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)
    r = {}
    if "history" in names:
        lens = [rng.choice([0, 1, rng.randint(0, history)]) for _ in range(n)]
        r["history"] = ints([3 + sum(lens[:i]) for i in range(n + 1)], torch.int64)  # rows need not start at 0
        ids = [rng.choice([0, vocab - 1, rng.randrange(vocab), rng.randrange(min(vocab, 9)), -1, vocab, 1 << 30, -(1 << 31)])
               for _ in range(3 + sum(lens))]
        r["tokens"] = ints(ids)
        if "generated" in names:
            r["generated"] = ints([rng.randint(0, k) for k in lens])
        for name, of in (("repetition", [1.0, 1.3, 0.7]), ("frequency", [0.0, 0.3, -0.2]), ("presence", [0.5, 0.0, -0.4])):
            if name in names:
                r[name] = ints([rng.choice(of) for _ in range(n)], torch.float32)
    if "bias" in names:
        lens = [rng.choice([0, 1, rng.randint(0, biases)]) for _ in range(n)]
        r["bias_start"] = ints([sum(lens[:i]) for i in range(n + 1)], torch.int64)
        ids = [rng.choice([rng.randrange(vocab), rng.randrange(min(vocab, 4)), -1, vocab]) for _ in range(sum(lens) + 1)]
        r["bias_tokens"], r["bias"] = ints(ids), torch.randn(len(ids), generator=g, device="cuda") * 3
    if "mask" in names:
        rows = n if "mask_row" not in names else max(1, n // 2)
        words = (vocab + 31) // 32 + 1
        r["mask"] = torch.randint(-(1 << 31), 1 << 31, (rows, words), generator=g, device="cuda", dtype=torch.int64).to(torch.int32)
        r["mask"][0] = 0  # a mask that allows nothing
        if "mask_row" in names:
            r["mask_row"] = ints([rng.choice([-1, rows, rng.randrange(rows)]) for _ in range(n)])
    return r


def descriptor(r):
    from dianoia_b200 import _lib
    p = lambda k: r[k].data_ptr() if r.get(k) is not None else None
    return _lib.LogitRules(p("tokens"), p("history"), p("generated"), p("repetition"), p("frequency"), p("presence"),
                           p("bias_tokens"), p("bias"), p("bias_start"), p("mask"), p("mask_row"),
                           r["mask"].shape[0] if "mask" in r else 0, r["mask"].shape[1] if "mask" in r else 0)


def apply(L, kind, x, out, vocab, rules, flags=0):
    rc = L.dn_logits_apply(ref.TYPES[kind][1], x.data_ptr(), x.stride(0), out.data_ptr(), out.stride(0), x.shape[0], vocab,
                           descriptor(rules), flags, stream())
    torch.cuda.synchronize()
    return rc


ALL = ("history", "generated", "repetition", "frequency", "presence", "bias", "mask", "mask_row")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n,vocab", [(1, 1), (3, 7), (5, 4096), (4, 4097), (7, 50257), (2, 151936), (33, 1000)])
def test_all_rules(cuda_lib, kind, n, vocab):
    dt, _, u = ref.TYPES[kind]
    rules = make_rules(n, vocab, ALL, seed=vocab)
    x = (torch.randn((n, vocab), device="cuda") * 4).to(dt)
    out = torch.full_like(x, 7.0)
    assert apply(cuda_lib, kind, x, out, vocab, rules) == 0
    want, tol = ref.logits(x, rules, vocab)
    ref.check(out, want, tol, u, "logits")


@pytest.mark.parametrize("names", [(), ("history", "repetition"), ("history", "frequency"), ("history", "generated", "presence"), ("history",),
                                   ("bias",), ("mask",), ("mask", "mask_row"), ("bias", "mask"), ("history", "repetition", "mask")])
def test_each_rule_alone(cuda_lib, names):
    rules = make_rules(6, 9001, names, seed=len(names))
    x = torch.randn((6, 9001), device="cuda") * 4
    out = torch.full_like(x, 7.0)
    assert apply(cuda_lib, "f32", x, out, 9001, rules) == 0
    want, tol = ref.logits(x, rules, 9001)
    ref.check(out, want, tol, ref.U32, str(names))
    if not names:
        assert torch.equal(out, x)


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
def test_strides_alignment_and_in_place(cuda_lib, kind):
    """Rows at every alignment of in and out, in place, another stream: the same bits; nothing past the vocabulary is written."""
    dt, _, u = ref.TYPES[kind]
    n, vocab = 9, 5003
    rules = make_rules(n, vocab, ALL, seed=4)
    x = (torch.randn((n, vocab), device="cuda") * 4).to(dt)
    first = torch.empty_like(x)
    assert apply(cuda_lib, kind, x, first, vocab, rules) == 0
    want, tol = ref.logits(x, rules, vocab)
    ref.check(first, want, tol, u, "logits")
    for off_in, off_out, more_in, more_out in ((0, 0, 5, 5), (1, 1, 0, 0), (3, 1, 2, 7), (0, 5, 5, 5), (2, 2, 5, 13)):
        a = torch.full((n * (vocab + more_in) + off_in,), 5.0, device="cuda", dtype=dt)[off_in:].view(n, vocab + more_in)
        b = torch.full((n * (vocab + more_out) + off_out,), 5.0, device="cuda", dtype=dt)[off_out:].view(n, vocab + more_out)
        a[:, :vocab] = x
        assert apply(cuda_lib, kind, a, b, vocab, rules) == 0
        assert torch.equal(b[:, :vocab], first) and (b[:, vocab:] == 5).all()
        assert apply(cuda_lib, kind, a, a, vocab, rules, flags=1) == 0
        assert torch.equal(a[:, :vocab], first) and (a[:, vocab:] == 5).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = torch.empty_like(x)
        assert apply(cuda_lib, kind, x, out, vocab, rules) == 0
        assert torch.equal(out, first)


def test_infinities_nan_and_empty_masks(cuda_lib):
    """A masked logit gives minus infinity whatever it was; others keep their infinities and NaN."""
    vocab = 300
    x = torch.randn((3, vocab), device="cuda")
    x[:, 10], x[:, 11], x[:, 12], x[:, 40], x[:, 41] = float("nan"), float("inf"), -float("inf"), float("nan"), float("inf")
    x[:, 50] = torch.finfo(torch.float32).min
    mask = torch.full((3, 10), -1, dtype=torch.int32, device="cuda")
    mask[:, 1] = 0  # tokens 32 .. 63
    mask[2] = 0
    out = torch.empty_like(x)
    assert apply(cuda_lib, "f32", x, out, vocab, {"mask": mask}) == 0
    want = x.clone()
    want[:, 32:64] = -float("inf")
    want[2] = -float("inf")
    assert torch.equal(out.nan_to_num(nan=9e9), want.nan_to_num(nan=9e9))


def test_counts_of_long_histories(cuda_lib):
    """One token 70000 times, and a long history: counts do not saturate."""
    vocab = 6000
    g = torch.Generator(device="cuda").manual_seed(1)
    tokens = torch.cat([torch.full((70000,), 4095, device="cuda"), torch.randint(0, vocab, (50000,), generator=g, device="cuda")]).int()
    rules = {"tokens": tokens, "history": ints([0, 120000], torch.int64), "frequency": ints([0.01], torch.float32),
             "presence": ints([0.1], torch.float32), "repetition": ints([1.2], torch.float32)}
    x = torch.randn((1, vocab), generator=g, device="cuda")
    out = torch.empty_like(x)
    assert apply(cuda_lib, "f32", x, out, vocab, rules) == 0
    want, tol = ref.logits(x, rules, vocab)
    ref.check(out, want, tol, ref.U32, "counts")


def test_biases_add_in_list_order(cuda_lib):
    """Many biases on one token add one after the other, the same each time."""
    k = 500
    b = torch.randn(k, device="cuda") * torch.logspace(-6, 6, k, device="cuda")
    rules = {"bias_start": ints([0, k], torch.int64), "bias_tokens": ints([77] * k), "bias": b}
    x = torch.zeros((1, 200), device="cuda")
    out = torch.empty_like(x)
    assert apply(cuda_lib, "f32", x, out, 200, rules) == 0
    import numpy as np
    total = np.float32(0)
    for v in b.cpu().numpy():
        total = np.float32(total + v)
    assert out[0, 77].item() == float(total) and out.abs().sum().item() == abs(float(total))


def test_refusals(cuda_lib):
    from dianoia_b200 import _lib
    L = cuda_lib
    x = torch.zeros((4, 64), device="cuda")
    z = torch.zeros(64, dtype=torch.int64, device="cuda").data_ptr()
    y = torch.full((4, 64), 5.0, device="cuda")
    none = lambda **kw: _lib.LogitRules(**kw)
    base = dict(type=0, x=x.data_ptr(), s=64, out=y.data_ptr(), os=64, n=4, vocab=64, rules=none(), flags=0, st=stream())
    call = lambda **kw: L.dn_logits_apply(*{**base, **kw}.values())
    for kw, rc in [(dict(type=3), -1), (dict(n=-1), -1), (dict(vocab=-1), -1), (dict(s=63), -1), (dict(os=63), -1), (dict(rules=None), -1),
                   (dict(x=None), -1), (dict(out=None), -1), (dict(x=x.data_ptr() + 2), -1), (dict(out=x.data_ptr() + 4), -1),
                   (dict(vocab=1 << 31, s=1 << 31, os=1 << 31), -5), (dict(s=1 << 41), -5),
                   (dict(rules=none(history=z)), -1), (dict(rules=none(bias_start=z)), -1),
                   (dict(rules=none(bias_start=z, bias=z)), -1), (dict(rules=none(mask=z, mask_rows=4, mask_stride=1)), -1),
                   (dict(rules=none(mask=z, mask_rows=3, mask_stride=2)), -1), (dict(rules=none(history=z + 4, tokens=z)), -1),
                   (dict(rules=none(history=z, tokens=z + 2)), -1), (dict(rules=none(mask=z, mask_rows=-1, mask_stride=2, mask_row=z)), -1)]:
        assert call(**kw) == rc, kw
    torch.cuda.synchronize()
    assert (y == 5).all()
    assert call(n=0) == 0 and call(vocab=0) == 0
    assert call() == 0


@pytest.mark.parametrize("kind", ["f32", "bf16"])
@pytest.mark.parametrize("repeats,others", [(2, 3), (20, 0), (30, 30)])
def test_repeated_biases_and_penalties_on_one_token(cuda_lib, kind, repeats, others):
    """A token that is seen, generated and biased several times, few or many biases in its range."""
    dt, _, u = ref.TYPES[kind]
    vocab = 5000
    g = torch.Generator(device="cuda").manual_seed(repeats)
    ids = [4090] * repeats + [4091 + i for i in range(others)]
    rules = {"bias_start": ints([0, len(ids)], torch.int64), "bias_tokens": ints(ids),
             "bias": torch.randn(len(ids), generator=g, device="cuda"),
             "history": ints([0, 5], torch.int64), "tokens": ints([4090, 7, 4090, 4092, 4090]), "generated": ints([3]),
             "repetition": ints([1.5], torch.float32), "frequency": ints([0.25], torch.float32),
             "presence": ints([0.5], torch.float32)}
    x = (torch.randn((1, vocab), generator=g, device="cuda") * 3).to(dt)
    out = torch.empty_like(x)
    assert apply(cuda_lib, kind, x, out, vocab, rules) == 0
    want, tol = ref.logits(x, rules, vocab)
    # Each bias rounds once more: the running sum is at most the terms' magnitudes.
    tol = tol + len(ids) * ref.U32 * (x[:1].double().abs() * 1.5 + 2 + rules["bias"].double().abs().sum())
    ref.check(out, want, tol, u, "biases")


@pytest.mark.parametrize("kind", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("vocab", [*range(4089, 4099), *range(8185, 8195), 32766, 65535])
def test_vocabularies_around_whole_ranges(cuda_lib, kind, vocab):
    """Vocabularies that end just before, at and after a multiple of a CTA's 4096 tokens, rows at every alignment,
    copied whole and element by element: a last CTA without tokens leaves everything alone."""
    dt, _, u = ref.TYPES[kind]
    n, whole = 3, 16 // dt.itemsize
    rules = make_rules(n, vocab, ALL, seed=vocab, history=300, biases=90)
    x = (torch.randn((n, vocab), device="cuda") * 4).to(dt)
    want, tol = ref.logits(x, rules, vocab)
    tol = tol * (6 + 90) / 6  # one more rounding for each of up to 90 biases of a token
    stride = -(-vocab // whole) * whole + whole  # every row at the alignment of the first
    first = None
    for off_in in range(whole):
        for off_out in (off_in, (off_in + 1) % whole):
            a = torch.full((n * stride + whole,), 5.0, device="cuda", dtype=dt)
            b = torch.full_like(a, 6.0)
            rows_in = a[off_in:off_in + n * stride].view(n, stride)
            rows_out = b[off_out:off_out + n * stride].view(n, stride)
            rows_in[:, :vocab] = x
            assert apply(cuda_lib, kind, rows_in, rows_out, vocab, rules) == 0
            got = rows_out[:, :vocab].clone()
            if first is None:
                first = got
                ref.check(first, want, tol, u, "logits")
            assert torch.equal(got, first)
            rows_out[:, :vocab] = 6.0
            assert (b == 6).all()
    assert cuda_lib.dn_device_status(1) == 0


def test_a_wait_that_runs_out_leaves_nothing_in_flight(cuda_lib):
    """With a wait limit shorter than a copy takes, calls come back, their status bit a copy's alone; the next one is right."""
    L, vocab = cuda_lib, 50257
    rules = make_rules(20, vocab, ALL, seed=9)
    x = torch.randn((20, vocab), device="cuda")
    first, out = torch.empty_like(x), torch.empty_like(x)
    assert apply(L, "f32", x, first, vocab, rules) == 0
    assert L.dn_set_wait_limit_ns(1) == 0
    try:
        for _ in range(3):
            assert apply(L, "f32", x, out, vocab, rules) == 0
    finally:
        torch.cuda.synchronize()
        assert L.dn_set_wait_limit_ns(0) == 0
    assert L.dn_device_status(1) & ~1 == 0
    assert apply(L, "f32", x, out, vocab, rules) == 0
    assert torch.equal(out, first) and L.dn_device_status(1) == 0
