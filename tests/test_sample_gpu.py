"""dn_sample against its definition in 64 bits: every rule alone and together,
ties, rows that a mask leaves empty or nearly so, infinities and NaN, every
type and alignment, vocabularies from none to the largest.

The kernel's sums are exact in steps of 2^-44 of the largest weight, the
reference's are f64: the two agree wherever no border lies next to the random
number's, top_p's or min_p's place (ref.choose says how near that is); a case's
seed is one where none does, which the tests assert."""
import math
import random

import numpy as np
import pytest

from tests import paged_q8_reference as ref

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

from dianoia_b200 import _lib  # noqa: E402

TYPES = ref.TYPES


def stream():
    return torch.cuda.current_stream().cuda_stream


def vec(values, dtype=torch.float32):
    return None if values is None else torch.tensor(values, dtype=dtype, device="cuda")


NAMES = ("temperature", "top_k", "top_p", "min_p", "u")


def run(L, logits, rules, flags=0):
    """tokens, logprobs, kept of rows under `rules` (dict of lists)."""
    n, vocab = logits.shape
    t = {k: vec(rules.get(k), torch.int32 if k == "top_k" else torch.float32) for k in NAMES}
    how = _lib.Sampling(*(None if t[k] is None else t[k].data_ptr() for k in NAMES))
    tokens, kept = (torch.full((n,), 77, dtype=torch.int32, device="cuda") for _ in range(2))
    logprobs = torch.full((n,), 7.0, device="cuda")
    kind = {v[0]: v[1] for v in TYPES.values()}[logits.dtype]
    assert L.dn_sample(kind, logits.data_ptr(), logits.stride(0), n, vocab, how, tokens.data_ptr(), logprobs.data_ptr(),
                       kept.data_ptr(), flags, stream()) == 0
    torch.cuda.synchronize()
    return tokens.tolist(), logprobs.tolist(), kept.tolist()


def check(L, logits, rules, some=False):
    """Every row's choice is determined, or, with `some`, is looked at where it is, in half of the rows at least."""
    got, unclear = run(L, logits, rules), 0
    x = logits.double().cpu().numpy()
    n, vocab = x.shape
    for r in range(n):
        one = {k: (np.float32(v[r]) if k != "top_k" else v[r]) for k, v in rules.items()}
        token, logprob, kept, margin = ref.choose(x[r], **one)
        if some and not margin > 1:
            unclear += 1
            continue
        assert margin > 1, "a border next to a place that decides: another seed"
        assert (got[0][r], got[2][r]) == (token, kept), (r, one)
        # The share's rounding to f32 after steps of 2^-45 of each weight: relative to the token's own weight.
        if math.isinf(logprob):
            assert got[1][r] == logprob
        else:
            assert abs(got[1][r] - logprob) <= 2.0 ** -24 * abs(logprob) + 2.0 ** -45 * vocab / math.exp(max(logprob, -20)) + 1e-12
    assert 2 * unclear <= n
    return got


def logits_of(kind, n, vocab, seed, spread=3.0, offset=0, pad=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    raw = torch.zeros(n * (vocab + pad) + offset, device="cuda", dtype=TYPES[kind][0])
    x = raw[offset:].view(n, vocab + pad)[:, :vocab]
    x.copy_(torch.randn((n, vocab), generator=g, device="cuda") * spread)
    return x


def rules_of(n, which, seed, vocab):
    rng = random.Random(seed)
    r = {"u": [rng.random() for _ in range(n)]}
    if "t" in which:
        r["temperature"] = [rng.choice([0.3, 0.7, 1.0, 1.5, 4.0]) for _ in range(n)]
    if "k" in which:
        r["top_k"] = [rng.choice([0, 1, 2, 3, 20, 50, 1000, vocab, vocab + 1, -1, rng.randint(1, vocab)]) for _ in range(n)]
    if "p" in which:
        r["top_p"] = [rng.choice([0.1, 0.5, 0.9, 0.99, 1.0, rng.random()]) for _ in range(n)]
    if "m" in which:
        r["min_p"] = [rng.choice([0.0, 0.01, 0.1, 0.5, 0.99, rng.random()]) for _ in range(n)]
    return r


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("which", ["", "t", "k", "p", "m", "kp", "tkpm", "pm", "km"])
@pytest.mark.parametrize("vocab", [1, 2, 33, 1000, 4097, 50257])
def test_rules(cuda_lib, kind, which, vocab):
    n = 13
    check(cuda_lib, logits_of(kind, n, vocab, vocab), rules_of(n, which, vocab, vocab))


@pytest.mark.parametrize("kind,vocab,n", [("f32", 151936, 3), ("bf16", 151936, 3), ("f32", 524288, 2), ("f16", 524287, 2), ("f32", 262145, 2)])
def test_large_vocabularies(cuda_lib, kind, vocab, n):
    for which in ("t", "kp", "p", "m"):
        for spread in (0.5, 2.5):
            check(cuda_lib, logits_of(kind, n, vocab, 5, spread), rules_of(n, which, 6, vocab))


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("offset,pad", [(0, 1), (1, 0), (3, 5), (0, 8)])
def test_alignment(cuda_lib, kind, offset, pad):
    for vocab in (64, 1001, 20000):
        check(cuda_lib, logits_of(kind, 6, vocab, 3, offset=offset, pad=pad), rules_of(6, "tkpm", 4, vocab))


@pytest.mark.parametrize("vocab", [7, 1000, 33000])
def test_ties(cuda_lib, vocab):
    """Few different logits: cuts fall among equal tokens, the lowest indices stay."""
    rng = random.Random(vocab)
    n = 24
    x = torch.randint(0, 4, (n, vocab), generator=torch.Generator(device="cuda").manual_seed(vocab), device="cuda").float()
    x[1] = 2.5
    x[2] = -0.0
    x[2, ::2] = 0.0
    rules = {"u": [rng.random() * 0.999 + 0.0003 for _ in range(n)], "top_k": [rng.choice([0, 0, 1, 2, vocab // 2, vocab - 1, 100]) for _ in range(n)],
             "top_p": [rng.choice([1.0, 0.3017, 0.7013, 0.9011]) for _ in range(n)]}
    for kind in TYPES:
        check(cuda_lib, x.to(TYPES[kind][0]), rules)


def test_equal_tokens_by_share(cuda_lib):
    """Equal logits: half of the tokens at top_p a half, exactly."""
    for vocab in (2, 1000, 4096):
        x = torch.full((1, vocab), 1.25, device="cuda")
        tokens, _, kept = run(cuda_lib, x, {"u": [0.0], "top_p": [0.5]})
        assert kept == [vocab // 2] and tokens == [0]
        tokens, logprobs, kept = run(cuda_lib, x, {"u": [0.75]})
        assert kept == [vocab] and tokens == [vocab * 3 // 4] and abs(logprobs[0] + math.log(vocab)) < 1e-6


def test_greedy(cuda_lib):
    inf, nan = math.inf, math.nan
    x = logits_of("f32", 8, 5000, 1)
    x[3, 17] = x[3, 4000] = 50.0
    x[4, 4999] = inf
    for t in (0.0, -1.0, nan):
        tokens, logprobs, kept = run(cuda_lib, x, {"u": [0.999] * 8, "temperature": [t] * 8, "top_k": [50] * 8, "top_p": [0.9] * 8})
        assert tokens == [int(np.argmax(r)) for r in x.cpu().numpy()] and tokens[3] == 17
        assert logprobs == [0.0] * 8 and kept == [1] * 8


def test_empty_and_odd_rows(cuda_lib):
    inf, nan = math.inf, math.nan
    for vocab in (40, 9000):
        x = torch.full((7, vocab), -inf, device="cuda")
        x[1] = nan
        x[2, 5] = -3e38
        x[3, 7], x[3, 30], x[3, 2] = inf, inf, 3.0
        x[4, 11], x[4, 12] = 1.0, nan
        x[5, 1], x[5, 2] = 3.4e38, -3.4e38
        x[6, 3], x[6, 4], x[6, 9] = 0.0, 1e-40, -1e-40
        for rules in ({}, {"top_k": [2] * 7}, {"top_p": [0.9] * 7}, {"top_k": [50] * 7, "top_p": [0.99] * 7, "min_p": [0.01] * 7}):
            tokens, logprobs, kept = run(cuda_lib, x, {"u": [0.6] * 7, **rules})
            assert tokens[:2] == [-1, -1] and kept[:2] == [0, 0] and logprobs[:2] == [-inf, -inf]
            assert tokens[2] == 5 and logprobs[2] == 0.0 and kept[2] == 1
            assert tokens[3] == 30 and tokens[4] == 11 and tokens[5] == 1 and kept[4] == 1
            assert abs(logprobs[3] + math.log(2)) < 1e-6
    tokens, logprobs, kept = run(cuda_lib, torch.zeros((3, 0), device="cuda"), {"u": [0.5] * 3})
    assert tokens == [-1] * 3 and kept == [0] * 3


def test_random_numbers_at_the_ends(cuda_lib):
    x = torch.full((8, 3000), -math.inf, device="cuda")
    x[:, 10], x[:, 20], x[:, 2900], x[:, 2950] = -200.0, 1.0, 1.0, -150.0
    u = [0.0, -1.0, 0.49999, 0.50001, 0.99999994, 1.0, 2.0, math.nan]
    tokens, _, kept = run(cuda_lib, x, {"u": u})
    assert tokens == [20, 20, 20, 2900, 2900, 2900, 2900, 20] and kept == [4] * 8


def test_rules_at_their_ends(cuda_lib):
    x = logits_of("f32", 9, 2000, 7)
    best = x.argmax(-1).tolist()
    for rules in ({"top_p": [0.0] * 9}, {"top_p": [-1.0] * 9}, {"min_p": [1.0] * 9}, {"min_p": [5.0] * 9}, {"top_k": [1] * 9}, {"top_p": [1e-30] * 9},
                  {"temperature": [1e-30] * 9}):
        tokens, logprobs, kept = run(cuda_lib, x, {"u": [0.7] * 9, **rules})
        assert tokens == best and logprobs == [0.0] * 9, rules
        assert kept == ([2000] * 9 if "temperature" in rules else [1] * 9)
    nan = math.nan
    free = run(cuda_lib, x, {"u": [0.7] * 9})
    for rules in ({"top_p": [nan] * 9}, {"top_p": [1.0] * 9}, {"min_p": [nan] * 9}, {"min_p": [-1.0] * 9}, {"top_k": [-(1 << 31)] * 9},
                  {"top_k": [(1 << 31) - 1] * 9}, {"temperature": [1.0] * 9}):
        assert run(cuda_lib, x, {"u": [0.7] * 9, **rules}) == free
    tokens, logprobs, kept = run(cuda_lib, x, {"u": [0.7001] * 9, "temperature": [math.inf] * 9})
    assert tokens == [1400] * 9 and abs(logprobs[0] + math.log(2000)) < 1e-6


def test_optional_outputs_and_batches(cuda_lib):
    """A row's token does not depend on its batch; logprobs and kept may be left out; replayed from a graph."""
    n, vocab = 300, 20011
    x = logits_of("bf16", n, vocab, 2)
    rules = rules_of(n, "tkpm", 3, vocab)
    whole = check(cuda_lib, x, rules)
    for r in (0, 77, 299):
        one = run(cuda_lib, x[r:r + 1], {k: [v[r]] for k, v in rules.items()})
        assert [o[0] for o in one] == [w[r] for w in whole]
    t = {k: vec(rules[k], torch.int32 if k == "top_k" else torch.float32) for k in NAMES}
    how = _lib.Sampling(*(t[k].data_ptr() for k in NAMES))
    tokens = torch.zeros(n, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for _ in range(2):
            assert cuda_lib.dn_sample(2, x.data_ptr(), vocab, n, vocab, how, tokens.data_ptr(), None, None, _lib.DN_FLAG_PDL,
                                      stream()) == 0
    for _ in range(3):
        tokens.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert tokens.tolist() == whole[0]


def test_two_streams_at_once(cuda_lib):
    x, y = logits_of("f32", 40, 151936, 2), logits_of("f16", 64, 50257, 3)
    rx, ry = rules_of(40, "tkp", 3, 151936), rules_of(64, "tpm", 4, 50257)
    want_x, want_y = run(cuda_lib, x, rx), run(cuda_lib, y, ry)
    outs = []
    for z, r, s in ((x, rx, torch.cuda.Stream()), (y, ry, torch.cuda.Stream())):
        t = {k: vec(r.get(k), torch.int32 if k == "top_k" else torch.float32) for k in NAMES}
        how = _lib.Sampling(*(None if t[k] is None else t[k].data_ptr() for k in NAMES))
        tokens = torch.zeros(z.shape[0], dtype=torch.int32, device="cuda")
        s.wait_stream(torch.cuda.current_stream())
        outs.append((z, how, t, tokens, s))
    for _ in range(10):
        for z, how, _, tokens, s in outs:
            assert cuda_lib.dn_sample(0 if z.dtype == torch.float32 else 1, z.data_ptr(), z.shape[1], z.shape[0], z.shape[1], how,
                                      tokens.data_ptr(), None, None, 0, s.cuda_stream) == 0
    torch.cuda.synchronize()
    assert outs[0][3].tolist() == want_x[0] and outs[1][3].tolist() == want_y[0]


def test_shares(cuda_lib):
    """Evenly spread random numbers choose each kept token as often as its share, to within one."""
    x = torch.tensor([[0.3, -1.0, 2.0, 0.0, 1.1, -3.0]], device="cuda").expand(4096, 6).contiguous()
    u = [(i + 0.5) / 4096 for i in range(4096)]
    tokens, _, kept = run(cuda_lib, x, {"u": u, "top_k": [4] * 4096, "temperature": [0.8] * 4096})
    w = np.exp(np.array([0.3, -1.0, 2.0, 0.0, 1.1, -3.0], dtype=np.float32).astype(np.float64) / float(np.float32(0.8)))
    w[[1, 5]] = 0
    for v in range(6):
        assert abs(tokens.count(v) - 4096 * w[v] / w.sum()) <= 1
    assert tokens == sorted(tokens) and kept == [4] * 4096


@pytest.mark.parametrize("kind,vocab", [("f32", 4097), ("f16", 50257), ("bf16", 4100), ("f32", 151937)])
def test_cuts_of_many_tokens_repeat(cuda_lib, kind, vocab):
    """top_k over what the lists hold, with top_p's border on top: rows whose last tokens are few lanes' alone, the same
    every time."""
    n = 8
    x = logits_of(kind, n, vocab, 7)
    for k in (800, 1600, 3000):
        for p in (0.5, 0.99):
            rules = {"u": [0.3] * n, "top_k": [k] * n, "top_p": [p] * n}
            first = check(cuda_lib, x, rules)
            for _ in range(4):
                assert run(cuda_lib, x, rules) == first


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("which", ["", "k", "p", "m", "kp", "tkpm", "pm"])
@pytest.mark.parametrize("vocab,offset,pad", [(1, 0, 0), (70, 1, 0), (4097, 0, 1), (30011, 3, 2)])
def test_many_rows(cuda_lib, kind, which, vocab, offset, pad):
    """Rows enough for a block each, those on both sides of that number alike."""
    n = 60
    x = logits_of(kind, n, vocab, vocab, offset=offset, pad=pad)
    rules = rules_of(n, which, vocab, vocab)
    whole = check(cuda_lib, x, rules)
    few = run(cuda_lib, x[:40], {k: v[:40] for k, v in rules.items()})
    assert [o[:40] for o in whole] == list(few)


@pytest.mark.parametrize("n", [5, 55])
def test_ties_at_every_cut(cuda_lib, n):
    """Equal logits at top_k's border and at top_p's, in the lists and over the row, the two at the same logit."""
    g = torch.Generator(device="cuda").manual_seed(n)
    rng = random.Random(n)
    for vocab, levels in ((300, 5), (20000, 40), (20000, 4000)):
        x = torch.randint(0, levels, (n, vocab), generator=g, device="cuda").float().mul_(8.0 / levels)
        for k in (3, 17, 100, 900, 2500):
            rules = {"u": [0.001 + 0.998 * rng.random() for _ in range(n)], "top_k": [min(k, vocab - 1)] * n,
                     "top_p": [rng.choice([0.3111, 0.5123, 0.9017, 0.9917]) for _ in range(n)]}
            check(cuda_lib, x, rules)
            check(cuda_lib, x, {"u": rules["u"], "top_k": rules["top_k"]})
        check(cuda_lib, x, {"u": rules["u"], "top_p": rules["top_p"]})


@pytest.mark.parametrize("n", [3, 60])
def test_masks_of_finite_numbers(cuda_lib, n):
    """Masked logits of the type's lowest value, or of a large negative one, among which a cut may fall."""
    for kind in TYPES:
        for low in (-1e4, torch.finfo(TYPES[kind][0]).min):
            x = logits_of(kind, n, 9001, 5)
            few = torch.rand(x.shape, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda") < 0.002
            x.copy_(torch.where(few, x, torch.full_like(x, low)))
            for which in ("k", "p", "kp", "m", ""):
                check(cuda_lib, x, rules_of(n, which, 3, 9001))


@pytest.mark.parametrize("n", [4, 64])
def test_logits_and_temperatures_of_every_size(cuda_lib, n):
    """Spreads from a billionth to a billion, temperatures that make weights steep or level."""
    for spread, offset in ((1e-9, 0.0), (1e-3, 5.0), (50.0, 0.0), (1e9, 0.0), (1e30, 0.0), (1.0, 1e6)):
        x = logits_of("f32", n, 5003, 11, spread=spread) + offset
        for t in (1e-3, 1.0, 1e4, 1e20):
            for which in ("", "k", "p", "m", "kp"):
                rules = {**rules_of(n, which, 13, 5003), "temperature": [t] * n}
                check(cuda_lib, x, rules, some=True)  # where all weights are equal, borders lie on round numbers
