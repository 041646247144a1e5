"""More of the batched decode step's operators, as cases that can be timed and checked.

A paged cache in 8 bits (dn_paged_q8_append quantizes a step's keys and values
as it writes them, dn_paged_q8_read reads them back, dn_paged_q8_attention
attends over them), what stands between two blocks of a layer
(dn_residual_norm: the norm after a block, its gate and residual scale, the
residual add and the norm before the next block) and the choice of a token from
the logits (dn_sample: temperature, top-k, top-p and min-p from given random
numbers).

listed() gives the cases, draw() more of the same ranges, prepare() a case's
inputs, run() one pass (the framework's kernels where `own` is true, else the
plain form in elementary torch operations), exact() the same in 64 bits.
"""
import math
import random

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZES = {"f32": 4, "f16": 2, "bf16": 2}
CODES = {"f32": 0, "f16": 1, "bf16": 2}  # DN_F32, DN_F16, DN_BF16


# ------------------------------------------------------------------ the cases


def listed():
    return [
        # One user, a short chat so far. Latency.
        attend("attend one short", "bf16", 1, 150, 1, 16, 8, 128, 16),
        # One user behind a book: few rows, the cache's length is all there is to split.
        attend("attend one long", "bf16", 1, 131072, 1, 28, 4, 128, 64),
        # A chat server's step on the 16-head, 8-kv-head, 128-wide model of the decode benchmarks.
        attend("attend chat 32", "bf16", 32, 4096, 1, 16, 8, 128, 16),
        # Draft tokens being verified: up to 5 queries a sequence, 96-wide heads, 3 heads a group.
        attend("attend drafts 24", "f16", 24, 3000, 5, 12, 4, 96, 32),
        # An f32 step with a window, a page size that is no power of two, wide heads.
        attend("attend f32 window", "f32", 9, 2500, 1, 8, 2, 256, 24, window=1000),
        # The largest: many long sequences, grouped heads.
        attend("attend many 64", "bf16", 64, 16384, 1, 32, 8, 128, 64),
        # A decode step's q, k, v (one fused f32 product) with the head norms; its rows read back.
        append("append decode 32", "f32", "bf16", 32, 16, 8, 128, 128, 16, True, 1),
        # A long prompt's keys and values, and its rows read back for the prompt's own attention.
        append("append prompt 16384", "bf16", "bf16", 16384, 32, 8, 128, 128, 64, False, 0),
        # A decode step of the 2048-wide model, norms on both sides of the block, in f32.
        join("join decode 16", "f32", "f32", 16, 2048, True, "none", 1.0),
        # A long prompt in 16 bits over an f32 residual stream, with a gate for each channel.
        join("join prompt 16384", "bf16", "f32", 16384, 4096, True, "one", 0.5),
        # One user's token out of the whole vocabulary of the decode benchmarks.
        sample("sample one", "f32", 1, 151936, "kp", 0.0),
        # A large batch in which every request has rules of its own, some behind a grammar mask.
        sample("sample batch 256", "f32", 256, 151936, "mixed", 0.1),
    ]


def attend(name, kind, seqs, length, q, heads, kv_heads, hd, page, window=0):
    return {"name": name, "op": "attend", "kind": kind, "seqs": seqs, "length": length, "q": q, "heads": heads,
            "kv_heads": kv_heads, "hd": hd, "page": page, "window": window}


def append(name, kind, out, n, heads, kv_heads, hd, rot, page, norm, pad):
    return {"name": name, "op": "append", "kind": kind, "out": out, "n": n, "heads": heads, "kv_heads": kv_heads,
            "hd": hd, "rot": rot, "page": page, "norm": norm, "pad": pad}


def join(name, kind, stream, n, cols, post, gate, scale):
    return {"name": name, "op": "join", "kind": kind, "stream": stream, "n": n, "cols": cols, "post": post, "gate": gate,
            "scale": scale}


def sample(name, kind, n, vocab, rules, masked):
    return {"name": name, "op": "sample", "kind": kind, "n": n, "vocab": vocab, "rules": rules, "masked": masked}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


HEADS = [(16, 8, 128), (32, 8, 128), (12, 4, 96), (8, 8, 64), (28, 4, 128), (8, 2, 256), (9, 3, 64), (16, 1, 128)]


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "join", "sample", "sample"])
    kind = rng.choice(["bf16", "f16", "bf16", "f32"])
    if op == "attend":
        heads, kv_heads, hd = rng.choice(HEADS)
        seqs = _log(rng, 1, 64)
        length = _log(rng, 1, 131072 if seqs == 1 else max(64, 1000000 // seqs * 1024 // (kv_heads * hd) // (4 if kind == "f32" else 1)))
        length = min(length, 131072)
        q = 1 if rng.random() < 0.7 else rng.randint(2, 8)
        window = _log(rng, 1, length) if rng.random() < 0.2 else 0
        c = attend("", kind, seqs, max(length, q), q, heads, kv_heads, hd, rng.choice([16, 32, 64, 16, 24, 7]), window)
    elif op == "append":
        heads, kv_heads, hd = rng.choice(HEADS)
        n = _log(rng, 1, 16384 if kind != "f32" and heads * hd <= 4096 else 8000)
        c = append("", kind, rng.choice(["bf16", "f16"]), n, heads, kv_heads, hd, rng.choice([hd, hd, hd // 2]),
                   rng.choice([16, 32, 64, 24]), rng.random() < 0.5, rng.randint(0, 1))
    elif op == "join":
        cols = rng.choice([1024, 2048, 4096, 5120, 8192, _log(rng, 64, 8192), 2 * _log(rng, 32, 4096)])
        n = _log(rng, 1, max(1, min(20000, (16384 if kind != "f32" else 8000) * 4096 // cols)))
        c = join("", kind, rng.choice(["f32", kind]), n, cols, rng.random() < 0.6, rng.choice(["none", "one", "each"]),
                 rng.choice([1.0, 0.5, 0.22]))
    else:
        c = sample("", kind, _log(rng, 1, 250), rng.choice([32000, 50257, 65536, 151936, _log(rng, 100, 150000)]),
                   rng.choice(["mixed", "mixed", "kp", "p", "k", "min", "all", "greedy"]), round(rng.random() / 2, 2))
    del c["name"]
    return c


def work(case):
    """The bytes and operations that one pass cannot do without, at the mean of the drawn lengths."""
    c = case
    if c["op"] == "attend":
        b = SIZES[c["kind"]]
        mean = c["length"] if c["seqs"] == 1 else (c["length"] + c["q"]) / 2
        tokens = c["seqs"] * (1 + c["q"]) / 2
        seen = min(mean, c["window"] + (c["q"] - 1) / 2 if c["window"] else mean)
        return {"bytes": c["seqs"] * seen * c["kv_heads"] * 2 * (c["hd"] + 4) + 2 * tokens * c["heads"] * c["hd"] * b,
                "flops": 4 * tokens * c["heads"] * c["hd"] * seen}
    if c["op"] == "append":
        b, o = SIZES[c["kind"]], SIZES[c["out"]]
        kv = c["n"] * 2 * c["kv_heads"]
        # In and q out, the rows into the cache, the rows out of it, the rows read back.
        return {"bytes": c["n"] * c["heads"] * c["hd"] * (b + o) + kv * (c["hd"] * (b + o) + 2 * (c["hd"] + 4)) + c["n"] * (8 + 4 * c["rot"]),
                "flops": 6 * c["n"] * (c["heads"] + 2 * c["kv_heads"]) * c["hd"]}
    if c["op"] == "join":
        b, s = SIZES[c["kind"]], SIZES[c["stream"]]
        each = c["n"] * c["cols"]
        return {"bytes": each * (2 * b + 2 * s + (b if c["gate"] == "each" else 0)) + c["cols"] * 8, "flops": 10 * each}
    return {"bytes": c["n"] * c["vocab"] * SIZES[c["kind"]] + c["n"] * 28, "flops": 4 * c["n"] * c["vocab"]}


# ----------------------------------------------------------------- the inputs


def prepare(case, seed):
    return {"attend": _prepare_attend, "append": _prepare_append, "join": _prepare_join,
            "sample": _prepare_sample}[case["op"]](dict(case), seed)


def _rngs(seed):
    return random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)


def _form(case):
    """What sets the outputs' shapes (a batch's queries, a pool's pages) goes by the case alone."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _quantized(x):
    """Rows of f32 as 8 bits with a scale, as the cache holds them."""
    scale = x.abs().amax(-1) / 127
    q = x / torch.where(scale > 0, scale, 1.0)[..., None]
    return (q.abs() + 0.5).floor().clamp_(max=127).mul_(q.sign()).to(torch.int8), scale


def _pool(pages, c, g):
    """A pool of quantized rows of different sizes; made in parts, which f32 takes four times the room of."""
    shape = (pages, c["kv_heads"], c["page"], c["hd"])
    rows, scales = torch.empty(shape, dtype=torch.int8, device="cuda"), torch.empty(shape[:3], device="cuda")
    step = max(1, (1 << 28) // (shape[1] * shape[2] * shape[3]))
    for at in range(0, pages, step):
        part = torch.randn((min(step, pages - at),) + shape[1:], generator=g, device="cuda")
        part *= torch.randn(part.shape[:3], generator=g, device="cuda").mul_(0.3).exp_()[..., None]
        rows[at:at + step], scales[at:at + step] = _quantized(part)
    return rows, scales


def _table(lengths, page, rng):
    need = [-(-n // page) for n in lengths]
    width, pages = max(1, max(need)), sum(need) + 1
    order = list(range(pages))
    rng.shuffle(order)
    table, at = [], 0
    for k in need:
        table.append(order[at:at + k] + [-1] * (width - k))
        at += k
    return table, pages


def _prepare_attend(c, seed):
    rng, g = _rngs(seed)
    dt, seqs = TYPES[c["kind"]], c["seqs"]
    form = _form(c)
    q_lens = [form.randint(1, c["q"]) for _ in range(seqs)]
    if seqs == 1:
        lengths = [c["length"]]
    else:
        lengths = [rng.randint(max(1, q), max(c["length"], q)) for q in q_lens]
    if seqs >= 7:
        lengths[rng.randrange(seqs)] = 0  # a slot of the batch that no request holds
    table, pages = _table(lengths, c["page"], rng)
    starts = [0]
    for q in q_lens:
        starts.append(starts[-1] + q)
    n = starts[-1]
    keys, key_scales = _pool(pages, c, g)
    values, value_scales = _pool(pages, c, g)
    return {
        "case": c, "keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales,
        "q": torch.randn((n, c["heads"], c["hd"]), generator=g, device="cuda").mul_(1.5).to(dt),
        "table": _ints(table), "lengths": _ints(lengths), "starts": _ints(starts),
        "out": torch.zeros((n, c["heads"], c["hd"]), device="cuda", dtype=dt),
        "n": n, "scale": c["hd"] ** -0.5,
    }


def _rope_table(rows, rot):
    at = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None]
    angle = at * (1e6 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot))[None]
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _prepare_append(c, seed):
    rng, g = _rngs(seed)
    dt, page, n = TYPES[c["kind"]], c["page"], c["n"]
    # Sequences of one to a few thousand new tokens, each behind some tokens that it has.
    form = _form(c)
    seq, pos, lengths = [], [], []
    while len(seq) < n:
        new = min(n - len(seq), form.choice([1, 1, 1, form.randint(1, 9)]) if n < 1000 else form.randint(500, 4000))
        first = form.randint(0, 2 * page if n < 1000 else 100)
        seq += [len(lengths)] * new
        pos += range(first, first + new)
        lengths.append(first + new)
    if c["pad"]:
        for i in range(0, n, 9):
            seq[i] = -1  # a padding token of the batch
    # One page more than the table names: the plain form writes the padding tokens there.
    table, pages = _table(lengths, page, rng)
    keys, key_scales = _pool(pages + 1, c, g)
    values, value_scales = _pool(pages + 1, c, g)
    odt, rows = TYPES[c["out"]], (n, c["kv_heads"], c["hd"])
    return {
        "case": c, "keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales,
        "qkv": torch.randn((n, (c["heads"] + 2 * c["kv_heads"]) * c["hd"]), generator=g, device="cuda").mul_(2).to(dt),
        "q_out": torch.zeros((n, c["heads"], c["hd"]), device="cuda", dtype=odt),
        "k_out": torch.zeros(rows, device="cuda", dtype=odt), "v_out": torch.zeros(rows, device="cuda", dtype=odt),
        "table": _ints(table), "seq": _ints(seq), "pos": _ints(pos), "rope": _rope_table(max(lengths), c["rot"]),
        "q_norm": 1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda"),
        "k_norm": 1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda"),
        "pages": pages,
    }


def _prepare_join(c, seed):
    _, g = _rngs(seed)
    n, cols, dt, sdt = c["n"], c["cols"], TYPES[c["kind"]], TYPES[c["stream"]]
    make = lambda *shape: torch.randn(shape, generator=g, device="cuda")  # noqa: E731
    return {
        "case": c, "y": make(n, cols).mul_(3).to(dt), "x": make(n, cols).mul_(2).to(sdt),
        "gate": make(n if c["gate"] == "each" else 1, cols).to(dt),
        "post": 1 + 0.2 * make(cols), "pre": 1 + 0.2 * make(cols),
        "x_out": torch.zeros((n, cols), device="cuda", dtype=sdt), "h": torch.zeros((n, cols), device="cuda", dtype=dt),
    }


def _prepare_sample(c, seed):
    rng, g = _rngs(seed)
    n, vocab = c["n"], c["vocab"]
    x = torch.randn((n, vocab), generator=g, device="cuda").mul_(2.2)
    # A step's likely tokens stand out of the rest, more in some rows than in others.
    likely = torch.randint(0, vocab, (n, 64), generator=g, device="cuda")
    height = 4 + 8 * torch.rand((n, 1), generator=g, device="cuda") + torch.randn((n, 64), generator=g, device="cuda").mul_(2)
    x.scatter_(1, likely, height)
    for r in range(n):
        if rng.random() < c["masked"]:  # a grammar allows few tokens or most of them
            few = rng.random() ** 4
            x[r].masked_fill_(torch.rand(vocab, generator=g, device="cuda") >= max(few, 2 / vocab), -math.inf)
    rules = [c["rules"] if c["rules"] != "mixed" else rng.choice(["kp", "p", "k", "min", "all", "greedy"]) for _ in range(n)]
    with_k, with_p = ("kp", "k"), ("kp", "p")
    return {
        "case": c, "logits": x.to(TYPES[c["kind"]]),
        "temperature": _ints([0.0 if r == "greedy" else rng.choice([0.6, 0.7, 0.8, 1.0, 1.2]) for r in rules], torch.float32),
        "top_k": _ints([rng.choice([20, 40, 50, 200, 1000]) if r in with_k else 0 for r in rules]),
        "top_p": _ints([rng.choice([0.5, 0.8, 0.9, 0.95, 0.99]) if r in with_p else 1.0 for r in rules], torch.float32),
        "min_p": _ints([rng.choice([0.02, 0.05, 0.1]) if r == "min" else 0.0 for r in rules], torch.float32),
        "uniform": torch.rand(n, generator=g, device="cuda"),
        "tokens": torch.zeros(n, dtype=torch.int32, device="cuda"), "kept": torch.zeros(n, dtype=torch.int32, device="cuda"),
        "logprobs": torch.zeros(n, device="cuda"),
    }


# ------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "join": _own_join, "sample": _own_sample}[op](state)
    return {"attend": _plain_attend, "append": _plain_append, "join": _plain_join, "sample": _plain_sample}[op](state)


def _kept(state, make):
    """The descriptors that a user's program makes once for its cache or its batch and passes to every call."""
    if "handle" not in state:
        state["handle"] = make(state)
    return state["handle"]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _done(rc, what):
    if rc != 0:
        raise RuntimeError("%s: %d" % (what, rc))


def _cache(s):
    from dianoia_b200 import _lib
    c, (pages, kvh, page, hd) = s["case"], s["keys"].shape
    return _lib.PagedQ8Cache(*(s[k].data_ptr() for k in ("keys", "values", "key_scales", "value_scales", "table")),
                             s.get("pages", pages), page, kvh, hd, s["table"].shape[0], s["table"].shape[1],
                             kvh * page * hd, kvh * page)


def _attend_kept(s):
    from dianoia_b200 import _lib
    c, cache = s["case"], _cache(s)
    need = _lib.lib().dn_paged_q8_attention_workspace(cache, c["heads"], s["n"], c["length"])
    return _lib.lib(), cache, torch.empty(need, dtype=torch.uint8, device="cuda")


def _own_attend(s):
    L, cache, ws = _kept(s, _attend_kept)
    c = s["case"]
    row = c["heads"] * c["hd"]
    _done(L.dn_paged_q8_attention(cache, CODES[c["kind"]], s["q"].data_ptr(), row, s["starts"].data_ptr(), s["lengths"].data_ptr(),
                                  c["length"], s["scale"], c["window"], s["out"].data_ptr(), row, c["heads"], s["n"],
                                  ws.data_ptr(), ws.numel(), 0, _stream()), "dn_paged_q8_attention")
    return {"out": s["out"]}


def _append_kept(s):
    from dianoia_b200 import _lib
    return _lib.lib(), _cache(s)


def _own_append(s):
    L, cache = _kept(s, _append_kept)
    c, qkv = s["case"], s["qkv"]
    q, size = qkv.data_ptr(), qkv.element_size()
    k = q + c["heads"] * c["hd"] * size
    v = k + c["kv_heads"] * c["hd"] * size
    out, row = CODES[c["out"]], c["kv_heads"] * c["hd"]
    _done(L.dn_paged_q8_append(cache, CODES[c["kind"]], q, qkv.shape[1], k, qkv.shape[1], v, qkv.shape[1], s["seq"].data_ptr(),
                               s["pos"].data_ptr(), s["rope"].data_ptr(), s["rope"].shape[0], c["rot"],
                               s["q_norm"].data_ptr() if c["norm"] else None, s["k_norm"].data_ptr() if c["norm"] else None, 1e-6,
                               out, s["q_out"].data_ptr(), c["heads"] * c["hd"], c["heads"], c["n"], 0, _stream()),
          "dn_paged_q8_append")
    _done(L.dn_paged_q8_read(cache, out, s["seq"].data_ptr(), s["pos"].data_ptr(), s["k_out"].data_ptr(), row,
                             s["v_out"].data_ptr(), row, c["n"], 0, _stream()), "dn_paged_q8_read")
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _own_join(s):
    from dianoia_b200 import _lib
    c, cols = s["case"], s["case"]["cols"]
    gate = s["gate"].data_ptr() if c["gate"] != "none" else None
    _done(_lib.lib().dn_residual_norm(CODES[c["kind"]], s["y"].data_ptr(), cols, s["post"].data_ptr() if c["post"] else None,
                                      gate, cols if c["gate"] == "each" else 0, c["scale"], CODES[c["stream"]],
                                      s["x"].data_ptr(), cols, s["x_out"].data_ptr(), cols, s["pre"].data_ptr(), 1e-6,
                                      s["h"].data_ptr(), cols, None, 0, c["n"], cols, 0, _stream()), "dn_residual_norm")
    return {"x": s["x_out"], "h": s["h"]}


def _sample_kept(s):
    from dianoia_b200 import _lib
    return _lib.lib(), _lib.Sampling(*(s[k].data_ptr() for k in ("temperature", "top_k", "top_p", "min_p", "uniform")))


def _own_sample(s):
    L, how = _kept(s, _sample_kept)
    c = s["case"]
    _done(L.dn_sample(CODES[c["kind"]], s["logits"].data_ptr(), c["vocab"], c["n"], c["vocab"], how, s["tokens"].data_ptr(),
                      s["logprobs"].data_ptr(), s["kept"].data_ptr(), 0, _stream()), "dn_sample")
    return {"tokens": s["tokens"], "logprobs": s["logprobs"], "kept": s["kept"]}


# ----------------------------------------------- the plain forms, in 32 bits


def _plain_attend(s):
    c = s["case"]
    seqs, heads, kvh, hd = c["seqs"], c["heads"], c["kv_heads"], c["hd"]
    group, n, q_max = heads // kvh, s["n"], c["q"]
    lengths, starts = s["lengths"].long(), s["starts"].long()
    q_lens = starts[1:] - starts[:-1]
    seq = torch.repeat_interleave(torch.arange(seqs, device="cuda"), q_lens, output_size=n)
    nth = torch.arange(n, device="cuda") - starts[seq]
    # Queries padded to the longest sequence's: [seqs, kv_heads, group * q_max, hd], and their positions (-1: none).
    q = torch.zeros((seqs, q_max, heads, hd), device="cuda")
    q[seq, nth] = s["q"].float()
    rows = q.view(seqs, q_max, kvh, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, kvh, group * q_max, hd)
    at = torch.full((seqs, q_max), -1, device="cuda", dtype=torch.int64)
    at[seq, nth] = (lengths - q_lens)[seq] + nth
    at = at[:, None, None, :, None].expand(seqs, 1, group, q_max, 1).reshape(seqs, 1, group * q_max, 1)
    low = at - c["window"] + 1 if c["window"] else torch.zeros_like(at)
    ids = s["table"].long().clamp(min=0)
    k = (s["keys"][ids] * s["key_scales"][ids][..., None]).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, hd)
    score = (rows @ k.transpose(2, 3)) * s["scale"]
    del k
    p = torch.arange(score.shape[-1], device="cuda")
    score = torch.where((p <= at) & (p >= low), score, -math.inf)
    top = score.amax(-1, keepdim=True)
    e = (score - torch.where(top == -math.inf, 0.0, top)).exp()
    total = e.sum(-1, keepdim=True)
    v = (s["values"][ids] * s["value_scales"][ids][..., None]).permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, hd)
    out = torch.where(total > 0, (e @ v) / torch.where(total > 0, total, 1.0), 0.0)
    out = out.view(seqs, kvh, group, q_max, hd).permute(0, 3, 1, 2, 4).reshape(seqs, q_max, heads, hd)
    return {"out": out[seq, nth].to(s["q"].dtype)}


def _plain_rotate(x, w, table, rot):
    """[n, heads, hd] in 32 bits: the head norm (w may be None), then the half-split rotation of the first `rot` values."""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w
    cos, sin = table[:, None, :rot // 2], table[:, None, rot // 2:]
    a, b = x[..., :rot // 2], x[..., rot // 2:rot]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., rot:]], -1)


def _plain_append(s):
    c = s["case"]
    heads, kvh, hd, page, n = c["heads"], c["kv_heads"], c["hd"], c["page"], c["n"]
    x = s["qkv"].float().view(n, heads + 2 * kvh, hd)
    seq, pos = s["seq"].long(), s["pos"].long()
    held = seq >= 0
    ids, slot = torch.where(held, s["table"].long()[seq.clamp(min=0), pos // page], s["pages"]), pos % page
    table = s["rope"][pos]
    q = _plain_rotate(x[:, :heads], s["q_norm"] if c["norm"] else None, table, c["rot"])
    k = _plain_rotate(x[:, heads:heads + kvh], s["k_norm"] if c["norm"] else None, table, c["rot"])
    s["keys"][ids, :, slot], s["key_scales"][ids, :, slot] = _quantized(k)
    s["values"][ids, :, slot], s["value_scales"][ids, :, slot] = _quantized(x[:, heads + kvh:])
    back = lambda rows, scales: torch.where(held[:, None, None], rows[ids, :, slot] * scales[ids, :, slot][..., None], 0.0)  # noqa: E731
    s["q_out"].copy_(torch.where(held[:, None, None], q, 0.0))
    s["k_out"].copy_(back(s["keys"], s["key_scales"]))
    s["v_out"].copy_(back(s["values"], s["value_scales"]))
    return {"q": s["q_out"], "k": s["k_out"], "v": s["v_out"]}


def _plain_norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w


def _plain_join(s):
    c = s["case"]
    b = s["y"].float()
    if c["post"]:
        b = _plain_norm(b, s["post"])
    if c["gate"] != "none":
        b = b * s["gate"].float()
    x = s["x"].float() + b * c["scale"]
    return {"x": x.to(s["x"].dtype), "h": _plain_norm(x, s["pre"]).to(s["y"].dtype)}


def _plain_sample(s):
    """Weights and their sums in 64 bits: a token's border in the cumulative sum may lie next to the random number."""
    x = s["logits"].float()
    x = torch.where(x.isnan(), -math.inf, x)
    top = x.amax(-1, keepdim=True)
    t = s["temperature"].double()[:, None]
    greedy = ~(t > 0)
    w = torch.where(x == top, 1.0, torch.where(greedy, 0.0, torch.exp((x - top).double() / torch.where(greedy, 1.0, t))))
    _, order = torch.sort(x, dim=-1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(x.shape[1], device="cuda")
    k, p = s["top_k"][:, None], s["top_p"].double()[:, None]
    keep = (x.gather(1, order) > -math.inf) & ((rank < k) | (k <= 0)) & ((rank < 1) | ~greedy)
    ws = torch.where(keep, ws, 0.0)
    before = ws.cumsum(-1)
    total = before[:, -1:].clone()
    before = torch.cat([torch.zeros_like(total), before[:, :-1]], -1)
    keep &= (before < p * total) | (rank == 0) | ~(p < 1)
    keep &= (ws >= s["min_p"].double()[:, None]) | (rank == 0)
    kept = torch.zeros_like(keep).scatter_(1, order, keep)
    mass = torch.where(kept, w, 0.0)
    run_to = mass.cumsum(-1)
    total = run_to[:, -1:].clone()
    token = (run_to <= s["uniform"].double()[:, None] * total).sum(-1, keepdim=True).clamp_(max=x.shape[1] - 1)
    none = total == 0  # a mask that allows no token: -1
    logprob = torch.where(none, 0.0, mass.gather(1, token) / torch.where(none, 1.0, total)).log()
    return {"tokens": torch.where(none, -1, token)[:, 0].int(), "logprobs": logprob[:, 0].float(), "kept": kept.sum(-1).int()}


# ------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "join": _exact_join, "sample": _exact_sample}[case["op"]](s)


def _exact_attend(s):
    """Row by row of the batch: the keys a query sees, their softmax, their values' mean."""
    c = s["case"]
    page, group = c["page"], c["heads"] // c["kv_heads"]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    out = torch.zeros(s["out"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["seqs"]):
        if lengths[b] == 0:
            continue
        where = torch.arange(lengths[b], device="cuda")
        block = s["table"][b].long()[where // page]
        for kv in range(c["kv_heads"]):
            heads = slice(kv * group, (kv + 1) * group)
            k = s["keys"][block, kv, where % page].double() * s["key_scales"][block, kv, where % page].double()[:, None]
            v = s["values"][block, kv, where % page].double() * s["value_scales"][block, kv, where % page].double()[:, None]
            for t in range(starts[b], starts[b + 1]):
                p = lengths[b] - (starts[b + 1] - t)
                lo = max(0, p - c["window"] + 1) if c["window"] else 0
                e = s["q"][t, heads].double() @ k[lo:p + 1].T / math.sqrt(c["hd"])
                out[t, heads] = torch.softmax(e, -1) @ v[lo:p + 1]
    return {"out": out}


def _exact_append(s):
    """What is read back, whole steps of its row's scale and all."""
    c = s["case"]
    heads, kvh, hd, rot, n = c["heads"], c["kv_heads"], c["hd"], c["rot"], c["n"]
    x = s["qkv"].double().reshape(n, heads + 2 * kvh, hd)
    turn = torch.complex(s["rope"][:, :rot // 2].double(), s["rope"][:, rot // 2:].double())[s["pos"].long()][:, None]

    def rotated(y, w):
        if c["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * w.double()
        z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
        return torch.cat([z.real, z.imag, y[..., rot:]], -1)

    def stepped(y):
        step = y.abs().max(-1, keepdim=True).values / 127
        return torch.sign(y) * torch.floor(y.abs() / step + 0.5) * step

    none = (s["seq"] < 0).nonzero()[:, 0]
    out = {"q": rotated(x[:, :heads], s["q_norm"]), "k": stepped(rotated(x[:, heads:heads + kvh], s["k_norm"])),
           "v": stepped(x[:, heads + kvh:].clone())}
    for rows in out.values():
        rows[none] = 0
    return out


def _exact_join(s):
    c, cols = s["case"], s["case"]["cols"]
    b = s["y"].double()
    if c["post"]:
        b = s["post"].double() * b / (b.pow(2).sum(-1, keepdim=True) / cols + 1e-6).sqrt()
    g = s["gate"].double() if c["gate"] != "none" else 1.0
    x = s["x"].double() + c["scale"] * (g * b)
    return {"x": x, "h": s["pre"].double() * x / (x.pow(2).sum(-1, keepdim=True) / cols + 1e-6).sqrt()}


def _exact_sample(s):
    """Row by row: the tokens sorted, cut, put back in their own order and run through."""
    n = s["case"]["n"]
    logits = s["logits"].double().cpu().numpy()
    rules = [s[k].double().tolist() for k in ("temperature", "top_k", "top_p", "min_p", "uniform")]
    import numpy as np
    tokens, logprobs, counts = [], [], []
    for r in range(n):
        t, k, p, least, u = (v[r] for v in rules)
        x = logits[r]
        order = np.argsort(-x, kind="stable")
        order = order[:np.count_nonzero(x > -math.inf)]
        if not len(order):
            tokens, logprobs, counts = tokens + [-1], logprobs + [-math.inf], counts + [0]
            continue
        if t <= 0:
            order = order[:1]
        w = np.exp((x[order] - x[order[0]]) / (t if t > 0 else 1.0))
        if k > 0:
            order, w = order[:int(k)], w[:int(k)]
        if p < 1:
            m = min(len(w), int(np.searchsorted(np.cumsum(w), p * np.sum(w), side="left")) + 1)
            order, w = order[:m], w[:m]
        m = max(1, np.count_nonzero(w >= least))
        order, w = order[:m], w[:m]
        by_index = np.argsort(order)
        order, w = order[by_index], w[by_index]
        total = np.cumsum(w)
        at = min(len(w) - 1, int(np.searchsorted(total, u * total[-1], side="right")))
        tokens.append(int(order[at]))
        logprobs.append(math.log(w[at] / total[-1]))
        counts.append(m)
    return {"tokens": _ints(tokens, torch.int64), "logprobs": torch.tensor(logprobs, dtype=torch.float64), "kept": _ints(counts, torch.int64)}
