"""The batched decode step's operators, as cases that can be timed and checked.

Three operators that serve many requests at once next to the quantized
products: dn_paged_append (a step's keys and values rotated and written into a
paged cache, its queries rotated on the way), dn_paged_attention (attention
over that cache for a batch whose requests share a long prefix, which is read
once for all of them) and dn_logits_apply (the penalties for repeated tokens,
the biases and the grammar masks on the logits the step ends with).

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
        # One user at a prompt: two short sequences behind a small system prompt. Latency.
        attend("attend two short", "bf16", 2, 64, 12, 1, 16, 8, 128, 16),
        # A chat server's step on the 16-head, 8-kv-head, 128-wide model of the decode benchmarks.
        attend("attend chat 32", "bf16", 32, 1024, 700, 1, 16, 8, 128, 16),
        # The f32 cache that the single-sequence layer keeps, at an odd batch, with a window.
        attend("attend f32 window", "f32", 7, 512, 333, 1, 16, 8, 128, 16, window=600),
        # Draft tokens being verified: up to 7 queries a sequence, 96-wide heads, 3 heads a group.
        attend("attend drafts 24", "f16", 24, 2048, 500, 7, 12, 4, 96, 32),
        # The largest: many requests on one long document, grouped heads.
        attend("attend document 192", "bf16", 192, 8192, 1024, 1, 32, 8, 128, 64),
        # A decode step's q, k, v (one fused f32 product) into a bf16 cache, with the head norms.
        append("append decode 16", "f32", "bf16", 16, 16, 8, 128, 128, 16, True, 0),
        # A ragged batch with padding tokens, 64-wide heads of which half is rotated, f16.
        append("append ragged 203", "f16", "f16", 203, 12, 4, 64, 32, 32, False, 1),
        # A long prompt's keys and values.
        append("append prompt 16384", "bf16", "bf16", 16384, 32, 8, 128, 128, 64, False, 0),
        # One request: the whole vocabulary of the decode benchmarks, 500 tokens so far, a grammar.
        shape("logits one", "f32", 1, 151936, 500, 20, 1.0),
        # An odd vocabulary in 16 bits: rows that start at any alignment.
        shape("logits odd 33", "bf16", 33, 50257, 1200, 50, 0.5),
        # A chat server's step: long histories, some rows under a grammar.
        shape("logits chat 64", "f32", 64, 151936, 4000, 300, 0.3),
        # A large batch, few rules.
        shape("logits batch 256", "f32", 256, 151936, 800, 10, 0.1),
    ]


def attend(name, kind, seqs, prefix, own_max, q, heads, kv_heads, hd, page, window=0):
    return {"name": name, "op": "attend", "kind": kind, "seqs": seqs, "prefix": prefix, "own_max": own_max, "q": q,
            "heads": heads, "kv_heads": kv_heads, "hd": hd, "page": page, "window": window}


def append(name, kind, cache, n, heads, kv_heads, hd, rot, page, norm, pad):
    return {"name": name, "op": "append", "kind": kind, "cache": cache, "n": n, "heads": heads, "kv_heads": kv_heads,
            "hd": hd, "rot": rot, "page": page, "norm": norm, "pad": pad}


def shape(name, kind, n, vocab, history, biases, masked):
    return {"name": name, "op": "logits", "kind": kind, "n": n, "vocab": vocab, "history": history, "biases": biases,
            "masked": masked}


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "append", "logits"])
    if op == "attend":
        kind = rng.choice(["bf16", "f16", "bf16", "f16", "f32"])
        heads, kv_heads, hd = rng.choice([(16, 8, 128), (32, 8, 128), (12, 4, 96), (8, 8, 64), (28, 4, 128), (8, 2, 256), (9, 3, 64)])
        page = rng.choice([16, 32, 64])
        seqs = _log(rng, 1, 32 if kind == "f32" else 160)  # f32: the single-user side of the range
        prefix = page * _log(rng, 1, 8192 // page) if rng.random() < 0.9 else 0
        own_max = _log(rng, 1, 1024)
        q = 1 if rng.random() < 0.7 else rng.randint(2, 8)
        if q > 1:
            seqs = min(seqs, 40)
        window = _log(rng, 16, prefix + own_max) if rng.random() < 0.2 and prefix + own_max > 16 else 0
        c = attend("", kind, seqs, prefix, max(own_max, q), q, heads, kv_heads, hd, page, window)
    elif op == "append":
        kind = rng.choice(["f32", "bf16", "f16"])
        cache = rng.choice(["bf16", "f16", "f32"]) if kind == "f32" else kind
        heads, kv_heads, hd = rng.choice([(16, 8, 128), (32, 8, 128), (12, 4, 96), (8, 8, 64), (28, 4, 128), (8, 2, 256), (9, 3, 64)])
        n = _log(rng, 1, 16384 if kind != "f32" and heads * hd <= 4096 else 8000)
        rot = rng.choice([hd, hd, hd // 2])
        c = append("", kind, cache, n, heads, kv_heads, hd, rot, rng.choice([16, 32, 64]), rng.random() < 0.5, rng.randint(0, 1))
    else:
        kind = rng.choice(["f32", "f32", "bf16", "f16"])
        c = shape("", kind, _log(rng, 1, 250), rng.choice([32000, 50257, 65536, 151936, _log(rng, 1000, 150000)]),
                  _log(rng, 1, 4000), _log(rng, 1, 300), round(rng.random(), 2))
    del c["name"]
    return c


def work(case):
    """The bytes and operations that one pass cannot do without, at the mean of the drawn lengths."""
    if case["op"] == "attend":
        b = SIZES[case["kind"]]
        mean = (case["own_max"] + case["q"]) / 2
        tokens = case["seqs"] * (1 + case["q"]) / 2
        row = case["kv_heads"] * case["hd"] * b * 2
        seen = min(case["prefix"] + mean, case["window"] or 1 << 60)
        # Positions of the prefix that some row's window still reaches.
        shared = case["prefix"] if not case["window"] else max(0, min(case["prefix"], case["window"]))
        private = min(mean, case["window"] or 1 << 60)
        return {"bytes": shared * row + case["seqs"] * private * row + 2 * tokens * case["heads"] * case["hd"] * b,
                "flops": 4 * tokens * case["heads"] * case["hd"] * seen}
    if case["op"] == "append":
        b, c = SIZES[case["kind"]], SIZES[case["cache"]]
        values = case["n"] * (case["heads"] + 2 * case["kv_heads"]) * case["hd"]
        return {"bytes": values * (b + c) + case["n"] * (8 + 4 * case["rot"]), "flops": 6 * values}
    b = SIZES[case["kind"]]
    return {"bytes": case["n"] * (2 * b * case["vocab"] + 4 * case["history"] * 0.75 + 8 * case["biases"] * 0.5)
            + case["n"] * case["masked"] * case["vocab"] / 8, "flops": 6 * case["n"] * case["vocab"]}


# ----------------------------------------------------------------- the inputs


def prepare(case, seed):
    return {"attend": _prepare_attend, "append": _prepare_append, "logits": _prepare_logits}[case["op"]](dict(case), seed)


def _rngs(seed):
    return random.Random(seed), torch.Generator(device="cuda").manual_seed(seed)


def _form(case):
    """What sets the outputs' shapes (a batch's queries, a pool's pages) goes by the case alone."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _prepare_attend(c, seed):
    rng, g = _rngs(seed)
    dt, page, seqs, prefix = TYPES[c["kind"]], c["page"], c["seqs"], c["prefix"]
    form = _form(c)
    q_lens = [form.randint(1, c["q"]) for _ in range(seqs)]
    lengths = [prefix + rng.randint(max(q, 1), max(c["own_max"], q)) for q in q_lens]
    if seqs >= 7:
        lengths[rng.randrange(seqs)] = 0  # a slot of the batch that no request holds
    shared = prefix // page
    width = -(-(prefix + c["own_max"]) // page)
    need = [max(0, -(-n // page) - shared) for n in lengths]
    pages = shared + sum(need) + 3
    order = list(range(pages))
    rng.shuffle(order)
    table, at = [], shared
    for n, k in zip(lengths, need):
        table.append((order[:shared] if n else [-1] * shared) + order[at:at + k] + [-1] * (width - shared - k))
        at += k
    starts = [0]
    for q in q_lens:
        starts.append(starts[-1] + q)
    n = starts[-1]
    pool = (pages, c["kv_heads"], page, c["hd"])
    state = {
        "case": c,
        "keys": torch.randn(pool, generator=g, device="cuda", dtype=torch.float32).to(dt),
        "values": torch.randn(pool, generator=g, device="cuda", dtype=torch.float32).to(dt),
        "q": torch.randn((n, c["heads"], c["hd"]), generator=g, device="cuda", dtype=torch.float32).mul_(1.5).to(dt),
        "table": _ints(table), "prefix_pages": _ints(order[:max(shared, 1)]), "lengths": _ints(lengths), "starts": _ints(starts),
        "out": torch.zeros((n, c["heads"], c["hd"]), device="cuda", dtype=dt),
        "n": n, "max_length": prefix + c["own_max"], "scale": c["hd"] ** -0.5,
    }
    return state


def _rope_table(rows, rot):
    at = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None]
    angle = at * (1e6 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2 / rot))[None]
    return torch.cat([angle.cos(), angle.sin()], 1).float()


def _prepare_append(c, seed):
    rng, g = _rngs(seed)
    dt, page, n = TYPES[c["kind"]], c["page"], c["n"]
    # Sequences of one to a few thousand new tokens, each behind some tokens that it has.
    form = _form(c)
    seq, pos, width, b = [], [], 1, 0
    while len(seq) < n:
        new = min(n - len(seq), form.choice([1, 1, 1, form.randint(1, 9)]) if n < 1000 else form.randint(500, 4000))
        first = form.randint(0, 2 * page if n < 1000 else 100)
        seq += [b] * new
        pos += range(first, first + new)
        width = max(width, -(-(first + new) // page))
        b += 1
    held = [0] * b  # pages of each sequence
    for i, p in zip(seq, pos):
        held[i] = max(held[i], p // page + 1)
    if c["pad"]:
        for i in range(0, n, 9):
            seq[i] = -1  # a padding token of the batch
    pages = sum(held)
    order = list(range(pages))
    rng.shuffle(order)
    table, at = [], 0
    for k in held:
        table.append(order[at:at + k] + [-1] * (width - k))
        at += k
    # One page more than the table names: the plain form writes the padding tokens there.
    pool = (pages + 1, c["kv_heads"], page, c["hd"])
    cdt = TYPES[c["cache"]]
    return {
        "case": c,
        "qkv": torch.randn((n, (c["heads"] + 2 * c["kv_heads"]) * c["hd"]), generator=g, device="cuda").mul_(2).to(dt),
        "keys": torch.randn(pool, generator=g, device="cuda").to(cdt),
        "values": torch.randn(pool, generator=g, device="cuda").to(cdt),
        "q_out": torch.zeros((n, c["heads"], c["hd"]), device="cuda", dtype=cdt),
        "table": _ints(table), "seq": _ints(seq), "pos": _ints(pos), "rope": _rope_table(width * page, c["rot"]),
        "q_norm": 1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda"),
        "k_norm": 1 + 0.2 * torch.randn(c["hd"], generator=g, device="cuda"),
        "pages": pages,
    }


def _prepare_logits(c, seed):
    rng, g = _rngs(seed)
    n, vocab = c["n"], c["vocab"]
    lens = [rng.randint(c["history"] // 2, c["history"]) for _ in range(n)]
    starts = [0]
    for k in lens:
        starts.append(starts[-1] + k)
    # Text repeats itself: tokens fall off like a power of a uniform number.
    u = torch.rand(starts[-1], generator=g, device="cuda")
    tokens = (u.pow(3) * vocab).to(torch.int64).mul_(7919).remainder_(vocab).to(torch.int32)
    bias_lens = [rng.randint(0, min(c["biases"], vocab)) for _ in range(n)]
    bias_starts = [0]
    for k in bias_lens:
        bias_starts.append(bias_starts[-1] + k)
    bias_tokens = [t for k in bias_lens for t in rng.sample(range(vocab), k)] or [0]
    # A third as many grammar states as rows, few or most of the tokens allowed in each.
    states = max(1, n // 3)
    words = -(-vocab // 32)
    bits = torch.rand((states, words * 32), generator=g, device="cuda") < torch.rand((states, 1), generator=g, device="cuda").pow(4)
    mask = (bits.view(states, words, 32).long() << torch.arange(32, device="cuda")).sum(-1)
    mask = torch.where(mask >= 1 << 31, mask - (1 << 32), mask).to(torch.int32)
    return {
        "case": c,
        "logits": torch.randn((n, vocab), generator=g, device="cuda").mul_(4).to(TYPES[c["kind"]]),
        "out": torch.zeros((n, vocab), device="cuda", dtype=TYPES[c["kind"]]),
        "tokens": tokens, "history": _ints(starts, torch.int64), "generated": _ints([rng.randint(0, k) for k in lens]),
        "repetition": _ints([rng.choice([1.0, 1.1, 1.3]) for _ in range(n)], torch.float32),
        "frequency": _ints([rng.choice([0.0, 0.2, 0.5]) for _ in range(n)], torch.float32),
        "presence": _ints([rng.choice([0.0, 0.4, -0.3]) for _ in range(n)], torch.float32),
        "bias_tokens": _ints(bias_tokens), "bias": torch.randn(len(bias_tokens), generator=g, device="cuda") * 5,
        "bias_start": _ints(bias_starts, torch.int64), "mask": mask,
        "mask_row": _ints([rng.randrange(states) if rng.random() < c["masked"] else -1 for _ in range(n)]),
        "total": starts[-1], "total_bias": bias_starts[-1],
    }


# ------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return {"attend": _own_attend, "append": _own_append, "logits": _own_logits}[op](state)
    return {"attend": _plain_attend, "append": _plain_append, "logits": _plain_logits}[op](state)


def _kept(state, make):
    """The descriptors that a user's program makes once for its cache or its batch and passes to every call."""
    if "kept" not in state:
        state["kept"] = make(state)
    return state["kept"]


def _stream():
    return torch.cuda.current_stream().cuda_stream


def _cache(s, pages):
    from dianoia_b200 import _lib
    c = s["case"]
    return _lib.PagedCache(s["keys"].data_ptr(), s["values"].data_ptr(), s["table"].data_ptr(), CODES[c.get("cache", c["kind"])],
                           pages, c["page"], c["kv_heads"], c["hd"], s["table"].shape[0], s["table"].shape[1],
                           c["kv_heads"] * c["page"] * c["hd"])


def _attend_kept(s):
    from dianoia_b200 import _lib
    c, cache = s["case"], _cache(s, s["keys"].shape[0])
    need = _lib.lib().dn_paged_attention_workspace(cache, c["heads"], s["n"], c["prefix"], s["max_length"])
    return _lib.lib(), cache, torch.empty(need, dtype=torch.uint8, device="cuda")


def _own_attend(s):
    L, cache, ws = _kept(s, _attend_kept)
    c = s["case"]
    row = c["heads"] * c["hd"]
    rc = L.dn_paged_attention(cache, s["q"].data_ptr(), row, s["starts"].data_ptr(), s["lengths"].data_ptr(),
                              s["prefix_pages"].data_ptr(), c["prefix"], s["max_length"], s["scale"], c["window"],
                              s["out"].data_ptr(), row, c["heads"], s["n"], ws.data_ptr(), ws.numel(), 0, _stream())
    if rc != 0:
        raise RuntimeError("dn_paged_attention: %d" % rc)
    return {"out": s["out"]}


def _append_kept(s):
    from dianoia_b200 import _lib
    return _lib.lib(), _cache(s, s["pages"])


def _own_append(s):
    L, cache = _kept(s, _append_kept)
    c, qkv = s["case"], s["qkv"]
    q, size = qkv.data_ptr(), qkv.element_size()
    k = q + c["heads"] * c["hd"] * size
    v = k + c["kv_heads"] * c["hd"] * size
    rc = L.dn_paged_append(cache, CODES[c["kind"]], q, qkv.shape[1], k, qkv.shape[1], v, qkv.shape[1], s["seq"].data_ptr(),
                           s["pos"].data_ptr(), s["rope"].data_ptr(), s["rope"].shape[0], c["rot"],
                           s["q_norm"].data_ptr() if c["norm"] else None, s["k_norm"].data_ptr() if c["norm"] else None, 1e-6,
                           s["q_out"].data_ptr(), c["heads"] * c["hd"], c["heads"], c["n"], 0, _stream())
    if rc != 0:
        raise RuntimeError("dn_paged_append: %d" % rc)
    return {"q": s["q_out"], "keys": s["keys"][:s["pages"]], "values": s["values"][:s["pages"]]}


def _logits_kept(s):
    from dianoia_b200 import _lib
    rules = _lib.LogitRules(*(s[k].data_ptr() for k in ("tokens", "history", "generated", "repetition", "frequency", "presence",
                                                         "bias_tokens", "bias", "bias_start", "mask", "mask_row")),
                            s["mask"].shape[0], s["mask"].shape[1])
    return _lib.lib(), rules


def _own_logits(s):
    L, rules = _kept(s, _logits_kept)
    c = s["case"]
    rc = L.dn_logits_apply(CODES[c["kind"]], s["logits"].data_ptr(), c["vocab"], s["out"].data_ptr(), c["vocab"], c["n"],
                           c["vocab"], rules, 0, _stream())
    if rc != 0:
        raise RuntimeError("dn_logits_apply: %d" % rc)
    return {"out": s["out"]}


# ----------------------------------------------- the plain forms, in 32 bits


def _plain_attend(s):
    c = s["case"]
    seqs, heads, kvh, hd, page, prefix = c["seqs"], c["heads"], c["kv_heads"], c["hd"], c["page"], c["prefix"]
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
    # Each sequence's own keys, padded to the longest.
    own_pages = s["table"][:, prefix // page:].long()
    ids = own_pages.clamp(min=0)
    k_own = s["keys"][ids].permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, hd).float()
    v_own = s["values"][ids].permute(0, 2, 1, 3, 4).reshape(seqs, kvh, -1, hd).float()
    p_own = prefix + torch.arange(k_own.shape[2], device="cuda")
    sees_own = (p_own <= at) & (p_own >= low)
    s_own = (rows @ k_own.transpose(2, 3)) * s["scale"]
    s_own = torch.where(sees_own, s_own, -math.inf)
    top = s_own.amax(-1, keepdim=True) if s_own.shape[-1] else torch.full_like(rows[..., :1], -math.inf)
    if prefix:
        all_rows = rows.transpose(0, 1).reshape(kvh, -1, hd)
        k_pre = s["keys"][s["prefix_pages"].long()].transpose(0, 1).reshape(kvh, prefix, hd).float()
        v_pre = s["values"][s["prefix_pages"].long()].transpose(0, 1).reshape(kvh, prefix, hd).float()
        p_pre = torch.arange(prefix, device="cuda")
        s_pre = (all_rows @ k_pre.transpose(1, 2)).mul_(s["scale"]).view(kvh, seqs, group * q_max, prefix).transpose(0, 1)
        s_pre = torch.where((p_pre <= at) & (p_pre >= low), s_pre, -math.inf)
        top = torch.maximum(top, s_pre.amax(-1, keepdim=True))
    top = torch.where(top == -math.inf, 0.0, top)
    e_own = (s_own - top).exp()
    total, out = e_own.sum(-1, keepdim=True), e_own @ v_own
    if prefix:
        e_pre = (s_pre - top).exp()
        total = total + e_pre.sum(-1, keepdim=True)
        out = out + (e_pre.transpose(0, 1).reshape(kvh, -1, prefix) @ v_pre).view(kvh, seqs, group * q_max, hd).transpose(0, 1)
    out = torch.where(total > 0, out / torch.where(total > 0, total, 1.0), 0.0)
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
    ids = torch.where(held, s["table"].long()[seq.clamp(min=0), pos // page], s["pages"])
    table = s["rope"][pos]
    q = _plain_rotate(x[:, :heads], s["q_norm"] if c["norm"] else None, table, c["rot"])
    k = _plain_rotate(x[:, heads:heads + kvh], s["k_norm"] if c["norm"] else None, table, c["rot"])
    s["keys"][ids, :, pos % page] = k.to(s["keys"].dtype)
    s["values"][ids, :, pos % page] = x[:, heads + kvh:].to(s["values"].dtype)
    s["q_out"].copy_(torch.where(held[:, None, None], q, 0.0))
    return {"q": s["q_out"], "keys": s["keys"][:s["pages"]], "values": s["values"][:s["pages"]]}


def _plain_logits(s):
    c = s["case"]
    n, vocab = c["n"], c["vocab"]
    x = s["logits"].float()
    lens = s["history"][1:] - s["history"][:-1]
    row = torch.repeat_interleave(torch.arange(n, device="cuda"), lens, output_size=s["total"])
    nth = torch.arange(s["total"], device="cuda") - s["history"][row]
    made = (nth >= (lens - s["generated"])[row]).float()
    flat = row * vocab + s["tokens"].long()
    seen = torch.zeros(n * vocab, device="cuda").index_fill_(0, flat, 1.0).view(n, vocab) > 0
    count = torch.zeros(n * vocab, device="cuda").index_add_(0, flat, made).view(n, vocab)
    r = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / r, x * r), x)
    x = x - (count * s["frequency"][:, None] + (count > 0).float() * s["presence"][:, None])
    bias_row = torch.repeat_interleave(torch.arange(n, device="cuda"), s["bias_start"][1:] - s["bias_start"][:-1], output_size=s["total_bias"])
    k = s["total_bias"]
    x = x.view(-1).index_add(0, bias_row * vocab + s["bias_tokens"][:k].long(), s["bias"][:k]).view(n, vocab)
    words = s["mask"][s["mask_row"].clamp(min=0).long()]
    bits = (words[:, :, None] >> torch.arange(32, device="cuda", dtype=torch.int32)) & 1
    allowed = (bits.view(n, -1)[:, :vocab] != 0) | (s["mask_row"] < 0)[:, None]
    return {"out": torch.where(allowed, x, -math.inf).to(s["logits"].dtype)}


# ------------------------------------------------ the definition, in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"attend": _exact_attend, "append": _exact_append, "logits": _exact_logits}[case["op"]](s)


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
        k = s["keys"][block, :, where % page].double().repeat_interleave(group, 1)
        v = s["values"][block, :, where % page].double().repeat_interleave(group, 1)
        first = lengths[b] - (starts[b + 1] - starts[b])
        for t in range(starts[b], starts[b + 1]):
            p = first + t - starts[b]
            lo = max(0, p - c["window"] + 1) if c["window"] else 0
            e = torch.einsum("hd,khd->hk", s["q"][t].double(), k[lo:p + 1]) / math.sqrt(c["hd"])
            out[t] = torch.einsum("hk,khd->hd", torch.softmax(e, -1), v[lo:p + 1])
    return {"out": out}


def _exact_append(s):
    c = s["case"]
    heads, kvh, hd, rot, n = c["heads"], c["kv_heads"], c["hd"], c["rot"], c["n"]
    x = s["qkv"].double().reshape(n, heads + 2 * kvh, hd)
    turn = torch.complex(s["rope"][:, :rot // 2].double(), s["rope"][:, rot // 2:].double())[s["pos"].long()][:, None]

    def rotated(y, w):
        if c["norm"]:
            y = y / (y.pow(2).sum(-1, keepdim=True) / hd + 1e-6).sqrt() * w.double()
        z = torch.complex(y[..., :rot // 2].contiguous(), y[..., rot // 2:rot].contiguous()) * turn
        return torch.cat([z.real, z.imag, y[..., rot:]], -1)

    held = (s["seq"] >= 0).nonzero()[:, 0]
    seq, pos = s["seq"][held].long(), s["pos"][held].long()
    block, slot = s["table"].long()[seq, pos // c["page"]], pos % c["page"]
    q = torch.zeros((n, heads, hd), dtype=torch.float64, device="cuda")
    q[held] = rotated(x[:, :heads], s["q_norm"])[held]
    keys, values = s["keys"][:s["pages"]].double(), s["values"][:s["pages"]].double()
    keys[block, :, slot] = rotated(x[:, heads:heads + kvh], s["k_norm"])[held]
    values[block, :, slot] = x[held, heads + kvh:]
    return {"q": q, "keys": keys, "values": values}


def _exact_logits(s):
    c = s["case"]
    n, vocab = c["n"], c["vocab"]
    hist, bias_start = s["history"].tolist(), s["bias_start"].tolist()
    generated, mask_row = s["generated"].tolist(), s["mask_row"].tolist()
    out = torch.empty((n, vocab), dtype=torch.float64, device="cuda")
    which = torch.arange(vocab, device="cuda")
    for r in range(n):
        x = s["logits"][r].double()
        ids = s["tokens"][hist[r]:hist[r + 1]].long()
        seen = torch.bincount(ids, minlength=vocab)
        count = torch.bincount(ids[ids.numel() - generated[r]:], minlength=vocab)
        p = s["repetition"][r].double()
        x[(seen > 0) & (x > 0)] /= p
        x[(seen > 0) & (s["logits"][r] <= 0)] *= p
        x -= s["frequency"][r].double() * count
        x[count > 0] -= s["presence"][r].double()
        a, b = bias_start[r], bias_start[r + 1]
        x[s["bias_tokens"][a:b].long()] += s["bias"][a:b].double()
        if mask_row[r] >= 0:
            word = s["mask"][mask_row[r]].long()[which // 32]
            x[(word >> (which % 32)) % 2 == 0] = -math.inf
        out[r] = x
    return {"out": out}
