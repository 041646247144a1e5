"""A batched decode step: many requests behind one shared prompt.

A random-init Q8_0 model of the 1.7B decode shapes (fewer layers by default)
serves `--requests` requests that share a prompt of `--prefix` tokens. The
prompt is run once and its keys and values stay in pages that every request's
cache names; then each step, for all requests together and in each layer:

    RMSNorm, q/k/v product            dn_rms_norm, dn_linear
    cache append, head norms, RoPE    dn_paged_append
    attention, prompt read once       dn_paged_attention
    o, gate/up, SwiGLU, down          dn_linear, dn_swiglu

and at its end the lm_head and the rules on its logits (penalties for what a
request has said so far, a bias, a mask) with dn_logits_apply, before the
greedy choice. Needs a B200 and torch:

    python examples/batched_decode.py --requests 32 --prefix 1024 --steps 16
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from dianoia_b200 import _lib  # noqa: E402

HIDDEN, HEADS, KV_HEADS, HEAD_DIM, INTER = 2048, 16, 8, 128, 6144
PAGE = 16
EPS = 1e-6


def ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


class Linear:
    """A Q8_0 matrix [rows, cols], quantized on the device from random weights."""

    def __init__(self, rows, cols, gen):
        w = torch.randn((rows, cols), device="cuda", generator=gen) * cols ** -0.5
        self.rows, self.cols = rows, cols
        self.qs = torch.empty(rows * cols, dtype=torch.int8, device="cuda")
        self.scales = torch.empty(rows * cols // 32, device="cuda")
        _lib.check(_lib.lib().dn_quantize_q8(w.data_ptr(), self.qs.data_ptr(), self.scales.data_ptr(), rows, cols, stream()))
        torch.cuda.current_stream().synchronize()  # w goes

    def __call__(self, x):
        n = x.shape[0]
        y = torch.empty((n, self.rows), device="cuda")
        xq = torch.empty(n * self.cols, dtype=torch.int8, device="cuda")
        xsc = torch.empty(n * self.cols // 32, device="cuda")
        _lib.check(_lib.lib().dn_linear(_lib.DN_Q8, self.qs.data_ptr(), self.scales.data_ptr(), x.data_ptr(), xq.data_ptr(),
                                        xsc.data_ptr(), y.data_ptr(), self.rows, self.cols, n, self.rows, 1,
                                        _lib.DN_PATH_AUTO, 0, stream()))
        return y


def stream():
    return torch.cuda.current_stream().cuda_stream


def norm(x, w):
    out = torch.empty_like(x)
    _lib.check(_lib.lib().dn_rms_norm(x.data_ptr(), w.data_ptr(), out.data_ptr(), None, 0, x.shape[0], x.shape[1], EPS, 0, 0,
                                      stream()))
    return out


class Layer:
    def __init__(self, pages, table, gen):
        weight = lambda n: 1 + 0.1 * torch.randn(n, device="cuda", generator=gen)
        self.qkv = Linear((HEADS + 2 * KV_HEADS) * HEAD_DIM, HIDDEN, gen)
        self.o = Linear(HIDDEN, HEADS * HEAD_DIM, gen)
        self.gate, self.up = Linear(INTER, HIDDEN, gen), Linear(INTER, HIDDEN, gen)
        self.down = Linear(HIDDEN, INTER, gen)
        self.norm1, self.norm2, self.q_norm, self.k_norm = weight(HIDDEN), weight(HIDDEN), weight(HEAD_DIM), weight(HEAD_DIM)
        shape = (pages, KV_HEADS, PAGE, HEAD_DIM)
        self.keys, self.values = (torch.zeros(shape, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        self.cache = _lib.PagedCache(self.keys.data_ptr(), self.values.data_ptr(), table.data_ptr(), _lib.DN_BF16, pages, PAGE,
                                     KV_HEADS, HEAD_DIM, table.shape[0], table.shape[1], KV_HEADS * PAGE * HEAD_DIM)


class Model:
    """`requests` sequences; row `requests` of the page table is the prompt's own."""

    def __init__(self, layers, vocab, requests, prefix, room, seed=0):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.requests, self.prefix, self.vocab = requests, prefix, vocab
        shared, each = -(-prefix // PAGE), -(-room // PAGE) + 1
        self.width = shared + each
        # A request's table: the prompt's whole pages, then its own (its own
        # from the page that the prompt ends in, which it may not write into).
        whole = prefix // PAGE
        rows, at = [], shared
        for _ in range(requests):
            own = list(range(at, at + self.width - whole))
            rows.append(list(range(whole)) + own)
            at += len(own)
        rows.append((list(range(shared)) + [-1] * self.width)[:self.width])
        self.table = ints(rows)
        self.pages = ints(list(range(max(1, shared))))
        self.max_length = self.width * PAGE
        angle = torch.arange(self.max_length, device="cuda")[:, None] * 1e6 ** (
            -torch.arange(HEAD_DIM // 2, device="cuda") * 2 / HEAD_DIM)
        self.rope = torch.cat([angle.cos(), angle.sin()], 1).float().contiguous()
        self.embed = torch.randn((vocab, HIDDEN), device="cuda", generator=gen)
        self.layers = [Layer(at, self.table, gen) for _ in range(layers)]
        self.final, self.head = 1 + 0.1 * torch.randn(HIDDEN, device="cuda", generator=gen), Linear(vocab, HIDDEN, gen)

    def forward(self, tokens, seq, pos, starts, lengths, prefix):
        """Hidden states of `tokens`, token i of sequence seq[i] at pos[i]; the cache gains their keys and values."""
        L, n = _lib.lib(), tokens.numel()
        x = self.embed[tokens.long()]
        q = torch.empty((n, HEADS * HEAD_DIM), dtype=torch.bfloat16, device="cuda")
        out = torch.empty_like(q)
        need = L.dn_paged_attention_workspace(self.layers[0].cache, HEADS, n, prefix, self.max_length)
        work = torch.empty(need, dtype=torch.uint8, device="cuda")
        for layer in self.layers:
            qkv = layer.qkv(norm(x, layer.norm1))
            k = qkv.data_ptr() + HEADS * HEAD_DIM * 4
            row = qkv.shape[1]
            _lib.check(L.dn_paged_append(layer.cache, _lib.DN_F32, qkv.data_ptr(), row, k, row, k + KV_HEADS * HEAD_DIM * 4, row,
                                         seq.data_ptr(), pos.data_ptr(), self.rope.data_ptr(), self.rope.shape[0], HEAD_DIM,
                                         layer.q_norm.data_ptr(), layer.k_norm.data_ptr(), EPS, q.data_ptr(), q.shape[1], HEADS, n,
                                         0, stream()))
            _lib.check(L.dn_paged_attention(layer.cache, q.data_ptr(), q.shape[1], starts.data_ptr(), lengths.data_ptr(),
                                            self.pages.data_ptr(), prefix, self.max_length, HEAD_DIM ** -0.5, 0, out.data_ptr(),
                                            out.shape[1], HEADS, n, work.data_ptr(), need, 0, stream()))
            x = x + layer.o(out.float())
            h = norm(x, layer.norm2)
            g, u = layer.gate(h), layer.up(h)
            _lib.check(L.dn_swiglu(g.data_ptr(), u.data_ptr(), None, g.numel(), 0, stream()))
            x = x + layer.down(g)
        return x

    def prompt(self, tokens):
        """Runs the shared prompt once, as the table's last sequence."""
        n, r = tokens.numel(), self.requests
        self.forward(tokens, ints([r] * n), torch.arange(n, dtype=torch.int32, device="cuda"), ints([0] * (r + 1) + [n]),
                     ints([0] * r + [n]), 0)

    def step(self, tokens, done):
        """Logits of one token for each request, `done` tokens of its own behind it."""
        r = self.requests
        seq, pos = torch.arange(r, dtype=torch.int32, device="cuda"), ints([self.prefix + done] * r)
        x = self.forward(tokens, seq, pos, ints(list(range(r + 1)) + [r]), ints([self.prefix + done + 1] * r + [0]), self.prefix)
        return self.head(norm(x, self.final))


def rules_of(history, vocab, banned):
    """The penalties, biases and the mask of a step; the tensors are kept with the descriptor."""
    n = len(history)
    keep = {
        "tokens": ints([t for h in history for t in h] or [0]),
        "history": ints([sum(len(h) for h in history[:i]) for i in range(n + 1)], torch.int64),
        "repetition": torch.full((n,), 1.1, device="cuda"), "frequency": torch.full((n,), 0.2, device="cuda"),
        "presence": torch.full((n,), 0.1, device="cuda"),
        "bias_tokens": ints([0] * n), "bias": torch.full((n,), -5.0, device="cuda"),
        "bias_start": torch.arange(n + 1, dtype=torch.int64, device="cuda"),
    }
    mask = torch.full((1, (vocab + 31) // 32), -1, dtype=torch.int32, device="cuda")
    for t in banned:
        mask[0, t // 32] &= ~(1 << (t % 32)) if t % 32 < 31 else 0x7fffffff
    keep["mask"], keep["mask_row"] = mask, ints([0] * n)
    rules = _lib.LogitRules(mask_rows=1, mask_stride=mask.shape[1], **{k: v.data_ptr() for k, v in keep.items()})
    return rules, keep


def decode(model, prompt, first, steps, banned=(1, 2, 3), forced=None):
    """Greedy tokens [steps][requests] and each step's ruled logits; with `forced`, those tokens are fed instead."""
    model.prompt(prompt)
    tokens, history, said, seen = first, [[t] for t in first.tolist()], [], []
    for i in range(steps):
        logits = model.step(tokens, i)
        rules, keep = rules_of(history, model.vocab, banned)
        _lib.check(_lib.lib().dn_logits_apply(_lib.DN_F32, logits.data_ptr(), model.vocab, logits.data_ptr(), model.vocab,
                                              model.requests, model.vocab, rules, 0, stream()))
        seen.append(logits)
        tokens = (logits.argmax(-1) if forced is None else forced[i]).int()
        said.append(tokens)
        for h, t in zip(history, tokens.tolist()):
            h.append(t)
    return said, seen


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--requests", type=int, default=32)
    ap.add_argument("--prefix", type=int, default=1024)
    ap.add_argument("--steps", type=int, default=16)
    ap.add_argument("--layers", type=int, default=4)
    ap.add_argument("--vocab", type=int, default=151936)
    a = ap.parse_args()
    model = Model(a.layers, a.vocab, a.requests, a.prefix, a.steps + 1)
    gen = torch.Generator(device="cuda").manual_seed(1)
    prompt = torch.randint(0, a.vocab, (a.prefix,), device="cuda", generator=gen, dtype=torch.int32)
    first = torch.randint(0, a.vocab, (a.requests,), device="cuda", generator=gen, dtype=torch.int32)
    decode(model, prompt, first, 2)
    begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
    begin.record()
    said, _ = decode(model, prompt, first, a.steps)
    end.record()
    torch.cuda.synchronize()
    ms = begin.elapsed_time(end)
    print("request 0: %s" % [int(t[0]) for t in said])
    print("%d requests, %d-token prompt, %d steps, %d layers: %.1f ms with the prompt, %.0f tokens/s"
          % (a.requests, a.prefix, a.steps, a.layers, ms, a.requests * a.steps / ms * 1e3))


if __name__ == "__main__":
    main()
