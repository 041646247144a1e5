"""examples/batched_decode.py over an 8-bit cache: append, attention, residual
norm, rules and drawn tokens together. A request of a batch gets the logits, and
with its own random numbers the tokens, that it gets alone; the cache holds what
the prompt's keys and values were, to their rounding."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def inputs(prefix, requests, vocab):
    gen = torch.Generator(device="cuda").manual_seed(prefix)
    return (torch.randint(0, vocab, (prefix,), device="cuda", generator=gen, dtype=torch.int32),
            torch.randint(0, vocab, (requests,), device="cuda", generator=gen, dtype=torch.int32))


@pytest.mark.parametrize("prefix,requests", [(64, 3), (203, 5), (600, 40)])
def test_batch_matches_one_request_alone(cuda_lib, prefix, requests):
    import batched_decode as ex
    vocab, steps = 4099, 4
    prompt, first = inputs(prefix, requests, vocab)
    together = ex.Model(2, vocab, requests, prefix, steps + 1, seed=7, cache="q8")
    said, seen = ex.decode(together, prompt, first, steps, choose=ex.Chooser(requests, 0.8, top_k=50, top_p=0.95))
    alone = ex.Model(2, vocab, 1, prefix, steps + 1, seed=7, cache="q8")
    for r in (0, requests - 1):
        forced = [t[r:r + 1] for t in said]
        _, single = ex.decode(alone, prompt, first[r:r + 1], steps, forced=forced)
        for a, b in zip(seen, single):
            x, y = a[r].double(), b[0].double()
            assert torch.equal(torch.isinf(x), torch.isinf(y))
            assert torch.isinf(x).sum() == 3  # the banned tokens
            ok = torch.isfinite(x)
            # Two layers of products on activations rounded to 8 bits a block and of
            # rows kept in 8 bits: a rounding that falls the other way is 2^-8 of a
            # value's block or row maximum.
            assert (x[ok] - y[ok]).norm() <= 0.02 * y[ok].norm()
        # Equal logits and numbers give equal tokens: the batch's own rows, chosen one at a time.
        one = ex.Chooser(1, 0.8, top_k=50, top_p=0.95, seed=r)
        assert [int(one(logits[r:r + 1].clone())) for logits in seen] == [int(t[r]) for t in said]
    assert cuda_lib.dn_device_status(1) == 0


def test_tokens_are_kept_ones(cuda_lib):
    """Every drawn token is among the rules' likeliest of its logits, and none is a banned one."""
    import batched_decode as ex
    vocab, steps, requests = 4099, 6, 17
    prompt, first = inputs(90, requests, vocab)
    model = ex.Model(1, vocab, requests, 90, steps + 1, seed=3, cache="q8")
    said, seen = ex.decode(model, prompt, first, steps, choose=ex.Chooser(requests, 1.0, top_k=8))
    for tokens, logits in zip(said, seen):
        floor = logits.topk(8, dim=-1).values[:, -1]
        assert (logits.gather(1, tokens.long()[:, None])[:, 0] >= floor).all()
    greedy, seen = ex.decode(model, prompt, first, steps, choose=ex.Chooser(requests, 0.0))
    for tokens, logits in zip(greedy, seen):
        assert torch.equal(tokens.long(), logits.argmax(-1)) or torch.equal(
            logits.gather(1, tokens.long()[:, None])[:, 0], logits.amax(-1))
    assert cuda_lib.dn_device_status(1) == 0


def test_cache_holds_the_prompt(cuda_lib):
    """The first layer's rows, read back, are what the 16-bit model's cache holds, to both roundings."""
    import batched_decode as ex
    vocab, prefix = 1000, 75
    prompt, _ = inputs(prefix, 1, vocab)
    models = [ex.Model(1, vocab, 1, prefix, 2, seed=5, cache=kind) for kind in ("bf16", "q8")]
    for model in models:
        model.prompt(prompt)
    wide, narrow = (model.layers[0] for model in models)
    seq, first, pos = ex.ints([1] * prefix), ex.ints([0] * prefix), torch.arange(prefix, dtype=torch.int32, device="cuda")
    row = ex.KV_HEADS * ex.HEAD_DIM
    k, v = (torch.empty((prefix, row), device="cuda") for _ in range(2))
    assert cuda_lib.dn_paged_q8_read(narrow.cache, 0, seq.data_ptr(), pos.data_ptr(), k.data_ptr(), row, v.data_ptr(), row,
                                     prefix, 0, ex.stream()) == 0
    torch.cuda.synchronize()
    # A request finds the same rows through its own table.
    mine = [torch.empty_like(k) for _ in range(2)]
    assert cuda_lib.dn_paged_q8_read(narrow.cache, 0, first.data_ptr(), pos.data_ptr(), mine[0].data_ptr(), row,
                                     mine[1].data_ptr(), row, prefix, 0, ex.stream()) == 0
    torch.cuda.synchronize()
    assert torch.equal(mine[0], k) and torch.equal(mine[1], v)
    pages = models[0].table[1].long()[:-(-prefix // ex.PAGE)]
    for got, pool in ((k, wide.keys), (v, wide.values)):
        got = got.view(prefix, ex.KV_HEADS, ex.HEAD_DIM)
        want = pool[pages].permute(0, 2, 1, 3).reshape(-1, ex.KV_HEADS, ex.HEAD_DIM)[:prefix].float()
        # Half a step of 8 bits (amax / 254, the amax of the unrounded row: 2^-8 more) and half a
        # step of bf16 (2^-8 of a value); 2^-10 for the norms' and the rotation's f32.
        bound = want.abs().amax(-1, keepdim=True) / 254 * (1 + 2 ** -7) + want.abs() * (2 ** -8 + 2 ** -10) + 1e-7
        assert ((got - want).abs() <= bound).all()
    assert cuda_lib.dn_device_status(1) == 0
