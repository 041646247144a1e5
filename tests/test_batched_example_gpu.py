"""examples/batched_decode.py: the batched step's operators together. A request
of a batch that shares its prompt gets the logits that it gets alone, the rules
hold on them, and a prompt that ends inside a page is shared all the same."""
import os
import sys

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


@pytest.mark.parametrize("prefix,requests", [(64, 3), (203, 5), (600, 40)])
def test_batch_matches_one_request_alone(cuda_lib, prefix, requests):
    import batched_decode as ex
    vocab, steps = 4099, 4
    gen = torch.Generator(device="cuda").manual_seed(prefix)
    prompt = torch.randint(0, vocab, (prefix,), device="cuda", generator=gen, dtype=torch.int32)
    first = torch.randint(0, vocab, (requests,), device="cuda", generator=gen, dtype=torch.int32)
    together = ex.Model(2, vocab, requests, prefix, steps + 1, seed=7)
    said, seen = ex.decode(together, prompt, first, steps)
    alone = ex.Model(2, vocab, 1, prefix, steps + 1, seed=7)
    for r in (0, requests - 1):
        forced = [t[r:r + 1] for t in said]
        _, single = ex.decode(alone, prompt, first[r:r + 1], steps, forced=forced)
        for a, b in zip(seen, single):
            x, y = a[r].double(), b[0].double()
            assert torch.equal(torch.isinf(x), torch.isinf(y))
            assert torch.isinf(x).sum() == 3  # the banned tokens
            ok = torch.isfinite(x)
            # Two layers of products on activations rounded to 8 bits a block and a
            # 16-bit cache: a rounding that falls the other way is 2^-8 of a value.
            assert (x[ok] - y[ok]).norm() <= 0.02 * y[ok].norm()
    assert cuda_lib.dn_device_status(1) == 0
