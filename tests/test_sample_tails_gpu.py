"""Drawn tokens out of a flat tail far below the largest logit: what the borders between tokens may be off by.

The bound: a weight is its exponential, off by 2^-28 of it (four roundings to 24 bits of a term of 0.011 at most, 2^-28.5; a table entry
and a product rounded to 2^-32 each, a series off by 2^-32, a fraction off by 2^-31), rounded to a multiple of 2^-40 of the largest
weight: off by 2^-28 w + 2^-41. Over a row of V logits a prefix and its rest are off by no more than 2^-28 of each + V 2^-41, and the
total W is 1 at least: a border c / W moves by 2^-28 + V 2^-41 at most. u times the total is rounded down to 2^-40."""
import pytest
import torch

from ml_framework_b200.ops import native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [4097, 128256, 1 << 20])
@pytest.mark.parametrize("depth", [20.0, 24.0, 27.0, 28.0, 28.5, 40.0])
def test_flat_tails(dtype, vocab, depth):
    """One large logit and all others `depth` temperatures below it, u within 2^-20 of 1: the token's borders in 64 bits hold u but for
    the bound."""
    u = 1.0 - torch.tensor([1.0, 2.0, 3.0, 5.0, 9.0, 13.0, 16.0, 0.0], device="cuda") * 2.0 ** -24
    u[7] = 0.5
    for t in (0.5, 1.0, 2.0):
        x = torch.full((8, vocab), -depth * t, device="cuda").to(dtype)
        x[:, 3] = 0.0
        got = native.sample_rows(x, vocab, u, torch.full((8,), t, device="cuda"))
        w = torch.exp(x[0].double() / t)
        run = torch.cumsum(w, 0)
        below, above = (run - w)[got] / run[-1], run[got] / run[-1]
        off = 2.0 ** -28 + vocab * 2.0 ** -41 + 2.0 ** -40
        assert (below - off <= u.double()).all() and (u.double() < above + off).all()
