"""Drawn tokens beside a largest logit next to 0, as log-probabilities have it: the differences of logits are exact there too.

The bound is that of any row: a border between two tokens lies within 2^-28 + vocab 2^-41 of its place in 64 bits (four roundings to 24 bits
of a term of 0.011 at most, a table entry and a product rounded to 2^-32 each, a series and a fraction off by 2^-32 and 2^-31; then each
weight to a multiple of 2^-40), and u times the total is rounded down to 2^-40. Log-probabilities are off by 2^-28 + vocab 2^-41 + 2^-28 and
their rounding to fp32."""
import pytest
import torch

from ml_framework_b200.ops import native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("top", [0.0, 1e-5, -3e-6, 2.0 ** -40, -2.0 ** -60, 1e-4, 4.4e-4, 4.5e-4, 1e-3, 0.01])
@pytest.mark.parametrize("which", ["", "p", "k", "m"])
def test_borders(dtype, top, which):
    rows, vocab = 600, 1000
    g = torch.Generator(device="cuda").manual_seed(3)
    t = torch.exp(4 * torch.rand(rows, device="cuda", generator=g) - 2)
    x = -(5.5 + 3.5 * torch.rand(rows, vocab, device="cuda", generator=g)) * t[:, None]
    x[:, 400] = top * t
    x = x.to(dtype)
    w = torch.exp((x.double() - x.double().amax(1, keepdim=True)) / t.double()[:, None])
    p = torch.full((rows,), 0.9999999, device="cuda") if "p" in which else None          # keeps every token: all weights lie above 1e-7 of the total
    k = torch.full((rows,), vocab - 1, dtype=torch.int32, device="cuda") if "k" in which else None
    m = torch.full((rows,), 1e-30, device="cuda") if "m" in which else None
    if k is not None:                                            # without the last of the order: the highest index of the smallest
        last = vocab - 1 - (w == w.amin(1, keepdim=True)).flip(1).int().argmax(1)
        w[torch.arange(rows, device="cuda"), last] = 0.0
    run = torch.cumsum(w, 1) / w.sum(1, keepdim=True)
    at = torch.randint(50, 950, (rows, 1), device="cuda", generator=g)
    u = run.gather(1, at)[:, 0].float()                          # next to a border between two tokens
    got, lp = native.sample_rows(x, vocab, u, t, k, p, m, want_logprobs=True)
    above = run.gather(1, got[:, None])[:, 0]
    weight = w.gather(1, got[:, None])[:, 0]
    below = above - weight / w.sum(1)
    off = 2.0 ** -28 + vocab * 2.0 ** -41 + 2.0 ** -40
    assert (weight > 0).all()
    assert (below - off <= u.double()).all() and (u.double() < above + off).all(), float(torch.maximum(below - u.double(), u.double() - above).max() * 2.0 ** 28)
    want = torch.log(weight / w.sum(1))
    assert ((lp.double() - want).abs() <= 2.0 ** -24 * want.abs() + 2 * off).all()
