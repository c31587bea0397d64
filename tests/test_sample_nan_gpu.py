"""Drawn tokens where NaN, infinities and the largest numbers stand among the logits, against the definition in 64 bits."""
import pytest
import torch

from ml_framework_b200.ops import native, reference

pytestmark = pytest.mark.gpu
INF, NAN, MOST = float("inf"), float("nan"), torch.finfo(torch.float32).max


def _same(x, vocab, u, *settings):
    got, lp = native.sample_rows(x, vocab, u, *settings, want_logprobs=True)
    want, want_lp = reference.sample_ref(x, vocab, u, *settings)
    assert torch.equal(got, want), (got != want).nonzero().flatten().tolist()
    assert ((lp - want_lp).abs() <= 2.0 ** -23 * want_lp.abs() + 2.0 ** -29).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [300, 5000, 40001, 140001])
@pytest.mark.parametrize("top", [INF, MOST])
@pytest.mark.parametrize("which", ["", "k", "p", "m", "kp"])
def test_nan_beside_the_largest_numbers(dtype, vocab, top, which):
    """NaN counts as -inf, and a finite logit weighs nothing beside an infinite one, the largest finite one included."""
    rows = 8
    g = torch.Generator(device="cuda").manual_seed(vocab)
    top = min(top, torch.finfo(dtype).max) if top != INF else top
    x = torch.randn(rows, vocab, device="cuda", generator=g)
    x[:, ::3] = NAN
    x[:, 1::5] = torch.finfo(dtype).max                         # beside infinities: no weight; else: all that counts
    x[:, 7] = top
    x[1::2, 200] = top
    x = x.to(dtype)
    u = torch.rand(rows, device="cuda", generator=g)
    t = torch.tensor([1.0, 1.0, 0.5, 2.0, 1e30, 1e20, 1.0, 0.7], device="cuda")
    k = torch.tensor([1, 2, 3, 50, 299, 4000, 0, 7], dtype=torch.int32, device="cuda") if "k" in which else None
    p = torch.tensor([0.9, 0.5, 0.99, 0.9, 0.7, 0.9999, 0.1, 0.0], device="cuda") if "p" in which else None
    m = torch.full((rows,), 0.1, device="cuda") if "m" in which else None
    _same(x, vocab, u, t, k, p, m)
