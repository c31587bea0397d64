"""Tokens from given random numbers against the definition in 64 bits. Tokens are compared exactly: the kernel's weights are good to
about 2^-30 and its sums exact, so that a draw differs only where u lies within some 2^-30 of a border between two tokens
(likelier than 1e-6 in none of these cases); where it does, and only then, the neighbour across that border is right too.
Log-probabilities: computed in 64 bits from weights that are each off by 2^-30 at most, 2^-29 in all, and rounded to fp32: 2^-24 of the
value."""
import pytest
import torch

from ml_framework_b200 import _lib
from ml_framework_b200.ops import native, reference

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _same(logits, vocab, u, *settings):
    got, lp = native.sample_rows(logits, vocab, u, *settings, want_logprobs=True)
    want, want_lp = reference.sample_ref(logits, vocab, u, *settings)
    assert got.dtype == torch.int64 and torch.equal(got, want), (got != want).nonzero().flatten().tolist()
    fin = torch.isfinite(want_lp)
    assert torch.equal(fin, torch.isfinite(lp)) and torch.equal(lp[~fin], want_lp[~fin])
    assert ((lp[fin] - want_lp[fin]).abs() <= 2.0 ** -23 * want_lp[fin].abs() + 2.0 ** -29).all()
    assert torch.equal(native.sample_rows(logits, vocab, u, *settings), got)
    return got


def _settings(rows, g, which):
    t = 0.3 + 1.5 * torch.rand(rows, device="cuda", generator=g)
    k = torch.randint(1, 300, (rows,), device="cuda", generator=g).to(torch.int32) if "k" in which else None
    p = 0.2 + 0.85 * torch.rand(rows, device="cuda", generator=g) if "p" in which else None
    m = 0.2 * torch.rand(rows, device="cuda", generator=g) if "m" in which else None
    return t, k, p, m


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,pad", [(1, 1, 0), (3, 2, 5), (7, 255, 1), (5, 1000, 24), (4, 4097, 63), (33, 32000, 0), (2, 50257, 47), (5, 128256, 0), (300, 700, 0)])
@pytest.mark.parametrize("which", ["", "k", "p", "m", "kp", "kpm"])
def test_matches_the_definition(dtype, rows, vocab, pad, which):
    g = _gen(rows * 1000 + vocab)
    x = 3 * torch.randn(rows, vocab + pad, device="cuda", generator=g)
    x[:, vocab:] = 100.0                                        # padding is not part of the vocabulary
    u = torch.rand(rows, device="cuda", generator=g)
    t, k, p, m = _settings(rows, g, which)
    t[::5] = 0
    _same(x.to(dtype), vocab, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", ["flat", "two values", "outlier", "narrow", "steep", "masked", "one left"])
@pytest.mark.parametrize("which", ["", "k", "p", "kp", "m"])
def test_shapes_of_distributions(dtype, shape, which):
    """All equal, many ties, one far above a dense cluster, everything within one bin, weights that underflow, masks."""
    rows, vocab = 9, 20011
    g = _gen(len(shape))
    x = torch.randn(rows, vocab, device="cuda", generator=g)
    if shape == "flat":
        x = torch.full_like(x, -3.25)
    elif shape == "two values":
        x = (x > 0.5).float() * 0.5
    elif shape == "outlier":
        x = x * 1e-3
        x[:, 17] = 5.0
    elif shape == "narrow":
        x = 100 + 0.25 * x
    elif shape == "steep":
        x = 200 * x
    elif shape == "masked":
        x[x < 1.5] = float("-inf")
    elif shape == "one left":
        x[:] = float("-inf")
        x[torch.arange(rows), torch.arange(rows) * 2000] = -7.0
    u = torch.rand(rows, device="cuda", generator=g)
    t = torch.full((rows,), 1.0, device="cuda")
    k = torch.tensor([1, 2, 100, 2048, 2049, 5000, 20010, 20011, 30000], dtype=torch.int32, device="cuda") if "k" in which else None
    p = torch.tensor([0.0, 1e-6, 0.1, 0.5, 0.9, 0.99, 0.9999, 1.0, 2.0], device="cuda") if "p" in which else None
    m = torch.tensor([0.0, 1e-30, 1e-4, 0.01, 0.1, 0.5, 0.9, 1.0, 2.0], device="cuda") if "m" in which else None
    _same(x.to(dtype), vocab, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [40000, 128256, 140000])
@pytest.mark.parametrize("shape", ["sorted", "few left", "first only", "hot bulk"])
def test_where_candidates_lie(dtype, vocab, shape):
    """Candidates side by side, a mask that leaves a handful, none in the first logits of every lane, a nucleus of most tokens;
    vocabularies that shared memory holds and one that it does not."""
    rows = 10
    g = _gen(vocab)
    x = 2 * torch.randn(rows, vocab, device="cuda", generator=g)
    if shape == "sorted":
        x = x.sort(1, descending=True)[0]
    elif shape == "few left":
        x = torch.where(torch.rand(rows, vocab, device="cuda", generator=g) < 1e-4, x, float("-inf"))
        x[:, 5] = 1.0
    elif shape == "first only":
        x[:, 3000:] = float("-inf")
    else:
        x[:, 77] = 9.0
    u = torch.rand(rows, device="cuda", generator=g)
    t = torch.tensor([1.0, 0.5, 1.5, 1.0, 0.7, 1.0, 2.0, 0.3, 1.0, 1.0], device="cuda")
    k = torch.tensor([0, 0, 0, 50, 300, 1500, 0, 40000, 600, 0], dtype=torch.int32, device="cuda")
    p = torch.tensor([0.9, 0.95, 0.99, 0.9, 1.0, 0.9, 0.5, 0.9, 1.0, 0.9999], device="cuda")
    m = torch.tensor([0, 0, 0, 0, 0.01, 0, 0, 0, 0, 0.001], device="cuda")
    _same(x.to(dtype), vocab, u, t, k, p, m)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_largest_vocabulary(dtype):
    """2^20 tokens, and one more, which is refused."""
    n = 1 << 20
    g = _gen(20)
    x = (3 * torch.randn(3, n + 8, device="cuda", generator=g)).to(dtype)
    u = torch.rand(3, device="cuda", generator=g)
    t = torch.tensor([0.7, 1.0, 1.3], device="cuda")
    p = torch.tensor([0.9, 1.0, 0.95], device="cuda")
    k = torch.tensor([0, 0, 700], dtype=torch.int32, device="cuda")
    _same(x, n, u, t, k, p)
    _same(x, n - 5, u, t, None, p)
    with pytest.raises(_lib.MlfError, match="vocabulary"):
        native.sample_rows(x, n + 1, u, t)


@pytest.mark.parametrize("vocab", [9001, 70001, 140001])
@pytest.mark.parametrize("shape", ["near zero", "far below", "negative", "small", "huge", "with nan and inf"])
def test_p_decides_anywhere(vocab, shape):
    """A p alone over bf16 logits that lie near 0 beside large ones, far below the first ones of the row, below 0, among the smallest normal
    numbers, among the largest, and beside NaN and infinities; temperatures that make most of them count."""
    rows = 8
    g = _gen(vocab + len(shape))
    x = torch.randn(rows, vocab, device="cuda", generator=g)
    heat = 1.0
    if shape == "near zero":
        x = x * 2.0 ** -16
        x[:, 11] = 8.0
        heat = 4.0
    elif shape == "far below":
        x[:, vocab // 9:] -= 1000.0
        heat = 2000.0
    elif shape == "negative":
        x = -20.0 - 3 * x.abs()
        heat = 3.0
    elif shape == "small":
        x = x * 2.0 ** -126
        heat = 2.0 ** -126
    elif shape == "huge":
        x = x * 2.0 ** 125
        heat = 2.0 ** 126
    else:
        x[:, ::7] = float("nan")
        x[:, 1::7] = -x[:, 1::7].abs()
        x[:, 2::7] = float("-inf")
        x[::2, 3] = float("inf")
    x = x.to(torch.bfloat16)
    if shape == "small":
        x = torch.where(x.float().abs() < 2.0 ** -126, 0.0, x.float()).to(torch.bfloat16)      # a subnormal logit counts as 0
    u = torch.rand(rows, device="cuda", generator=g)
    t = heat * torch.tensor([1.0, 0.5, 1.5, 1.0, 0.7, 1.0, 2.0, 0.3], device="cuda")
    p = torch.tensor([0.1, 0.3, 0.5, 0.7, 0.9, 0.99, 0.9999, 0.6], device="cuda")
    _same(x, vocab, u, t, None, p)
    _same(x, vocab, u, t, None, p, torch.full((rows,), 0.05, device="cuda"))


def test_ends_of_u_and_odd_numbers():
    x = torch.tensor([[1.0, 3.0, 2.0, 3.0, float("nan"), float("-inf")]] * 6, device="cuda")
    x[3, 1] = float("inf")
    x[4] = float("-inf")
    x[5] = float("nan")
    t = torch.tensor([1.0, 1.0, float("inf"), 1.0, 1.0, 0.0], device="cuda")
    u = torch.tensor([0.0, 1.0 - 2.0 ** -24, 0.6, 0.99, 0.5, 0.5], device="cuda")
    tok, lp = native.sample_rows(x, 6, u, t, want_logprobs=True)
    assert tok.tolist() == [0, 3, 2, 1, 0, 0]
    assert torch.isneginf(lp[4]) and torch.isneginf(lp[5]) and abs(float(lp[3])) == 0 and abs(float(lp[2]) + 1.3862944) < 1e-6
    zero = torch.tensor([[0.0, -0.0, -1.0]], device="cuda")       # equal logits: the lower index is first
    one = torch.tensor([1], dtype=torch.int32, device="cuda")
    assert native.sample_rows(zero, 3, u[1:2], t[:1], one).item() == 0
    assert native.sample_rows(zero, 3, u[1:2], t[:1] * 0).item() == 0


@pytest.mark.parametrize("top", [float("inf"), 0.0, -1.1754944e-38, 3.3895314e38])
def test_ties_at_odd_values(top):
    """The lowest indices of equal logits at infinity, zero, the largest bf16 and minus the smallest normal number."""
    x = torch.full((3, 5000), -5.0, device="cuda")
    x[:, 100:4000] = top
    if top == 0.0:
        x[:, 200:300] = -0.0
    u = torch.tensor([0.0, 0.5, 0.999], device="cuda")
    k = torch.tensor([3000, 3000, 2], dtype=torch.int32, device="cuda")
    t = torch.ones(3, device="cuda")
    for dtype in (torch.float32, torch.bfloat16):
        assert native.sample_rows(x.to(dtype), 5000, u, t, k).tolist() == [100, 1600, 101]


def test_a_row_does_not_depend_on_the_others():
    """The same row alone (a cluster of CTAs), and in a batch of 600 (fewer CTAs for it)."""
    g = _gen(4)
    x = (3 * torch.randn(600, 40000, device="cuda", generator=g)).to(torch.bfloat16)
    u = torch.rand(600, device="cuda", generator=g)
    t, k, p, m = _settings(600, g, "kpm")
    k[::2] = 0
    p[::3] = 1.0
    m[::5] = 0
    every, lp = native.sample_rows(x, 40000, u, t, k, p, m, want_logprobs=True)
    for i in (0, 1, 2, 3, 6, 599):
        s = slice(i, i + 1)
        a, b = native.sample_rows(x[s], 40000, u[s], t[s], k[s], p[s], m[s], want_logprobs=True)
        assert a.item() == every[i].item() and b.item() == lp[i].item()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("vocab", [9000, 130001])
@pytest.mark.parametrize("mask", ["lowest", -1e4, -1e9, float("-inf")])
@pytest.mark.parametrize("left", [1, 5, 600, 5000])
def test_masked_by_a_large_number(dtype, vocab, mask, left):
    """Few tokens left beside the type's lowest value, -1e4, -1e9 or -inf, at places that no sample of the row needs to meet."""
    rows = 12
    g = _gen(left)
    x = torch.full((rows, vocab), torch.finfo(dtype).min if mask == "lowest" else mask, device="cuda")
    at = torch.rand(rows, vocab, device="cuda", generator=g).topk(left, 1)[1]
    if left == 600:
        at = torch.arange(vocab - left, vocab, device="cuda").expand(rows, -1)
    x.scatter_(1, at, 3 * torch.randn(rows, left, device="cuda", generator=g))
    x = x.to(dtype)
    u = torch.rand(rows, device="cuda", generator=g)
    t = torch.tensor([1.0, 0.0, 0.5, 1.0, 0.7, 1.3], device="cuda").repeat(2)
    k = torch.tensor([0, 0, 50, 0, 3000, 700], dtype=torch.int32, device="cuda").repeat(2)
    p = torch.tensor([0.9, 0.9, 0.9, 1.0, 0.95, 1.0], device="cuda").repeat(2)
    m = torch.tensor([0.0] * 6 + [0.05] * 6, device="cuda")
    _same(x, vocab, u, t, k, p, m)
    _same(x, vocab, u, t, None, p)


@pytest.mark.parametrize("rows", [200, 300, 513, 1000, 1024, 1025])
def test_every_row_of_a_large_batch(rows):
    """More rows than run at once, of all kinds in any order, without settings too: each gets its own token."""
    vocab = 9000
    g = _gen(rows)
    x = (3 * torch.randn(rows, vocab, device="cuda", generator=g)).to(torch.bfloat16)
    u = torch.rand(rows, device="cuda", generator=g)
    t, k, p, m = _settings(rows, g, "kpm")
    kind = torch.randint(0, 6, (rows,), device="cuda", generator=g)
    t[kind == 0] = 0.0
    k[(kind == 1) | (kind >= 4)] = 0
    p[(kind == 2) | (kind == 5)] = 1.0
    m[kind != 3] = 0.0
    _same(x, vocab, u, t, k, p, m)
    _same(x, vocab, u, t)
    _same(x, vocab, u, t, None, p)


def test_frequencies():
    """200 K draws of a known distribution: counts within six standard deviations."""
    n = 200_000
    pr = torch.tensor([0.5, 0.25, 0.125, 0.0625, 0.0625], device="cuda")
    u = torch.rand(n, device="cuda", generator=_gen(1))
    x = torch.log(pr)[None].expand(n, 5).contiguous()
    got = torch.bincount(native.sample_rows(x, 5, u, torch.ones(n, device="cuda")), minlength=5).double()
    assert ((got - n * pr.double()).abs() <= 6 * (n * pr * (1 - pr)).sqrt()).all()


def test_captured():
    g = _gen(2)
    x = 3 * torch.randn(4, 32000, device="cuda", generator=g)
    u = torch.rand(4, device="cuda", generator=g)
    t, k, p, m = _settings(4, g, "kpm")
    native.sample_rows(x, 32000, u, t, k, p, m)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = native.sample_rows(x, 32000, u, t, k, p, m)
    for i in range(5):
        u.uniform_(generator=g)
        k.random_(1, 100, generator=g)
        graph.replay()
        assert torch.equal(out, reference.sample_ref(x, 32000, u, t, k, p, m)[0])
