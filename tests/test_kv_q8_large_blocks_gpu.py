"""Single-token attention over an 8-bit cache whose blocks are so large, and whose splits so many, that the places where splits would
begin pass 2^31 and 2^32."""
import pytest
import torch

from ml_framework_b200.ops import native, reference

pytestmark = pytest.mark.gpu
D = 128


@pytest.mark.parametrize("dtype", [torch.float8_e4m3fn, torch.int8])
@pytest.mark.parametrize("bs,longest", [(65536, 8_000_000), (65536, 4_300_000), (40000, 8_380_000), (50001, 8_000_000)])
def test_splits_far_behind_the_last_token(dtype, bs, longest):
    """128 tokens a split by the call, a block each by the kernel: all but the first three have nothing to do."""
    g = torch.Generator(device="cuda").manual_seed(bs)
    n = 2 * bs + 77
    cache = reference.q8_round_ref(60 * torch.randn(3, 2, bs, 1, D, device="cuda", generator=g), dtype)
    scale = torch.full((3, 2, 1), 0.125, device="cuda")
    table = torch.zeros(1, longest // bs + 1, dtype=torch.int32, device="cuda")
    table[0, :3] = torch.tensor([2, 0, 1])
    lens = torch.tensor([n], dtype=torch.int32, device="cuda")
    q = torch.randn(1, 2, D, device="cuda", generator=g).to(torch.bfloat16)
    got = native.paged_decode(q, cache, table, lens, longest, split_tokens=128, kv_scale=scale).double()
    kv = (cache[table[0, :3].long()].float() * 0.125).transpose(0, 1).reshape(2, -1, D)[:, :n].double()
    x = q[0].double() @ kv[0].T * D ** -0.5
    p = torch.softmax(x, -1)
    want, size = p @ kv[1], p @ kv[1].abs()
    big = (q[0].double().abs() @ kv[0].abs().T * D ** -0.5).amax()
    # weights in f16, a quarter of that for the exponentials, scores as sums of 128 fp32 products, the result in bf16; weights below 2^-29 of
    # the largest are off by 2^-40 of it, each times a number of 8 bits
    small = 2.0 ** -40 * p.amax() * kv[1].abs().sum(0)
    assert ((got[0] - want).abs() <= 2.0 ** -8 * want.abs() + (2.0 ** -11 + 2.0 ** -13 + 2.0 ** -16 * big) * size + small).all()
