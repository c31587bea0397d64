"""The gather from an 8-bit cache where a thread takes two rows: from 65536 (token, head) pairs on, its remainders and bad table entries."""
import pytest
import torch

from ml_framework_b200 import _lib
from ml_framework_b200.ops import native, reference

pytestmark = pytest.mark.gpu
D = 128
KINDS = [torch.float8_e4m3fn, torch.int8]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _cache(nb, bs, Hkv, dtype, g):
    n = torch.randn(nb, 2, bs, Hkv, D, device="cuda", generator=g) * 60
    return reference.q8_round_ref(n, dtype), torch.exp2(torch.randint(-9, 3, (nb, 2, Hkv), device="cuda", generator=g).float())


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("bs,Hkv,n", [(16, 8, 8191), (16, 8, 8192), (16, 8, 8195), (24, 3, 21845), (24, 3, 21847), (16, 1, 65537), (16, 1, 65551), (16, 40, 1639),
                                      (5, 2, 32783)])
def test_gather_around_two_rows_a_thread(dtype, bs, Hkv, n):
    """Both sides of 65536 rows, and remainders of a CTA's 32."""
    g = _gen(n)
    nb = (n + bs - 1) // bs + 3
    cache, scale = _cache(nb, bs, Hkv, dtype, g)
    row = torch.randperm(nb, device="cuda", generator=g)[:(n + bs - 1) // bs].to(torch.int32)
    k, v = native.kv_gather(cache, row, n, kv_scale=scale)
    want = reference.kv_values_ref(cache[row.long()], scale[row.long()]).transpose(0, 1).reshape(2, -1, Hkv, D)[:, :n].to(torch.bfloat16)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.parametrize("bad", [-1, 4100, 1 << 30])
@pytest.mark.parametrize("entry", [0, 1, 4096])
def test_gather_reports_a_bad_entry(bad, entry):
    """In the first and the second row of a thread, and in the remainder: reported, and every other block's rows are right."""
    bs, Hkv, n = 16, 1, 65537 + 9
    g = _gen(5)
    cache, scale = _cache(4100, bs, Hkv, torch.int8, g)
    row = torch.randperm(4100, device="cuda", generator=g)[:(n + bs - 1) // bs].to(torch.int32)
    row[entry] = bad
    k, v = native.kv_gather(cache, row, n, kv_scale=scale)
    assert _lib.read_status(True) == 7
    row[entry] = 0
    want = reference.kv_values_ref(cache[row.long()], scale[row.long()]).transpose(0, 1).reshape(2, -1, Hkv, D)[:, :n].to(torch.bfloat16)
    keep = torch.arange(n, device="cuda") // bs != entry
    assert torch.equal(k[keep], want[0][keep]) and torch.equal(v[keep], want[1][keep])
