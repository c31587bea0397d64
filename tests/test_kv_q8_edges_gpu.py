"""Writes and appends to 8-bit blocks whose scales, given by the caller, are no powers of two: the bytes of the PyTorch statement, which
divides."""
import pytest
import torch

from ml_framework_b200.ops import native, reference

pytestmark = pytest.mark.gpu
D = 128
KINDS = [torch.float8_e4m3fn, torch.int8]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _bytes(t):
    return t.view(torch.uint8)


SCALES = [3.0, 5.0, 0.75, 1.5, 1.125, 7.0 / 64, 1.0]


def _uneven(nb, bs, Hkv, dtype, g):
    """Blocks under scales that are no powers of two (and some that are)."""
    n = torch.randn(nb, 2, bs, Hkv, D, device="cuda", generator=g) * 20
    pick = torch.randint(0, len(SCALES), (nb, 2, Hkv), device="cuda", generator=g)
    return reference.q8_round_ref(n, dtype), torch.tensor(SCALES, device="cuda")[pick]


def _halves(scale, shape, g):
    """Numbers half way between two steps of the scales: as many as bf16 holds exactly, and a few beyond the block's range."""
    n = torch.randint(-40, 40, shape, device="cuda", generator=g).float() + 0.5
    return (n * scale[..., None]).to(torch.bfloat16)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("bs,Hkv,T", [(16, 2, 1), (16, 8, 40), (16, 2, 300), (24, 3, 50), (8, 1, 2100), (72, 2, 100), (5, 2, 33)])
def test_write_behind_rows_of_any_scale(dtype, bs, Hkv, T):
    """Later rows of blocks that keep their scale, or leave it for a larger one: the bytes of the statement, ties included."""
    g = _gen(T + bs)
    nb = T // max(bs - 1, 1) + 2
    cache, scale = _uneven(nb, bs, Hkv, dtype, g)
    t = torch.arange(T, device="cuda")
    blk, off = t // (bs - 1), t % (bs - 1) + 1                  # never a block's first row
    slots = blk * bs + off
    k, v = (_halves(scale[blk, j], (T, Hkv, D), g) for j in (0, 1))
    grow = (blk % 3 == 2)[:, None, None]
    k, v = torch.where(grow, k * 16, k), torch.where(grow, v * 16, v)
    want_c, want_s = cache.clone(), scale.clone()
    reference.kv_write_ref(want_c, k, v, slots, want_s)
    native.kv_cache_write(cache, k, v, slots, kv_scale=scale)
    assert torch.equal(scale, want_s)
    assert torch.equal(_bytes(cache), _bytes(want_c))


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("bs", [16, 24])
def test_append_behind_rows_of_any_scale(dtype, bs):
    """The append inside the attention holds what the statement of a write holds, and so attends to the same."""
    lens, Hq, Hkv = [2, 16, 30, 7, 100, 130], 8, 2
    B = len(lens)
    g = _gen(bs)
    need = [(n + bs - 1) // bs for n in lens]
    table = torch.zeros(B, max(need), dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = torch.arange(at, at + n, device="cuda")
        at += n
    cache, scale = _uneven(at, bs, Hkv, dtype, g)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    slots = torch.stack([table[i, (n - 1) // bs].long() * bs + (n - 1) % bs for i, n in enumerate(lens)])
    qkv = torch.randn(B, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(torch.bfloat16)
    qkv[:, (Hq + Hkv) * D:] = _halves(scale[slots // bs, 1], (B, Hkv, D), g).view(B, -1)
    rot = native.rope_qkv(qkv, sl.long() - 1, Hq, Hkv, 5e5)
    want_c, want_s = cache.clone(), scale.clone()
    reference.kv_write_ref(want_c, rot[:, Hq * D:(Hq + Hkv) * D].view(B, Hkv, D), rot[:, (Hq + Hkv) * D:].view(B, Hkv, D), slots, want_s)
    want = native.paged_decode(rot[:, :Hq * D].view(B, Hq, D), want_c, table, sl, max(lens), split_tokens=0, kv_scale=want_s)
    got = native.paged_decode_rope(qkv, cache, table, sl, slots, Hq, Hkv, max(lens), 5e5, kv_scale=scale)
    assert torch.equal(scale, want_s) and torch.equal(_bytes(cache), _bytes(want_c))
    assert torch.equal(got, want)
