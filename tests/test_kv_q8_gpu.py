"""A paged cache in 8 bits: writes bit for bit against the PyTorch statement, attention against 64 bits within the roundings that
the kernel makes, the fused append against its two steps, copies of blocks.

Attention's tolerance, with A = sum_t p_t |v_t| and x = max_t scale sum_d |q_d k_td|: the weights are rounded to f16 (2^-11 of each, and a
quarter of that for the exponentials), a score is a sum of 128 fp32 products (at most 2^-17 x, which its weight takes over) and the
result is rounded to bf16: 2^-8 |o| + (2^-11 + 2^-13 + 2^-16 x) A. Weights p_t s_V(t) that f16 holds with fewer bits, those below
2^-29 of the largest, are off by 2^-40 of that one at most, each times a number |V_t| of 8 bits:
+ 2^-40 max_t(p_t s_V(t)) sum_t |V_t|."""
import pytest
import torch

from ml_framework_b200 import _lib
from ml_framework_b200.ops import native, reference

pytestmark = pytest.mark.gpu
D = 128
KINDS = [torch.float8_e4m3fn, torch.int8]


def _bytes(t):
    return t.view(torch.uint8)


def _random_cache(nb, bs, Hkv, dtype, g, power=True):
    n = torch.randn(nb, 2, bs, Hkv, D, device="cuda", generator=g) * 60
    s = torch.exp2(torch.randint(-9, 3, (nb, 2, Hkv), device="cuda", generator=g).float())
    if not power:
        s = s * (1 + torch.rand(nb, 2, Hkv, device="cuda", generator=g))
    return reference.q8_round_ref(n, dtype), s


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


# ------------------------------------------------------------------ writes
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("bs,Hkv", [(16, 8), (16, 1), (24, 3), (8, 2), (40, 5), (1, 2), (72, 2)])
@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 37, 255, 256, 300])
def test_write_matches_the_statement(dtype, bs, Hkv, T):
    g = _gen(T * 100 + bs)
    nb = T // bs + 5
    cache, scale = _random_cache(nb, bs, Hkv, dtype, g)
    wide = torch.randn(T, 3, Hkv, D, device="cuda", generator=g) * torch.exp2(torch.randint(-4, 7, (T, 1, Hkv, 1), device="cuda", generator=g).float())
    wide = wide.to(torch.bfloat16)
    k, v = wide[:, 1], wide[:, 2]                              # strided rows, as in a packed projection
    order = torch.randperm(nb, device="cuda", generator=g)
    pos = torch.arange(bs // 2, bs // 2 + T, device="cuda")    # begins inside a block (its first row for blocks of one)
    slots = order[pos // bs] * bs + pos % bs
    if T > 2:
        slots[T // 2] = -1
    want_c, want_s = cache.clone(), scale.clone()
    reference.kv_write_ref(want_c, k, v, slots, want_s)
    shuffled = torch.randperm(T, device="cuda", generator=g)
    for order in (None, shuffled):
        c, s = cache.clone(), scale.clone()
        if order is None:
            native.kv_cache_write(c, k, v, slots, kv_scale=s)
        else:
            native.kv_cache_write(c, k[order], v[order], slots[order], kv_scale=s)
        assert torch.equal(s, want_s)
        assert torch.equal(_bytes(c), _bytes(want_c))


@pytest.mark.parametrize("bs,T", [(16, 2048), (16, 2049), (24, 2200), (72, 300), (72, 2100)])
def test_long_writes(bs, T):
    """Calls, and blocks, beyond what a CTA looks through."""
    test_write_matches_the_statement(torch.int8, bs, 2, T)


@pytest.mark.parametrize("dtype", KINDS)
def test_write_extremes(dtype):
    """Zeros, the borders between two scales, infinities, NaN, values beyond the largest scale; one row at a time."""
    top = 448.0 if dtype == torch.float8_e4m3fn else 127.0
    rows = [0.0, top, top * 1.01, top * 2.0 ** -41, 2.0 ** -60, 3e38, float("inf"), float("nan"), 1.0, top * 2.0 ** 41]
    bs, nb = 16, 2
    cache = torch.zeros(nb, 2, bs, 1, D, device="cuda").to(dtype)
    scale = torch.zeros(nb, 2, 1, device="cuda")
    want_c, want_s = cache.clone(), scale.clone()
    for i, r in enumerate(rows):
        k = torch.linspace(-1, 1, D, device="cuda").mul(1.0 if r != r or r in (float("inf"),) else r).to(torch.bfloat16).view(1, 1, D).clone()
        if r != r or r == float("inf"):
            k[0, 0, 5], k[0, 0, 6] = r, -r
        slots = torch.tensor([bs + i], device="cuda")
        native.kv_cache_write(cache, k, -k, slots, kv_scale=scale)
        reference.kv_write_ref(want_c, k, -k, slots, want_s)
        assert torch.equal(scale, want_s), r
        a, b = cache.float(), want_c.float()
        assert torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()), r


def test_write_same_slot_twice_and_bad_slots():
    g = _gen(3)
    cache, scale = _random_cache(4, 16, 2, torch.int8, g)
    k = torch.randn(3, 2, D, device="cuda", generator=g).to(torch.bfloat16)
    slots = torch.tensor([16, 16, 4 * 16], device="cuda")            # twice, and a block that does not exist
    c, s = cache.clone(), scale.clone()
    native.kv_cache_write(c, k, k, slots, kv_scale=s)
    got = reference.kv_values_ref(c, s)[1, 0, 0]
    ok = False
    for i in (0, 1):
        wc, ws = cache.clone(), scale.clone()
        reference.kv_write_ref(wc, k[i:i + 1], k[i:i + 1], slots[i:i + 1], ws)
        ok = ok or (torch.equal(_bytes(wc), _bytes(c)) and torch.equal(ws, s))
    assert ok and got.isfinite().all()
    assert _lib.read_status(True) == 7                                # the rejected index is reported


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("T", [1, 40, 300])
def test_rope_write_is_rotation_then_write(dtype, T):
    Hq, Hkv, bs = 8, 2, 16
    g = _gen(T)
    qkv = torch.randn(T, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(torch.bfloat16)
    pos = torch.randint(0, 5000, (T,), device="cuda", generator=g)
    cache, scale = _random_cache(T // bs + 2, bs, Hkv, dtype, g)
    slots = torch.arange(3, 3 + T, device="cuda")
    want, wc, ws = qkv.clone(), cache.clone(), scale.clone()
    native.rope_qkv(want, pos, Hq, Hkv, 5e5, out=want)
    reference.kv_write_ref(wc, want[:, Hq * D:(Hq + Hkv) * D].view(T, Hkv, D), want[:, (Hq + Hkv) * D:].view(T, Hkv, D), slots, ws)
    native.rope_kv_write_(qkv, pos, slots, cache, Hq, Hkv, 5e5, kv_scale=scale)
    assert torch.equal(qkv, want) and torch.equal(scale, ws) and torch.equal(_bytes(cache), _bytes(wc))


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("bs,Hkv,n", [(16, 8, 1), (16, 1, 37), (24, 3, 500), (16, 8, 3001)])
def test_gather(dtype, bs, Hkv, n):
    g = _gen(n)
    nb = n // bs + 3
    cache, scale = _random_cache(nb, bs, Hkv, dtype, g)
    row = torch.randperm(nb, device="cuda", generator=g)[:(n + bs - 1) // bs].to(torch.int32)
    k, v = native.kv_gather(cache, row, n, kv_scale=scale)
    want = reference.kv_values_ref(cache[row.long()], scale[row.long()]).transpose(0, 1).reshape(2, -1, Hkv, D)[:, :n].to(torch.bfloat16)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


# ------------------------------------------------------------------ attention
def _tables(lens, bs, g):
    need = [(n + bs - 1) // bs for n in lens]
    perm = torch.randperm(sum(need) + 1, generator=g, device="cuda")[1:] if sum(need) else torch.zeros(0, dtype=torch.int64, device="cuda")
    table = torch.full((len(lens), max(max(need), 1)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = perm[at:at + n].to(torch.int32)
        at += n
    return table, sum(need) + 1


def _exact(q, cache, scale, table, lens, sm_scale):
    """(o, tolerance) in 64 bits."""
    bs, Hkv = cache.shape[2], cache.shape[3]
    G = q.shape[1] // Hkv
    o = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(o)
    for b, n in enumerate(lens):
        if n == 0:
            continue
        pages = table[b, :(n + bs - 1) // bs].long()
        kv = (cache[pages].double() * scale[pages].double()[:, :, None, :, None]).transpose(0, 1).reshape(2, -1, Hkv, D)[:, :n]
        qb = q[b].double().view(Hkv, G, D)
        x = torch.einsum("hgd,lhd->hgl", qb, kv[0]) * sm_scale
        p = torch.softmax(x, -1)
        o[b] = torch.einsum("hgl,lhd->hgd", p, kv[1]).reshape(-1, D)
        A = torch.einsum("hgl,lhd->hgd", p, kv[1].abs()).reshape(-1, D)
        sv = scale[pages, 1].double().repeat_interleave(bs, 0)[:n].T[:, None]                        # [Hkv, 1, n]
        small = (2.0 ** -40 * (p * sv).amax(-1)[:, :, None] * (kv[1].abs() / sv[:, 0].T[:, :, None]).sum(0)[:, None]).reshape(-1, D)
        big = (torch.einsum("hgd,lhd->hgl", qb.abs(), kv[0].abs()) * sm_scale).amax(-1).reshape(-1, 1)
        tol[b] = 2.0 ** -8 * o[b].abs() + (2.0 ** -11 + 2.0 ** -13 + 2.0 ** -16 * big) * A + small
    return o, tol


def _check(got, want, tol):
    worst = ((got.double() - want).abs() - tol).max()
    assert got.isfinite().all() and worst <= 0, float(worst)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (32, 8), (12, 4), (8, 1), (16, 1), (14, 2), (11, 1)])
@pytest.mark.parametrize("bs,split,power", [(16, 0, True), (16, 128, False), (24, 256, True), (40, 0, False), (7, 128, True), (64, 128, True), (256, 128, True)])
def test_attention(dtype, Hq, Hkv, bs, split, power):
    lens = [1, 0, 2, 15, 16, 17, 63, 64, 65, 128, 129, 500, 1000, 7]
    g = _gen(Hq * 31 + bs)
    table, nb = _tables(lens, bs, g)
    cache, scale = _random_cache(nb, bs, Hkv, dtype, g, power)
    scale = scale * 2.0 ** -3
    wide = torch.randn(len(lens), Hq * D + 2, device="cuda", generator=g).to(torch.bfloat16)
    q = wide[:, 2:].view(len(lens), Hq, D) if Hq == 12 else wide[:, :Hq * D].view(len(lens), Hq, D)   # 4-byte aligned rows too
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = native.paged_decode(q, cache, table, sl, max(lens), split_tokens=split, kv_scale=scale)
    want, tol = _exact(q, cache, scale, table, lens, D ** -0.5)
    _check(got, want, tol)
    assert (got[1] == 0).all()


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("split,bs,Hq", [(128, 16, 8), (128, 24, 8), (256, 16, 32), (0, 16, 8), (1024, 16, 2), (400, 48, 8)])
def test_attention_many_splits(dtype, split, bs, Hq):
    """Splits that a cluster merges (two to eight) and more, which a second kernel does; sequences that end in any of them."""
    lens = [20000, 1, 0, 129, 1025, 2048, 7777, 17000]
    g = _gen(split)
    table, nb = _tables(lens, bs, g)
    cache, scale = _random_cache(nb, bs, 2, dtype, g)
    scale = scale * 2.0 ** -4
    q = torch.randn(len(lens), Hq, D, device="cuda", generator=g).to(torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, tol = _exact(q, cache, scale, table, lens, D ** -0.5)
    got = native.paged_decode(q, cache, table, sl, max(lens), split_tokens=split, kv_scale=scale)
    _check(got, want, tol)
    assert (got[2] == 0).all()


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("B,n,Hq,Hkv", [(150, 333, 8, 4), (200, 300, 12, 4), (300, 60, 16, 8), (300, 130, 24, 8), (40, 100, 16, 8), (65, 450, 16, 8),
                                        (130, 450, 8, 8), (160, 450, 16, 8), (300, 450, 4, 4), (30, 1600, 16, 8)])
def test_attention_forms_of_the_launch(dtype, B, n, Hq, Hkv):
    """Four, three and two warps to a CTA: by the places that the rounds of CTAs take, and short sequences; then with the append."""
    g = _gen(B)
    lens = torch.randint(1, n + 1, (B,), generator=torch.Generator().manual_seed(B)).tolist()
    lens[0] = n
    table, nb = _tables(lens, 16, g)
    cache, scale = _random_cache(nb, 16, Hkv, dtype, g)
    scale = scale * 2.0 ** -4
    q = torch.randn(B, Hq, D, device="cuda", generator=g).to(torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, tol = _exact(q, cache, scale, table, lens, D ** -0.5)
    _check(native.paged_decode(q, cache, table, sl, n, split_tokens=0, kv_scale=scale), want, tol)
    qkv = torch.randn(B, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(torch.bfloat16)
    slots = table.gather(1, ((sl.long() - 1) // 16)[:, None])[:, 0].long() * 16 + (sl.long() - 1) % 16
    a_c, a_s, rot = cache.clone(), scale.clone(), qkv.clone()
    native.rope_kv_write_(rot, sl.long() - 1, slots, a_c, Hq, Hkv, 5e5, kv_scale=a_s)
    want = native.paged_decode(rot[:, :Hq * D].view(B, Hq, D), a_c, table, sl, n, split_tokens=0, kv_scale=a_s)
    got = native.paged_decode_rope(qkv, cache, table, sl, slots, Hq, Hkv, n, 5e5, kv_scale=scale)
    assert torch.equal(got, want) and torch.equal(_bytes(cache), _bytes(a_c)) and torch.equal(scale, a_s)


@pytest.mark.parametrize("dtype", KINDS)
def test_attention_wide_ranges(dtype):
    """Scales 2^-40 to 2^40 side by side, queries of very different size, one key that takes all the weight."""
    lens, bs, Hkv, G = [300, 77], 16, 2, 4
    g = _gen(5)
    table, nb = _tables(lens, bs, g)
    cache, _ = _random_cache(nb, bs, Hkv, dtype, g)
    scale = torch.exp2(torch.randint(-12, -5, (nb, 2, Hkv), device="cuda", generator=g).float())
    scale[:, 1] = torch.exp2(torch.randint(-40, 41, (nb, Hkv), device="cuda", generator=g).float())
    q = torch.randn(2, Hkv * G, D, device="cuda", generator=g) * torch.exp2(torch.randint(-30, 1, (2, Hkv * G, 1), device="cuda", generator=g).float())
    q[0, 0] = 0
    q = q.to(torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, tol = _exact(q, cache, scale, table, lens, D ** -0.5)
    for split in (128, 1024):
        _check(native.paged_decode(q, cache, table, sl, 300, split_tokens=split, kv_scale=scale), want, tol)


def test_attention_ignores_what_lies_behind_a_sequence():
    """NaN numbers behind the last token, stale scales in unused blocks, table entries of -1."""
    lens, bs = [5, 33], 16
    g = _gen(6)
    table, nb = _tables(lens, bs, g)
    cache, scale = _random_cache(nb, bs, 1, torch.float8_e4m3fn, g)
    scale = scale * 2.0 ** -3
    q = torch.randn(2, 4, D, device="cuda", generator=g).to(torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want = native.paged_decode(q, cache, table, sl, 33, kv_scale=scale)
    raw = _bytes(cache)
    raw[table[0, 0].long(), :, 5:] = 0x7f
    raw[table[1, 2].long(), :, 1:] = 0x7f
    unused = [b for b in range(nb) if not (table == b).any()]
    assert len(unused) == 1
    raw[unused] = 0x7f
    scale[unused] = float("nan")
    assert torch.equal(native.paged_decode(q, cache, table, sl, 33, kv_scale=scale), want)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("n,split", [(40, 0), (700, 128), (3000, 128)])
def test_attention_keeps_nan(dtype, n, split):
    """A NaN in a query head, or (e4m3) in a cached key or value, is one of that head's outputs, and of no other's."""
    g = _gen(n)
    cache, scale = _random_cache(n // 16 + 2, 16, 2, dtype, g)
    table = torch.arange(n // 16 + 2, device="cuda", dtype=torch.int32)[None].expand(2, -1).contiguous()
    lens = torch.tensor([n, n], device="cuda", dtype=torch.int32)
    q = torch.randn(2, 8, D, device="cuda", generator=g).bfloat16()
    good = native.paged_decode(q, cache, table, lens, n, split_tokens=split, kv_scale=scale)
    q[1, 5, 17] = float("nan")
    got = native.paged_decode(q, cache, table, lens, n, split_tokens=split, kv_scale=scale)
    assert got[1, 5].isnan().all()
    got[1, 5] = good[1, 5]
    assert torch.equal(got, good)
    if dtype == torch.float8_e4m3fn:
        q[1, 5, 17] = 0.0
        bad = cache.clone()
        _bytes(bad)[1, 0, 3, 1, 9] = 0x7f                      # token 19: the key of head 1
        got = native.paged_decode(q, bad, table, lens, n, split_tokens=split, kv_scale=scale)
        assert got[:, 4:].isnan().all() and torch.equal(got[0, :4], good[0, :4])
        bad = cache.clone()
        _bytes(bad)[1, 1, 3, 0, 9] = 0x7f                      # a value of head 0
        got = native.paged_decode(q, bad, table, lens, n, split_tokens=split, kv_scale=scale)
        assert got[:, :4, 9].isnan().all() and not got[:, :4, :9].isnan().any() and torch.equal(got[0, 4:], good[0, 4:])


def test_operands_at_odd_addresses():
    """Rows that start on no 16 (queries: 4) bytes, contiguous ones too, are copied before the launch."""
    g = _gen(77)
    for T in (1, 5):
        cache, scale = _random_cache(3, 16, 2, torch.int8, g)
        flat = torch.randn(2 * T * 2 * D + 3, device="cuda", generator=g).bfloat16()
        k, v = flat[1:1 + T * 2 * D].view(T, 2, D), flat[3 + T * 2 * D:].view(T, 2, D)
        slots = torch.arange(20, 20 + T, device="cuda")
        want_c, want_s = cache.clone(), scale.clone()
        native.kv_cache_write(want_c, k.clone(), v.clone(), slots, kv_scale=want_s)
        native.kv_cache_write(cache, k, v, slots, kv_scale=scale)
        assert torch.equal(_bytes(cache), _bytes(want_c)) and torch.equal(scale, want_s)
        table, lens = torch.ones(T, 1, device="cuda", dtype=torch.int32), torch.full((T,), 16, device="cuda", dtype=torch.int32)
        want = native.paged_decode(k.clone(), cache, table, lens, 16, kv_scale=scale)
        assert torch.equal(native.paged_decode(k, cache, table, lens, 16, kv_scale=scale), want)


def test_attention_long_cache():
    """Cache offsets past 2^32 bytes."""
    bs, Hkv, nb = 16, 8, (1 << 32) // (2 * 16 * 8 * D) + 4
    lens = [100]
    cache = torch.zeros(nb, 2, bs, Hkv, D, dtype=torch.int8, device="cuda")
    scale = torch.zeros(nb, 2, Hkv, device="cuda")
    table = torch.arange(nb - 8, nb - 1, dtype=torch.int32, device="cuda")[None]
    g = _gen(8)
    k = torch.randn(100, Hkv, D, device="cuda", generator=g).to(torch.bfloat16)
    v = torch.randn(100, Hkv, D, device="cuda", generator=g).to(torch.bfloat16)
    slots = table[0, torch.arange(100, device="cuda") // bs].long() * bs + torch.arange(100, device="cuda") % bs
    native.kv_cache_write(cache, k, v, slots, kv_scale=scale)
    q = torch.randn(1, 32, D, device="cuda", generator=g).to(torch.bfloat16)
    got = native.paged_decode(q, cache, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), 100, kv_scale=scale)
    want, tol = _exact(q, cache, scale, table, lens, D ** -0.5)
    _check(got, want, tol)
    assert int((cache[:nb - 9] != 0).sum()) == 0


# ------------------------------------------------------------------ append and attend
@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("Hq,Hkv", [(4, 4), (16, 4), (16, 1)])
@pytest.mark.parametrize("bs,split,static", [(16, 0, False), (16, 128, True), (24, 128, True), (64, 128, False), (5, 0, True)])
def test_append_is_write_then_attention(dtype, Hq, Hkv, bs, split, static):
    lens = [1, 2, 16, 17, 63, 64, 65, 128, 129, 385, 640, 1000]
    B = len(lens)
    g = _gen(Hq + bs)
    table, nb = _tables(lens, bs, g)
    cache, scale = _random_cache(nb, bs, Hkv, dtype, g)
    scale = scale * 2.0 ** -4
    wide = torch.randn(B, (Hq + 2 * Hkv) * D + 64, device="cuda", generator=g)
    wide *= torch.exp2(torch.randint(-3, 6, (B, 1), device="cuda", generator=g).float())         # some blocks' scales grow
    qkv = wide.to(torch.bfloat16)[:, :(Hq + 2 * Hkv) * D]
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    slots = torch.stack([table[i, (n - 1) // bs].long() * bs + (n - 1) % bs for i, n in enumerate(lens)])
    a_c, a_s, rot = cache.clone(), scale.clone(), qkv.clone()
    native.rope_kv_write_(rot, sl.long() - 1, slots, a_c, Hq, Hkv, 5e5, kv_scale=a_s)
    want = native.paged_decode(rot[:, :Hq * D].view(B, Hq, D), a_c, table, sl, max(lens), split_tokens=split, kv_scale=a_s)
    b_c, b_s = cache.clone(), scale.clone()
    got = native.paged_decode_rope(qkv, b_c, table, sl, slots, Hq, Hkv, max(lens), 5e5, split_tokens=split, inputs_static=static, kv_scale=b_s)
    assert torch.equal(a_s, b_s) and torch.equal(_bytes(a_c), _bytes(b_c))
    assert torch.equal(got, want)


@pytest.mark.parametrize("dtype", KINDS)
def test_append_without_a_slot(dtype):
    """A padding row attends to its newest token, in 8 bits under a scale of its own, and writes nothing."""
    lens, bs, Hq, Hkv = [1, 40, 17, 30], 16, 8, 2
    B = len(lens)
    g = _gen(9)
    table, nb = _tables(lens, bs, g)
    cache, scale = _random_cache(nb, bs, Hkv, dtype, g)
    scale = scale * 2.0 ** -4
    qkv = torch.randn(B, (Hq + 2 * Hkv) * D, device="cuda", generator=g).to(torch.bfloat16)
    sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
    before, before_s = cache.clone(), scale.clone()
    got = native.paged_decode_rope(qkv, cache, table, sl, torch.full((B,), -1, device="cuda"), Hq, Hkv, 40, 5e5, kv_scale=scale)
    assert torch.equal(_bytes(cache), _bytes(before)) and torch.equal(scale, before_s)
    rot = native.rope_qkv(qkv, sl.long() - 1, Hq, Hkv, 5e5)
    # the same with every newest token in a block of its own
    big_c, big_s = torch.cat([cache.view(torch.uint8), torch.zeros(B, 2, bs, Hkv, D, dtype=torch.uint8, device="cuda")]).view(dtype), \
        torch.cat([scale, torch.zeros(B, 2, Hkv, device="cuda")])
    native.kv_cache_write(big_c, rot[:, Hq * D:(Hq + Hkv) * D].view(B, Hkv, D), rot[:, (Hq + Hkv) * D:].view(B, Hkv, D),
                          (nb + torch.arange(B, device="cuda")) * bs, kv_scale=big_s)
    for b, n in enumerate(lens):
        val = reference.kv_values_ref(big_c, big_s)
        pages = table[b, :(n + bs - 1) // bs].long()
        kv = val[pages].transpose(0, 1).reshape(2, -1, Hkv, D)[:, :n].clone()
        kv[:, n - 1] = val[nb + b, :, 0]
        o, tol = _exact(rot[b:b + 1, :Hq * D].view(1, Hq, D), kv[None].reshape(1, 2, n, Hkv, D), torch.ones(1, 2, Hkv, device="cuda"),
                        torch.zeros(1, 1, dtype=torch.int32, device="cuda"), [n], D ** -0.5)
        _check(got[b:b + 1], o, tol)


@pytest.mark.parametrize("dtype", KINDS)
def test_captured_and_on_another_stream(dtype):
    """Two captured graphs of different shapes replayed on two streams at once give what the eager calls give."""
    g = _gen(10)
    cases = []
    for lens in ([700], [33, 1200, 5]):
        table, nb = _tables(lens, 16, g)
        cache, scale = _random_cache(nb, 16, 2, dtype, g)
        q = torch.randn(len(lens), 8, D, device="cuda", generator=g).to(torch.bfloat16)
        kv = torch.randn(len(lens), 2, 2, D, device="cuda", generator=g).to(torch.bfloat16) * 90
        sl = torch.tensor(lens, dtype=torch.int32, device="cuda")
        slots = torch.stack([table[i, (n - 1) // 16].long() * 16 + (n - 1) % 16 for i, n in enumerate(lens)])

        def step(c, s, q=q, kv=kv, table=table, sl=sl, slots=slots, longest=max(lens)):
            native.kv_cache_write(c, kv[:, 0], kv[:, 1], slots, kv_scale=s)
            return native.paged_decode(q, c, table, sl, longest, split_tokens=128, kv_scale=s)
        c0, s0 = cache.clone(), scale.clone()
        want = step(c0, s0)
        c1, s1 = cache.clone(), scale.clone()
        torch.cuda.synchronize()
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            out = step(c1, s1)
        cases.append((graph, side, out, want, c1, c0, (s1, step)))       # what the graph reads lives as long as it
    for _ in range(20):
        for graph, side, *_ in cases:
            with torch.cuda.stream(side):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, want, c1, c0, _ in cases:
        assert torch.equal(out, want) and torch.equal(_bytes(c1), _bytes(c0))


# ------------------------------------------------------------------ copies of blocks
@pytest.mark.parametrize("layers,nb,pairs,shape,dtype", [
    (1, 3, 1, (2, 16, 8, D), torch.bfloat16), (3, 50, 20, (2, 16, 2, D), torch.int8), (70, 9, 4, (5,), torch.float32),
    (2, 1000, 500, (3,), torch.uint8), (2, 40, 11, (7, 3), torch.bfloat16), (1, 900, 390, (2, 16, 1, D), torch.bfloat16)])
def test_copy_blocks(layers, nb, pairs, shape, dtype):
    g = _gen(nb)
    ts = [torch.randint(0, 100, (nb, *shape), device="cuda", generator=g).to(dtype) for _ in range(layers)]
    scales = torch.rand(nb, 2, 3, device="cuda", generator=g)
    at = torch.randperm(nb, generator=torch.Generator().manual_seed(1))[:2 * pairs].tolist()
    src = at[:pairs]
    src[-1] = src[0]                                        # one block copied twice
    pr = list(zip(src, at[pairs:]))
    want = [t.clone() for t in ts + [scales]]
    for w in want:
        w[at[pairs:]] = w[src]
    native.kv_copy_blocks_(ts + [scales], pr)
    assert all(torch.equal(a, b) for a, b in zip(ts + [scales], want))


def test_copy_blocks_refuses():
    t = torch.zeros(4, 8, device="cuda")
    for bad in ([(0, 4)], [(-1, 2)], [(0, 1), (2, 1)], [(0, 1), (1, 2)], [(3, 3)]):
        with pytest.raises(_lib.MlfError):
            native.kv_copy_blocks_([t], bad)
    native.kv_copy_blocks_([t], [])
