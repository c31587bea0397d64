"""What the calls over an 8-bit cache and the copies of blocks refuse (none of it reaches a kernel), and the PyTorch statement of
a write on the host."""
import pytest
import torch

from ml_framework_b200.ops import native, reference

E4, I8, BF = torch.float8_e4m3fn, torch.int8, torch.bfloat16


def _cache(dtype=I8, nb=4, bs=16, H=2):
    return torch.zeros(nb, 2, bs, H, 128, dtype=torch.uint8).view(dtype), torch.ones(nb, 2, H)


def _decode(cache, scale, B=3, Hq=4, lens=None, table=None, q=None, **kw):
    return native.paged_decode(torch.zeros(B, Hq, 128, dtype=BF) if q is None else q, cache, torch.zeros(B, 2, dtype=torch.int32) if table is None else table,
                               torch.ones(B, dtype=torch.int32) if lens is None else lens, 32, kv_scale=scale, **kw)


@pytest.mark.parametrize("dtype", [E4, I8])
def test_attention_refuses(dtype):
    c, s = _cache(dtype)
    with pytest.raises(ValueError, match="needs kv_scale"):
        _decode(c, None)
    with pytest.raises(ValueError, match="kv_scale must be"):
        _decode(c, s[:3])
    with pytest.raises(ValueError, match="kv_scale must be"):
        _decode(c, s.double())
    with pytest.raises(TypeError):
        _decode(torch.zeros(4, 2, 16, 2, 128, dtype=BF), s)
    with pytest.raises(ValueError, match="cache must be"):
        _decode(torch.zeros(4, 2, 16, 2, 64, dtype=I8), s)
    with pytest.raises(ValueError, match="groups of 1 to 16"):
        _decode(c, s, Hq=3)
    with pytest.raises(ValueError, match="groups of 1 to 16"):
        _decode(c, s, Hq=34)
    with pytest.raises(ValueError, match="seq_lens"):
        _decode(c, s, lens=torch.ones(3, dtype=torch.int64))
    with pytest.raises(ValueError, match="block_table"):
        _decode(c, s, table=torch.zeros(2, 2, dtype=torch.int32))
    with pytest.raises(ValueError, match="bfloat16"):
        _decode(c, s, q=torch.zeros(3, 4, 128))
    with pytest.raises(ValueError, match="current CUDA device"):
        _decode(c, s)


def test_no_heads_are_refused():
    for H, Hq in ((0, 4), (2, 0), (0, 0)):
        c, s = _cache(H=H)
        with pytest.raises(ValueError, match="groups of 1 to 16"):
            _decode(c, s, Hq=Hq)
        with pytest.raises(ValueError):
            native.paged_decode_rope(torch.zeros(3, (Hq + 2 * H) * 128, dtype=BF), c, torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32),
                                     torch.zeros(3, dtype=torch.int64), Hq, H, 32, 1e4, kv_scale=s)


def test_append_refuses():
    c, s = _cache()
    qkv, table, lens, slots = torch.zeros(3, 8 * 128, dtype=BF), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
    call = lambda qkv=qkv, slots=slots, theta=1e4, **kw: native.paged_decode_rope(qkv, c, table, lens, slots, 4, 2, 32, theta, kv_scale=s, **kw)   # noqa: E731
    with pytest.raises(ValueError, match="qkv must be"):
        call(qkv=qkv[:, :-128])
    with pytest.raises(ValueError, match="theta"):
        call(theta=0.0)
    with pytest.raises(ValueError, match="slots"):
        call(slots=slots.int())
    with pytest.raises(ValueError, match="inputs_static"):
        call(slots=torch.zeros(6, dtype=torch.int64)[::2], inputs_static=True)
    with pytest.raises(ValueError, match="current CUDA device"):
        call()


def test_write_and_gather_refuse():
    c, s = _cache()
    k = torch.zeros(3, 2, 128, dtype=BF)
    slots = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(ValueError, match="k must be"):
        native.kv_cache_write(c, k[:, :1], k, slots, s)
    with pytest.raises(ValueError, match="values"):
        native.kv_cache_write(c, k, k[:2], slots, s)
    with pytest.raises(ValueError, match="slots"):
        native.kv_cache_write(c, k, k, slots[:2], s)
    with pytest.raises(ValueError, match="needs kv_scale"):
        native.kv_cache_write(c, k, k, slots)
    with pytest.raises(ValueError, match="16-byte"):
        native.rope_kv_write_(torch.zeros(3, 8 * 128 + 4, dtype=BF)[:, 4:], slots, slots, c, 4, 2, 1e4, s)
    with pytest.raises(ValueError, match="entries"):
        native.kv_gather(c, torch.zeros(2, dtype=torch.int32), 33, s)
    with pytest.raises(ValueError, match="current CUDA device"):
        native.kv_cache_write(c, k, k, slots, s)
    with pytest.raises(ValueError, match="current CUDA device"):
        native.kv_gather(c, torch.zeros(2, dtype=torch.int32), 32, s)


def test_copies_refuse():
    with pytest.raises(ValueError, match="same number of blocks"):
        native.kv_copy_blocks_([torch.zeros(4, 2), torch.zeros(5, 2)], [(0, 1)])
    with pytest.raises(ValueError, match="same number of blocks"):
        native.kv_copy_blocks_([torch.zeros(4, 4)[:, :2]], [(0, 1)])
    with pytest.raises(ValueError, match="block numbers"):
        native.kv_copy_blocks_([torch.zeros(4, 2)], [(0, 1, 2)])
    with pytest.raises(ValueError, match="current CUDA device"):
        native.kv_copy_blocks_([torch.zeros(4, 2)], [(0, 1)])


@pytest.mark.parametrize("dtype,top", [(E4, 448.0), (I8, 127.0)])
def test_scales_are_the_smallest_that_fit(dtype, top):
    amax = torch.tensor([0.0, 1e-30, top * 2.0 ** -40, top * 0.999, top, top * 1.01, 1.0, 1e30, float("inf")])
    s = reference.q8_scale_ref(amax, dtype)
    assert torch.equal(torch.log2(s), torch.log2(s).round())
    for a, x in zip(amax.tolist(), s.tolist()):
        assert 2.0 ** -40 <= x <= 2.0 ** 40
        assert a <= top * x or x == 2.0 ** 40
        assert a > top * x / 2 or x == 2.0 ** -40


@pytest.mark.parametrize("dtype", [E4, I8])
def test_values_come_back_within_half_a_step(dtype):
    """Rows appended one at a time, growing: a held value is rounded once for every scale that its block has had, each time by half
    a step at most, and the steps double: less than one step of the last scale (e4m3: 2^-4 of the value, or half of 2^-9 of a
    scale, each time)."""
    torch.manual_seed(0)
    c, s = _cache(dtype, nb=1)
    rows = torch.randn(16, 2, 128) * torch.exp2(torch.arange(16.0) / 4)[:, None, None]
    for i in range(16):
        reference.kv_write_ref(c, rows[i:i + 1].to(BF), rows[i:i + 1].to(BF), torch.tensor([i]), s)
    got = reference.kv_values_ref(c, s)[0, 0]
    want = rows.to(BF).float()
    step = s[0, 0][None, :, None]
    err = (got - want).abs()
    if dtype == I8:
        assert (err <= step).all()
    else:
        assert (err <= 2.0 ** -4 * want.abs() + 2.0 ** -9 * step).all()


def test_argument_types_follow_the_entries():
    """The letters with which an entry is called name the types that its C++ definition has."""
    import re
    from pathlib import Path

    import ml_framework_b200
    root = Path(ml_framework_b200.__file__).parent
    source = "\n".join(p.read_text() for p in sorted((root / "csrc").rglob("*.cu")))
    calls = re.findall(r'_function\("(\w+)", "(\w+)"\)\(', (root / "ops" / "native.py").read_text())
    assert len(calls) >= 5
    for name, letters in calls:
        args = re.search(r"MLF_API int " + name + r"\(([^)]*)\)\s*\{", source).group(1).split(",")
        want = "".join("p" if "*" in a else "u" if "uint64_t" in a else "l" if "long long" in a else "f" if "float" in a else "i" for a in args)
        assert letters == want, name


def test_splits_fill_one_round_at_most():
    for pairs in (1, 2, 8, 31, 32, 104, 128, 200, 222, 223, 296, 297, 444, 512, 10000):
        for n in (0, 1, 128, 384, 385, 700, 1024, 2500, 4000, 60001, 1 << 20):
            splits = native._decode_splits_q8(pairs, n, 148)
            assert 1 <= splits <= 96 and (splits == 1 or (splits * pairs <= (592 if splits == 2 and n >= 1500 else 444) and n > 384 and -(-n // splits) >= 87))
            assert splits == 1 or n // 128 >= splits - 1
            assert native._decode_splits_q8(pairs, n, 148, 2, False) * pairs <= max(pairs, 296)
    assert native._decode_splits_q8(256, 4096, 148) == 2 and native._decode_splits_q8(256, 1000, 148) == 1
    assert native._decode_splits_q8(8, 4000, 148) == 16 and native._decode_splits_q8(512, 4000, 148) == 1
