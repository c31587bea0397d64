"""The operators of a decode step together, as the executor runs them: an 8-bit cache, drawn tokens, forks, compaction."""
import pytest
import torch

from ml_framework_b200.models.llama import Llama, LlamaConfig
from ml_framework_b200.ops import native, reference
from ml_framework_b200.serving.executor import ExecutorConfig, PagedLlamaExecutor
from ml_framework_b200.serving.kv_cache import KVCacheBlockManager
from ml_framework_b200.serving.paged_attention_layer import AttentionPhase, PagedAttentionLayer
from ml_framework_b200.serving.scheduler import Batch, Request, SamplingParameters

pytestmark = pytest.mark.gpu
KINDS = [torch.float8_e4m3fn, torch.int8]


def _executor(dtype, graphs=True, chunk=64, blocks=300, bs=16):
    torch.manual_seed(5)
    cfg = LlamaConfig(2, 512, 4, 2, 128, 1024, 500, 2048)
    m = Llama(cfg, torch.bfloat16, "cuda").eval()
    with torch.no_grad():                     # tokens with a clear winner: the head points from each token to the next one
        m.embed.weight.normal_(0, 1)
        m.lm_head.copy_(m.embed.weight.roll(1, 0) * 0.05)
    kv = KVCacheBlockManager(blocks, bs, 128, cfg.n_layers, cfg.n_kv_heads, device="cuda", dtype=dtype)
    return PagedLlamaExecutor(m, kv, ExecutorConfig(max_seq_len=1024, prefill_chunk=chunk, use_cuda_graphs=graphs)), kv


def _run(ex, reqs, steps, between=None):
    while any(r.prefilled < len(r.prompt_tokens) for r in reqs):
        todo = [r for r in reqs if r.prefilled < len(r.prompt_tokens)]
        for i, t in ex.execute_batch(Batch(reqs, prefill=todo)).generated_tokens.items():
            next(r for r in reqs if r.id == i).generated.append(t)
    for s in range(steps):
        if between:
            between(s)
        out = ex.execute_batch(Batch(reqs, decode=reqs)).generated_tokens
        for r in reqs:
            r.generated.append(out[r.id])
    return [r.generated for r in reqs]


def _requests(lens, **kw):
    return [Request([(11 * i + 5 * j) % 499 + 1 for j in range(n)], id=100 + i, **kw) for i, n in enumerate(lens)]


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("bs", [16, 32, 12])
def test_first_layer_holds_the_rounded_rows(dtype, bs):
    """Keys and values of the first layer follow from the tokens alone: the 8-bit cache holds, bit for bit, what the rows of a bf16
    cache filled by the same tokens are rounded to in the same calls."""
    lens, steps = [5, 40, 130, 64], 20
    want_ex, want_kv = _executor(torch.bfloat16, False, bs=bs)
    reqs = _requests(lens)
    tokens = _run(want_ex, reqs, steps)
    ex, kv = _executor(dtype, False, bs=bs)
    got = _requests(lens)
    for r in got:                             # the same tokens, whatever the 8-bit model would have said
        while r.prefilled < len(r.prompt_tokens):
            ex.execute_batch(Batch(got, prefill=[r]))
    for s in range(steps):
        for r, t in zip(got, tokens):
            r.generated.append(t[s])
        ex.execute_batch(Batch(got, decode=got))
    for r, n in zip(got, lens):
        blocks, theirs = kv.get_sequence_blocks(r.id), want_kv.get_sequence_blocks(r.id)
        rows = want_kv.caches[0][theirs].transpose(1, 2).reshape(-1, 2, 2, 128)
        total = n + steps
        c = torch.zeros(len(blocks), 2, bs, 2, 128, device="cuda").to(dtype)
        s = torch.zeros(len(blocks), 2, 2, device="cuda")
        calls = [(a, min(a + 64, n)) for a in range(0, n, 64)] + [(i, i + 1) for i in range(n, total)]
        for a, b in calls:
            reference.kv_write_ref(c, rows[a:b, 0], rows[a:b, 1], torch.arange(a, b, device="cuda"), s)
        assert torch.equal(kv.scales[0][blocks], s)
        flat = lambda t: t.view(torch.uint8).transpose(1, 2).reshape(-1, 2, 2, 128)[:total]       # noqa: E731
        assert torch.equal(flat(kv.caches[0][blocks]), flat(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16] + KINDS)
@pytest.mark.parametrize("drawn", [False, True])
def test_graphs_and_launches_agree(dtype, drawn):
    """Prompts and decode steps replayed from captured graphs give the tokens of the same steps launched one by one, with and
    without drawing, also where only some of the requests draw."""
    lens = [5, 33, 70]
    sampling = [SamplingParameters(0.8, 20, 0.95, 0.01, seed=4), None, SamplingParameters(1.3, seed=9)] if drawn else [None] * 3
    outs = []
    for graphs in (True, False):
        ex, kv = _executor(dtype, graphs)
        for turn in range(3):
            reqs = _requests(lens)
            for r, s in zip(reqs, sampling):
                r.sampling = s
            outs.append(_run(ex, reqs, 12))
            for r in reqs:
                kv.free_sequence_blocks(r.id)
    assert all(o == outs[0] for o in outs)
    if drawn:
        assert outs[0][1] != outs[0][0]


@pytest.mark.parametrize("dtype", [torch.bfloat16] + KINDS)
def test_forks_and_compaction_change_no_token(dtype):
    """A sequence forked after its prompt goes on like one that had the prompt to itself, beside its parent; a pool that is compacted
    between steps gives the tokens of one that is not."""
    outs = []
    for disturbed in (False, True):
        ex, kv = _executor(dtype)
        filler = Request([3] * 100, id=1)
        _run(ex, [filler], 0)
        reqs = _requests([21, 37])
        _run(ex, reqs, 0)
        if disturbed:
            kv.fork(100, 900)
            child = Request(list(reqs[0].prompt_tokens), id=900, generated=list(reqs[0].generated), prefilled=21)
        else:
            child = Request(list(reqs[0].prompt_tokens), id=900)
            _run(ex, [child], 0)

        def between(step):
            if disturbed and step == 3:
                kv.free_sequence_blocks(1)
                assert kv.compact() > 0
        outs.append(_run(ex, reqs + [child], 10, between))
    assert outs[0] == outs[1] and outs[1][0] == outs[1][2]


@pytest.mark.parametrize("dtype", KINDS)
def test_layer_like_its_float_statement(dtype):
    """The layer over an 8-bit cache on the GPU, against the same layer over the values that the cache ends up with: prompt in
    two chunks, then single tokens. Attention over equal values differs by bf16 roundings between operators: 2^-6 of the norm."""
    torch.manual_seed(2)
    layer = PagedAttentionLayer(512, 8, 2, head_dim=128, dtype=torch.bfloat16, device="cuda")
    x = torch.randn(60, 512, device="cuda").to(torch.bfloat16)
    kv = KVCacheBlockManager(16, 16, 128, 1, 2, device="cuda", dtype=dtype)
    with torch.no_grad():
        layer(x[:30], kv, [5], AttentionPhase.PREFILL)
        chunk = layer(x[30:50], kv, [5], AttentionPhase.PREFILL)
        qkv = torch.nn.functional.linear(x[30:50].float(), layer.qkv.weight.float())
        q = reference.rope_ref(qkv[:, :8 * 128].view(20, 8, 128), torch.arange(30, 50, device="cuda"), 5e5)
        k, v = native.kv_gather(kv.caches[0], torch.tensor(kv.get_sequence_blocks(5), dtype=torch.int32, device="cuda"), 50, kv_scale=kv.scales[0])
        o, _ = reference.attention_ref(q[None].float(), k[None].float(), v[None].float(), causal=True, start_pos=30)
        want = o[0].reshape(20, -1) @ layer.proj.weight.float().t()
        assert (chunk.float() - want).norm() <= 2.0 ** -6 * want.norm()
        for i in range(50, 60):
            one = layer(x[i:i + 1], kv, [5], AttentionPhase.DECODE)
            qkv = torch.nn.functional.linear(x[i:i + 1].float(), layer.qkv.weight.float())
            q = reference.rope_ref(qkv[:, :8 * 128].view(1, 8, 128), torch.tensor([i], device="cuda"), 5e5)
            k, v = native.kv_gather(kv.caches[0], torch.tensor(kv.get_sequence_blocks(5), dtype=torch.int32, device="cuda"), i + 1, kv_scale=kv.scales[0])
            o, _ = reference.attention_ref(q[None].float(), k[None].float(), v[None].float(), causal=False)
            want = o[0].reshape(1, -1) @ layer.proj.weight.float().t()
            assert (one.float() - want).norm() <= 2.0 ** -6 * want.norm()
