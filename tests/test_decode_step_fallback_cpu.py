"""An 8-bit cache where the operators' PyTorch statements run: what they convert is the blocks that the call's tables name, not the pool."""
import pytest
import torch

from ml_framework_b200.models.llama import Llama, LlamaConfig
from ml_framework_b200.ops import reference
from ml_framework_b200.serving.executor import ExecutorConfig, PagedLlamaExecutor
from ml_framework_b200.serving.kv_cache import KVCacheBlockManager
from ml_framework_b200.serving.paged_attention_layer import AttentionPhase, PagedAttentionLayer
from ml_framework_b200.serving.scheduler import Batch, Request

KINDS = [torch.float8_e4m3fn, torch.int8]
POOL = 500


@pytest.fixture
def converted(monkeypatch):
    """Blocks that each conversion to floating point was handed."""
    seen = []
    inner = reference.kv_values_ref

    def note(cache, scale):
        seen.append(cache.shape[0])
        return inner(cache, scale)
    monkeypatch.setattr(reference, "kv_values_ref", note)
    return seen


@pytest.mark.parametrize("dtype", KINDS)
def test_executor_converts_the_blocks_in_use(converted, dtype):
    torch.manual_seed(0)
    cfg = LlamaConfig(n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, head_dim=16, d_ff=96, vocab_size=97, max_seq=128)
    kv = KVCacheBlockManager(POOL, 4, cfg.head_dim, cfg.n_layers, cfg.n_kv_heads, dtype=dtype)
    ex = PagedLlamaExecutor(Llama(cfg, torch.float32, "cpu").eval(), kv, ExecutorConfig(max_seq_len=64, prefill_chunk=8))
    reqs = [Request([3] * n, id=i) for i, n in enumerate((5, 21))]
    while any(r.prefilled < len(r.prompt_tokens) for r in reqs):
        ex.execute_batch(Batch(reqs, prefill=[r for r in reqs if r.prefilled < len(r.prompt_tokens)]))
    for r in reqs:
        r.generated.append(1)
    ex.execute_batch(Batch(reqs, decode=reqs))
    assert converted and max(converted) <= kv.blocks_needed(22)


@pytest.mark.parametrize("dtype", [torch.float32] + KINDS)
def test_layer_converts_the_blocks_in_use(converted, dtype):
    torch.manual_seed(1)
    layer = PagedAttentionLayer(64, 4, 2, head_dim=16, dtype=torch.float32)
    kv = KVCacheBlockManager(POOL, 4, 16, 1, 2, dtype=dtype)
    x = torch.randn(14, 64)
    layer(x[:9], kv, [5], AttentionPhase.PREFILL)
    layer(x[9:13], kv, [5], AttentionPhase.PREFILL)
    layer(x[13:], kv, [5], AttentionPhase.DECODE)
    assert converted and max(converted) <= kv.blocks_needed(14)


@pytest.mark.parametrize("dtype", KINDS)
def test_attention_over_pages_is_attention_over_the_values(dtype):
    """The statement with scales gives what it gives over the pool's values, number for number."""
    torch.manual_seed(2)
    cache = reference.q8_round_ref(torch.randn(12, 2, 4, 2, 16) * 60, dtype)
    scale = torch.exp2(torch.randint(-9, 3, (12, 2, 2)).float())
    table = torch.randperm(12)[:9].view(3, 3).to(torch.int32)
    q, lens = torch.randn(3, 4, 16), [12, 1, 6]
    want = reference.paged_attention_ref(q, reference.kv_values_ref(cache, scale), table, lens)
    assert torch.equal(reference.paged_attention_ref(q, cache, table, lens, kv_scale=scale), want)
