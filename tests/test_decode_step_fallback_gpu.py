"""An 8-bit cache on the GPU where the kernels do not go, heads of other than 128 elements and fp32 weights: the PyTorch statements serve."""
import pytest
import torch

from ml_framework_b200.models.llama import Llama, LlamaConfig
from ml_framework_b200.serving.executor import ExecutorConfig, PagedLlamaExecutor
from ml_framework_b200.serving.kv_cache import KVCacheBlockManager
from ml_framework_b200.serving.paged_attention_layer import AttentionPhase, PagedAttentionLayer
from ml_framework_b200.serving.scheduler import Batch, Request, SamplingParameters

pytestmark = pytest.mark.gpu
KINDS = [torch.float8_e4m3fn, torch.int8]


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("weights,head_dim", [(torch.bfloat16, 64), (torch.float32, 128)])
def test_executor(dtype, weights, head_dim):
    torch.manual_seed(0)
    cfg = LlamaConfig(n_layers=2, d_model=128, n_heads=4, n_kv_heads=2, head_dim=head_dim, d_ff=256, vocab_size=97, max_seq=128)
    kv = KVCacheBlockManager(300, 4, cfg.head_dim, cfg.n_layers, cfg.n_kv_heads, device="cuda", dtype=dtype)
    ex = PagedLlamaExecutor(Llama(cfg, weights, "cuda").eval(), kv, ExecutorConfig(max_seq_len=64, prefill_chunk=8))
    reqs = [Request([3] * n, id=i, sampling=s) for i, (n, s) in enumerate(((5, None), (21, SamplingParameters(0.8, 20, 0.9, seed=1))))]
    while any(r.prefilled < len(r.prompt_tokens) for r in reqs):
        for i, t in ex.execute_batch(Batch(reqs, prefill=[r for r in reqs if r.prefilled < len(r.prompt_tokens)])).generated_tokens.items():
            reqs[i].generated.append(t)
    kv.fork(1, 2)
    reqs.append(Request(list(reqs[1].prompt_tokens), id=2, generated=list(reqs[1].generated), prefilled=21, sampling=reqs[1].sampling))
    for _ in range(5):
        for i, t in ex.execute_batch(Batch(reqs, decode=reqs)).generated_tokens.items():
            reqs[i].generated.append(t)
    assert all(len(r.generated) == 6 and all(0 <= t < 97 for t in r.generated) for r in reqs)
    assert reqs[1].generated == reqs[2].generated


@pytest.mark.parametrize("dtype", KINDS)
def test_layer(dtype):
    """fp32 on the GPU against the same on the host. Rows that are rounded alike give results that differ by sums in another order; one
    whose keys lie next to a border may take a neighbouring number, half a step of 8 bits: 2^-4 of the norm."""
    torch.manual_seed(1)
    host = PagedAttentionLayer(64, 4, 2, head_dim=16, dtype=torch.float32)
    dev = PagedAttentionLayer(64, 4, 2, head_dim=16, dtype=torch.float32, device="cuda")
    dev.load_state_dict(host.state_dict())
    x = torch.randn(23, 64)
    out = []
    for layer, where in ((host, "cpu"), (dev, "cuda")):
        kv = KVCacheBlockManager(200, 4, 16, 1, 2, device=where, dtype=dtype)
        y = x.to(where)
        parts = [layer(y[:9], kv, [5], AttentionPhase.PREFILL), layer(y[9:20], kv, [5], AttentionPhase.PREFILL)]
        parts += [layer(y[i:i + 1], kv, [5], AttentionPhase.DECODE) for i in range(20, 23)]
        out.append(torch.cat(parts).cpu())
    assert (out[0] - out[1]).norm() <= 2.0 ** -4 * out[0].norm()
