"""Settings of drawn tokens of other types than their own: refused where a request is made, so that no step of a batch meets them."""
import numpy as np
import pytest
import torch

from ml_framework_b200.models.llama import Llama, LlamaConfig
from ml_framework_b200.serving.executor import ExecutorConfig, PagedLlamaExecutor
from ml_framework_b200.serving.kv_cache import KVCacheBlockManager
from ml_framework_b200.serving.scheduler import Batch, GenerationOptions, Request, SamplingParameters


@pytest.mark.parametrize("bad", [dict(top_k=50.5), dict(top_k=50.0), dict(top_k="5"), dict(top_k=None), dict(seed=1.5), dict(seed="7"), dict(temperature="1"),
                                 dict(temperature=None), dict(top_p="0.9"), dict(min_p=None), dict(temperature=1j)])
def test_other_types_are_refused(bad):
    with pytest.raises(TypeError):
        SamplingParameters(**bad)
    if bad.get("temperature", 1.0):
        with pytest.raises(TypeError):
            GenerationOptions(**{"temperature": 1.0, **bad}).sampling()


def test_numbers_of_other_libraries_are_taken_for_what_they_are():
    s = SamplingParameters(np.float32(0.5), np.int64(40), torch.tensor(0.75), 1, np.uint32(9))
    assert s == SamplingParameters(0.5, 40, 0.75, 1.0, 9)
    assert [type(v) for v in (s.temperature, s.top_k, s.top_p, s.min_p, s.seed)] == [float, int, float, float, int]


def test_a_step_takes_what_was_accepted():
    torch.manual_seed(0)
    cfg = LlamaConfig(n_layers=1, d_model=32, n_heads=2, n_kv_heads=1, head_dim=16, d_ff=48, vocab_size=31, max_seq=64)
    kv = KVCacheBlockManager(16, 4, cfg.head_dim, cfg.n_layers, cfg.n_kv_heads)
    ex = PagedLlamaExecutor(Llama(cfg, torch.float32, "cpu").eval(), kv, ExecutorConfig(max_seq_len=32))
    reqs = [Request([1, 2], id=1, sampling=SamplingParameters(np.float64(1e300), np.int32(3), 1, True, -1)), Request([3], id=2)]
    out = ex.execute_batch(Batch(reqs, prefill=reqs)).generated_tokens
    assert sorted(out) == [1, 2] and all(0 <= t < 31 for t in out.values())
