"""Drawn tokens, an 8-bit cache, forks and compaction through the scheduler, the executor and the block manager on the host."""
import random

import pytest
import torch

from ml_framework_b200.models.llama import Llama, LlamaConfig
from ml_framework_b200.ops import reference
from ml_framework_b200.serving.executor import ExecutorConfig, PagedLlamaExecutor
from ml_framework_b200.serving.kv_cache import KVCacheBlockManager
from ml_framework_b200.serving.paged_attention_layer import AttentionPhase, PagedAttentionLayer
from ml_framework_b200.serving.scheduler import (CompletionConfiguration, ContinuousBatchScheduler, ContinuousBatchSchedulerClient,
                                                 GenerationOptions, Request, SamplingParameters, SchedulerConfiguration, uniform_at)

KINDS = [torch.float8_e4m3fn, torch.int8]


def _serve(dtype=torch.float32, sampling=(), prompts=4, chunk=16, graphs=False):
    torch.manual_seed(0)
    cfg = LlamaConfig(n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, head_dim=16, d_ff=96, vocab_size=97, max_seq=128)
    model = Llama(cfg, torch.float32, "cpu").eval()
    kv = KVCacheBlockManager(64, 4, cfg.head_dim, cfg.n_layers, cfg.n_kv_heads, dtype=dtype)
    ex = PagedLlamaExecutor(model, kv, ExecutorConfig(max_batch=8, max_seq_len=128, prefill_chunk=chunk))
    s = ContinuousBatchScheduler(ex, kv, SchedulerConfiguration(max_batch_size=8, warmup_iterations=0),
                                 completion=CompletionConfiguration(eos_token_id=-1, default_max_tokens=12))
    futures = [s.enqueue(Request([(7 * i + 3 * j) % 96 + 1 for j in range(5 + 9 * i)], max_tokens=12, sampling=sampling[i] if i < len(sampling) else None))
               for i in range(prompts)]
    s.run_until_idle()
    return [f.result(1).tokens for f in futures], kv


def test_draws_are_a_function_of_seed_and_position():
    hot = SamplingParameters(temperature=1.5, seed=11)
    greedy, _ = _serve()
    a, _ = _serve(sampling=[hot, None, SamplingParameters(1.5, top_k=5, seed=3)])
    b, _ = _serve(sampling=[hot, None, SamplingParameters(1.5, top_k=5, seed=3)])
    assert a == b
    assert a[1] == greedy[1] and a[3] == greedy[3] and a[0] != greedy[0]
    # temperature 0, or top_k 1, is the likeliest token
    c, _ = _serve(sampling=[SamplingParameters(0.0), SamplingParameters(2.0, top_k=1), SamplingParameters(2.0, top_p=0.0), SamplingParameters(2.0, min_p=1.0)])
    assert c == greedy
    # no seed: a seed of its own for every request
    r = [Request([1, 2], sampling=SamplingParameters(1.0)) for _ in range(4)]
    assert len({q.next_draw()[0] for q in r}) == 4 and r[0].next_draw() == r[0].next_draw()


def test_uniform_numbers():
    u = torch.tensor([uniform_at(s, p) for s in range(100) for p in range(100)], dtype=torch.float64)
    assert u.min() >= 0 and u.max() < 1 and torch.equal(u.float().double(), u)
    assert abs(u.mean() - 0.5) < 6 * (1 / 12 / 1e4) ** 0.5 and len(set(u.tolist())) > 9950
    assert 0 <= uniform_at(-5, 0) < 1 and 0 <= uniform_at(1 << 70, 1 << 40) < 1


@pytest.mark.parametrize("bad", [dict(temperature=-1.0), dict(temperature=float("nan")), dict(temperature=float("inf")), dict(top_k=-1), dict(top_k=1 << 31),
                                 dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0), dict(min_p=float("nan"))])
def test_sampling_parameters_refuse(bad):
    with pytest.raises(ValueError):
        SamplingParameters(**bad)


def test_client_passes_options_on():
    class Scheduler:
        def enqueue(self, r):
            self.r = r

    class Tok:
        def encode(self, t):
            return [1, 2, 3]
    s = Scheduler()
    c = ContinuousBatchSchedulerClient(s, Tok())
    c.submit("x")
    assert s.r.sampling is None
    c.submit("x", options=GenerationOptions(temperature=0.7, top_k=40, top_p=0.9, min_p=0.05, seed=5))
    assert s.r.sampling == SamplingParameters(0.7, 40, 0.9, 0.05, 5)


@pytest.mark.parametrize("dtype", KINDS)
@pytest.mark.parametrize("chunk", [8, 64])
def test_serving_from_eight_bits(dtype, chunk):
    """The first layer's cache holds what its rows are rounded to; tokens come out for every request."""
    toks, kv = _serve(dtype, chunk=chunk)
    assert [len(t) for t in toks] == [12] * 4
    assert kv.caches[0].dtype == dtype and kv.scales[0].shape == (64, 2, 2)
    v = reference.kv_values_ref(kv.caches[0], kv.scales[0])
    assert torch.isfinite(v).all() and float(v.abs().max()) > 0
    again, _ = _serve(dtype, chunk=chunk)
    assert again == toks


@pytest.mark.parametrize("dtype", KINDS)
def test_layer_over_eight_bits(dtype):
    """One prompt in one pass and in chunks with decode steps behind: close to the same layer over an fp32 cache, within what
    rounding keys and values to 8 bits leaves (relative 2^-4 for e4m3, half a step of a block's range for int8)."""
    torch.manual_seed(1)
    layer = PagedAttentionLayer(64, 4, 2, head_dim=16, dtype=torch.float32)
    x = torch.randn(23, 64)
    out = {}
    for t in (torch.float32, dtype):
        kv = KVCacheBlockManager(16, 4, 16, 1, 2, dtype=t)
        parts = [layer(x[:9], kv, [5], AttentionPhase.PREFILL), layer(x[9:20], kv, [5], AttentionPhase.PREFILL)]
        parts += [layer(x[i:i + 1], kv, [5], AttentionPhase.DECODE) for i in range(20, 23)]
        out[t] = torch.cat(parts)
    assert (out[dtype] - out[torch.float32]).norm() <= 2.0 ** -3 * out[torch.float32].norm()
    assert not torch.equal(out[dtype], out[torch.float32])


def _fill(m, seq):
    """Values that name the sequence, the position and the layer."""
    for layer, c in enumerate(m.caches):
        for pos in range(m.get_sequence_length(seq)):
            b = m.get_sequence_blocks(seq)[pos // m.block_size]
            c[b, :, pos % m.block_size] = float(1000 * layer + 100 * seq + pos) % 120 if c.element_size() == 1 else 1000 * layer + 100 * seq + pos
        if m.scales[layer] is not None:
            for i, b in enumerate(m.get_sequence_blocks(seq)):
                m.scales[layer][b] = 100 * seq + i


def _contents(m, seq):
    blocks, n = m.get_sequence_blocks(seq), m.get_sequence_length(seq)
    return [c[blocks].float().transpose(1, 2).reshape(-1, 2, *c.shape[3:])[:n].clone() for c in m.caches] + \
        [s[blocks].clone() for s in m.scales if s is not None]


@pytest.mark.parametrize("dtype", [torch.float32, torch.int8])
def test_compaction_keeps_every_sequence(dtype):
    rng = random.Random(2)
    m = KVCacheBlockManager(40, 4, 8, 2, 2, dtype=dtype)
    for s in range(1, 9):
        m.append_tokens(s, rng.randint(1, 18))
        _fill(m, s)
    m.fork(3, 20)                             # shared blocks move once
    m.fork(3, 21, 4)
    for s in (1, 4, 6):
        m.free_sequence_blocks(s)
    before = {s: _contents(m, s) for s in (2, 3, 5, 7, 8, 20, 21)}
    free, refs = m.free_blocks, {s: [m.reference_count(b) for b in m.get_sequence_blocks(s)] for s in before}
    moved = m.compact()
    live = 40 - free
    assert moved > 0 and m.free_blocks == free and m.compact() == 0
    assert all(b < live for s in before for b in m.get_sequence_blocks(s))
    for s, was in before.items():
        assert all(torch.equal(a, b) for a, b in zip(was, _contents(m, s)))
        assert [m.reference_count(b) for b in m.get_sequence_blocks(s)] == refs[s]
    # the pool goes on as before: a fork that appends takes a copy, freed blocks come back
    slots, cow = m.append_tokens(20, 1)
    assert (cow is not None) == (m.get_sequence_length(3) % 4 != 0) and int(slots[0]) >= 0
    assert all(torch.equal(a, b) for a, b in zip(before[3], _contents(m, 3)))
    for s in before:
        m.free_sequence_blocks(s)
    assert m.free_blocks == 40 and m.compact() == 0


def test_compaction_of_empty_and_full_pools():
    m = KVCacheBlockManager(4, 4, 8, 1, 1)
    assert m.compact() == 0
    m.append_tokens(1, 16)
    assert m.compact() == 0 and m.get_sequence_blocks(1) == [0, 1, 2, 3]


def test_copy_on_write_takes_the_scales_along():
    m = KVCacheBlockManager(8, 4, 8, 2, 2, dtype=torch.int8)
    m.append_tokens(1, 6)
    _fill(m, 1)
    m.fork(1, 2)
    was = _contents(m, 1)
    _, cow = m.append_tokens(2, 1)
    src, dst = cow
    for c, s in zip(m.caches, m.scales):
        assert torch.equal(c[src], c[dst]) and torch.equal(s[src], s[dst])
    assert all(torch.equal(a, b) for a, b in zip(was, _contents(m, 1)))


def test_a_following_rank_draws_the_same_tokens():
    """The leader's plan says how each next token is drawn: an executor that follows it fills its cache alike."""
    import copy

    from ml_framework_b200.serving.tp_driver import TPLeaderExecutor, follower_loop

    class Wire:
        def __init__(self):
            self.plans = []

        def broadcast_object(self, plan, src):
            if plan is not None or self.sending:
                self.plans.append(copy.deepcopy(plan))
                return plan
            return self.plans.pop(0)
    wire = Wire()
    sides = []
    for _ in range(2):
        torch.manual_seed(0)
        cfg = LlamaConfig(n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, head_dim=16, d_ff=96, vocab_size=97, max_seq=128)
        model = Llama(cfg, torch.float32, "cpu").eval()
        kv = KVCacheBlockManager(64, 4, cfg.head_dim, cfg.n_layers, cfg.n_kv_heads, dtype=torch.int8)
        ex = PagedLlamaExecutor(model, kv, ExecutorConfig(max_batch=8, max_seq_len=128, prefill_chunk=8))
        seen = []
        ex._draws = (lambda inner, seen: lambda reqs, rows: (lambda d: (seen.append(None if d is None else d.tolist()), d)[1])(inner(reqs, rows)))(ex._draws, seen)
        sides.append((ex, kv, seen))
    wire.sending = True
    leader = TPLeaderExecutor(sides[0][0], wire)
    s = ContinuousBatchScheduler(leader, sides[0][1], SchedulerConfiguration(max_batch_size=8, warmup_iterations=0),
                                 completion=CompletionConfiguration(eos_token_id=-1, default_max_tokens=6))
    leader.live_ids_fn = lambda: [q.id for q in s.batch_manager.running]
    for i, p in enumerate((SamplingParameters(1.2, 30, 0.9), None, SamplingParameters(0.9))):
        s.enqueue(Request([(7 * i + j) % 96 + 1 for j in range(5 + 6 * i)], max_tokens=6, sampling=p))
    s.run_until_idle()
    leader.shutdown()
    wire.sending = False
    follower_loop(sides[1][0], wire)
    (_, a, drawn), (_, b, followed) = sides
    assert drawn == followed and any(d is not None for d in drawn)
    assert all(torch.equal(x, y) for x, y in zip(a.caches + a.scales, b.caches + b.scales))
