"""Worker for test_serve_draws_tp_cpu (one gloo process per rank): a tensor-parallel Llama on the host serves requests of which some
draw their tokens. Every rank settles the next tokens from the gathered logits, and all of them alike."""
import json
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def main():
    from ml_framework_b200.dist.process_group import destroy_process_group, init_process_group
    from ml_framework_b200.models.llama import LlamaConfig
    from ml_framework_b200.models.llama_tp import LlamaTP
    from ml_framework_b200.ops import reference
    from ml_framework_b200.parallel.tensor_parallel import TPContext
    from ml_framework_b200.serving.executor import ExecutorConfig, PagedLlamaExecutor
    from ml_framework_b200.serving.kv_cache import KVCacheBlockManager
    from ml_framework_b200.serving.scheduler import (BatchConstraints, CompletionConfiguration, ContinuousBatchScheduler, Request, SamplingParameters,
                                                     SchedulerConfiguration)
    from ml_framework_b200.serving.tp_driver import TPLeaderExecutor, follower_loop
    torch.set_num_threads(1)
    pg = init_process_group("gloo")
    W, r = pg.world_size, pg.rank
    # a vocabulary that fills neither rank's share of the padded head to its end
    cfg = LlamaConfig(n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, head_dim=16, d_ff=96, vocab_size=300, max_seq=128)
    hot = [SamplingParameters(1.5, 30, 0.95, 0.01, seed=5), None, SamplingParameters(0.9, seed=9), SamplingParameters(3.0, top_p=0.9, seed=1), SamplingParameters(2.0, top_k=1)]
    outs = []
    for dtype in (torch.float32, torch.int8):
        for sampling in (hot, [None] * 5):
            torch.manual_seed(100 + r)
            tp = TPContext(pg, None, False)
            model = LlamaTP(cfg, tp, sequence_parallel=False, dtype=torch.float32, device="cpu").eval()
            with torch.no_grad():
                model.lm_head.mul_(20.0)                 # logits that differ
            for p in model.replicated_parameters():
                pg.broadcast(p.data, src=0)
            kv = KVCacheBlockManager(64, 4, cfg.head_dim, cfg.n_layers, cfg.n_kv_heads // W, dtype=dtype)
            ex = PagedLlamaExecutor(model, kv, ExecutorConfig(max_batch=8, max_seq_len=128, prefill_chunk=16), tp=tp)
            seen = []
            inner = ex._logits_draw

            def draw(logits, draws):
                """The executor's draw, checked against the statement over the shares put together, and noted."""
                got = inner(logits, draws)
                full = torch.cat(pg.all_gather_object(logits), -1)
                assert full.shape[1] > cfg.vocab_size > logits.shape[1]
                u, t, p, m = draws[:4].view(torch.float32)
                assert torch.equal(got, reference.sample_ref(full, cfg.vocab_size, u, t, draws[4], p, m)[0])
                seen.append((got.tolist(), draws.tolist()))
                return got
            ex._logits_draw = draw
            if r == 0:
                leader = TPLeaderExecutor(ex, pg)
                sched = ContinuousBatchScheduler(leader, kv, SchedulerConfiguration(max_batch_size=8, warmup_iterations=0), BatchConstraints(max_batch_size=8),
                                                 completion=CompletionConfiguration(eos_token_id=-1, default_max_tokens=8))
                leader.live_ids_fn = lambda: [q.id for q in sched.batch_manager.running]
                futs = [sched.enqueue(Request([(11 * i + 5 * j) % 299 + 1 for j in range(5 + 9 * i)], max_tokens=8, sampling=s)) for i, s in enumerate(sampling)]
                sched.run_until_idle()
                leader.shutdown()
                outs.append([f.result(1).tokens for f in futs])
            else:
                assert follower_loop(ex, pg) > 0
            both = pg.all_gather_object(seen)
            assert both[0] == both[1] and bool(seen) == (sampling is hot)
    if r == 0:
        print(json.dumps({"tokens": outs}))
    destroy_process_group()


if __name__ == "__main__":
    main()
