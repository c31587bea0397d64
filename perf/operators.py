"""Operators of a decode step, measured through the calls that a serving program makes of them.

``decode``  one query token per sequence against a paged cache whose keys and values are held in 8 bits (e4m3 or int8) with a
            scale for each block of tokens and head: ``native.paged_decode(..., kv_scale=...)``.
``write``   new keys and values into that cache and the sequence's values back out of it, what a later chunk of a prompt
            attends to: ``native.kv_cache_write(..., kv_scale=...)`` and ``native.kv_gather(..., kv_scale=...)``.
``copy``    blocks of a cache to other places, over all layers: forked sequences that diverge, compaction
            (``native.kv_copy_blocks_``).
``sample``  the next tokens from logits and given random numbers: temperature, top-k, top-p and min-p of each row
            (``native.sample_rows``).

Cache layout: ``[blocks, 2 (K, V), tokens of a block, KV heads, 128]`` and scales ``[blocks, 2, KV heads]``; a value is its 8-bit
number times its scale. The scale of a block and head is the smallest power of two (from 2^-40 to 2^40) under which the largest
magnitude written there fits (448 for e4m3, 127 for int8). A write to a block's first row starts the block anew; one to later
rows keeps the larger of the old scale and the new rows' own, and rounds what the block held to the larger scale.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

D = 128                     # head dimension of every preset
PAGE = 16                   # tokens per block


# ------------------------------------------------------------------------------------------ the cases
def _decode(kind, batch, tokens, heads, kv_heads):
    return {"op": "decode", "kind": kind, "batch": batch, "tokens": tokens, "heads": heads, "kv_heads": kv_heads}


def _write(kind, prefix, tokens, kv_heads):
    return {"op": "write", "kind": kind, "prefix": prefix, "tokens": tokens, "kv_heads": kv_heads}


def _copy(layers, blocks, pairs, kv_heads):
    return {"op": "copy", "layers": layers, "blocks": blocks, "pairs": pairs, "kv_heads": kv_heads}


def _sample(rows, vocab, dtype, mode):
    return {"op": "sample", "rows": rows, "vocab": vocab, "dtype": dtype, "mode": mode}


def listed():
    return [
        # A single user's chat: latency per token.
        dict(_decode("e4m3", 1, 700, 32, 8), name="decode e4m3 1x700"),
        # A moderate, odd batch with longer contexts.
        dict(_decode("int8", 13, 2500, 32, 8), name="decode int8 13x2500"),
        # The serving benchmark's batch.
        dict(_decode("e4m3", 64, 576, 32, 8), name="decode e4m3 64x576"),
        # Multi-head attention without grouping.
        dict(_decode("int8", 24, 900, 40, 40), name="decode int8 mha 24x900"),
        # Few sequences with very long contexts: the longest of them decides.
        dict(_decode("e4m3", 4, 60001, 32, 8), name="decode e4m3 4x60001"),
        # A short chat turn enters the cache.
        dict(_write("e4m3", 0, 37, 8), name="write e4m3 37"),
        # A later chunk of a long prompt, behind a prefix that ends inside a block.
        dict(_write("int8", 1111, 2048, 8), name="write int8 1111+2048"),
        # A forked sequence appends its first token: its last block is copied in every layer.
        dict(_copy(32, 128, 1, 8), name="copy 32 layers 1 block"),
        # Compaction of a cache after many requests have ended.
        dict(_copy(8, 1500, 700, 8), name="copy 8 layers 700 blocks"),
        # A single user: top-k and top-p, the usual settings of a chat.
        dict(_sample(1, 128256, "bf16", "chat"), name="sample 1x128256"),
        # A moderate batch, each request with settings of its own, in fp32.
        dict(_sample(33, 50257, "fp32", "mixed"), name="sample fp32 33x50257"),
        # The largest batch that the executor takes by default.
        dict(_sample(256, 128256, "bf16", "mixed"), name="sample 256x128256"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("decode", "decode", "write", "copy", "sample", "sample"))
    if op == "decode":
        heads, kv_heads = rng.choice(((32, 8), (32, 8), (40, 40), (16, 4), (8, 1), (12, 4), (16, 1)))
        batch = _log(rng, 1, 256)
        return _decode(rng.choice(("e4m3", "int8")), batch, _log(rng, 1, max(2, min(60000, 1800000 // (batch * kv_heads)))), heads, kv_heads)
    if op == "write":
        return _write(rng.choice(("e4m3", "int8")), rng.choice((0, _log(rng, 1, 4000))), _log(rng, 1, 4096), rng.choice((1, 4, 8, 8)))
    if op == "copy":
        layers, pairs = rng.choice((1, 4, 8, 32)), _log(rng, 1, 160)
        return _copy(layers, 2 * pairs + rng.randint(1, 60), pairs, rng.choice((1, 4, 8)))
    rows = _log(rng, 1, 256)
    vocab = rng.choice((1000, 32000, 50257, 128256, _log(rng, 2, 128000)))
    return _sample(rows, vocab, rng.choice(("bf16", "bf16", "fp32")), rng.choice(("chat", "plain", "mixed", "nucleus")))


# ------------------------------------------------------------------------------------------ inputs from the seed
def _gen(seed, salt=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed * 1000003 + salt)
    return g


def _pages(n):
    return (n + PAGE - 1) // PAGE


def _lengths(c):
    """Cached tokens of each sequence: from half of ``tokens`` up to it."""
    n = c["tokens"]
    return [n - (i * 37) % (n // 2 + 1) for i in range(c["batch"])]


def _exponent(amax, kind):
    """The scale's exponent: the smallest under which ``amax`` fits."""
    frac, e = torch.frexp(amax.float())
    top, bits = (448.0 / 512.0, 9) if kind == "e4m3" else (127.0 / 128.0, 7)
    e = torch.where(frac <= top, e - bits, e - bits + 1)
    return torch.where(amax == 0, torch.full_like(e, -40), e).clamp(-40, 40)


def _round8(x, kind):
    """Numbers in units of their scale, rounded to 8 bits (ties to even), as the values that these stand for."""
    if kind == "e4m3":
        return x.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    return x.round().clamp(-127.0, 127.0)


def _bytes_of(x, kind):
    return x.to(torch.float8_e4m3fn) if kind == "e4m3" else x.to(torch.int8)


def _rows(cache, at):
    """``cache.flatten(...)[at]`` as fp32, also where indexing does not know the 8-bit type."""
    return cache.view(torch.uint8)[at].view(cache.dtype).float()


def _outliers(t, seed, salt):
    """Channels of keys that are several times as large as the others."""
    return t * (1.0 + 7.0 * (torch.rand(t.shape[-2], D, generator=_gen(seed, salt), device="cuda") < 0.03).to(t.dtype))


def _cache(blocks, kv_heads, kind, seed):
    x = torch.randn(blocks, 2, PAGE, kv_heads, D, generator=_gen(seed, 1), device="cuda")
    x[:, 0] = _outliers(x[:, 0], seed, 2)
    scale = torch.ldexp(torch.ones((), device="cuda"), _exponent(x.abs().amax((2, 4)), kind)).float()
    return _bytes_of(_round8(x / scale[:, :, None, :, None], kind), kind), scale


def _settings(c, seed):
    """Temperature, top-k, top-p and min-p of each row."""
    n, g = c["rows"], _gen(seed, 3)
    t = 0.5 + torch.rand(n, generator=g, device="cuda")
    k = torch.zeros(n, dtype=torch.int32, device="cuda")
    p = torch.ones(n, device="cuda")
    mp = torch.zeros(n, device="cuda")
    if c["mode"] == "chat":
        return t, k + 50, p * 0.9, mp
    if c["mode"] == "nucleus":
        return t, k, p * 0.95, mp
    if c["mode"] == "mixed":
        # what a batch of requests asks for: some greedy, some without any limit, top-k or top-p alone, both, min-p
        i = torch.arange(n, device="cuda")
        t = torch.where(i % 8 == 7, torch.zeros_like(t), t)
        k = torch.where((i % 8 == 1) | (i % 8 == 3) | (i % 8 == 4), torch.randint(1, 200, (n,), generator=g, device="cuda"), 0).to(torch.int32)
        p = torch.where((i % 8 == 2) | (i % 8 == 3) | (i % 8 == 6), 0.5 + 0.5 * torch.rand(n, generator=g, device="cuda"), p)
        mp = torch.where((i % 8 == 4) | (i % 8 == 5), 0.1 * torch.rand(n, generator=g, device="cuda"), mp)
    return t, k, p, mp


def prepare(case, seed):
    c = case
    g = _gen(seed)
    if c["op"] == "decode":
        lens = _lengths(c)
        need = [_pages(n) for n in lens]
        cache, scale = _cache(sum(need), c["kv_heads"], c["kind"], seed)
        perm = torch.randperm(sum(need), generator=g, device="cuda").to(torch.int32)
        width = max(need)
        first = torch.tensor(np.concatenate([[0], np.cumsum(need)[:-1]]), device="cuda")
        at = first[:, None] + torch.arange(width, device="cuda")[None, :]
        there = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
        table = torch.where(there, perm[at.clamp(max=sum(need) - 1)], torch.zeros((), dtype=torch.int32, device="cuda")).contiguous()
        q = torch.randn(c["batch"], c["heads"], D, generator=g, device="cuda").to(torch.bfloat16)
        return {"case": c, "q": q, "cache": cache, "scale": scale, "table": table, "lens": torch.tensor(lens, dtype=torch.int32, device="cuda"),
                "longest": max(lens)}
    if c["op"] == "write":
        total = c["prefix"] + c["tokens"]
        blocks = _pages(total) + 5
        cache, scale = _cache(blocks, c["kv_heads"], c["kind"], seed)
        table = torch.randperm(blocks, generator=g, device="cuda")[:_pages(total)].to(torch.int32)
        pos = torch.arange(c["prefix"], total, device="cuda")
        slots = table[pos // PAGE].long() * PAGE + pos % PAGE
        # keys and values stand side by side in the projection's rows; written again, they leave the cache as it is
        kv = torch.randn(c["tokens"], 2, c["kv_heads"], D, generator=g, device="cuda").to(torch.bfloat16) * 1.5
        kv[:, 0] = _outliers(kv[:, 0], seed, 2)
        return {"case": c, "k": kv[:, 0], "v": kv[:, 1], "slots": slots, "table": table, "cache": cache, "scale": scale}
    if c["op"] == "copy":
        caches = [torch.randn(c["blocks"], 2, PAGE, c["kv_heads"], D, generator=g, device="cuda").to(torch.bfloat16) for _ in range(c["layers"])]
        at = torch.randperm(c["blocks"], generator=g, device="cuda")[:2 * c["pairs"]].cpu()
        src, dst = at[:c["pairs"]], at[c["pairs"]:]
        # the block manager knows the copies on the host
        return {"case": c, "caches": caches, "pairs": list(zip(src.tolist(), dst.tolist()))}
    dtype = torch.bfloat16 if c["dtype"] == "bf16" else torch.float32
    ld = (c["vocab"] + 127) // 128 * 128              # the head's rows are padded
    x = 2.5 * torch.randn(c["rows"], ld, generator=g, device="cuda")
    hot = torch.randint(0, c["vocab"], (c["rows"], 12), generator=g, device="cuda")
    x.scatter_add_(1, hot, 6.0 + 3.0 * torch.rand(c["rows"], 12, generator=g, device="cuda"))
    t, k, p, mp = _settings(c, seed)
    return {"case": c, "logits": x.to(dtype), "u": torch.rand(c["rows"], generator=g, device="cuda"), "temperature": t, "top_k": k, "top_p": p, "min_p": mp}


# ------------------------------------------------------------------------------------------ one pass
def run(state):
    c = state["case"]
    if own:
        from ml_framework_b200.ops import native
        if c["op"] == "decode":
            return native.paged_decode(state["q"], state["cache"], state["table"], state["lens"], state["longest"], split_tokens=0, kv_scale=state["scale"])
        if c["op"] == "write":
            native.kv_cache_write(state["cache"], state["k"], state["v"], state["slots"], kv_scale=state["scale"])
            k, v = native.kv_gather(state["cache"], state["table"], c["prefix"] + c["tokens"], kv_scale=state["scale"])
            return {"k": k, "v": v, "scale": state["scale"]}
        if c["op"] == "copy":
            native.kv_copy_blocks_(state["caches"], state["pairs"])
            return state["caches"]
        tokens, logprobs = native.sample_rows(state["logits"], c["vocab"], state["u"], state["temperature"], state["top_k"], state["top_p"],
                                              state["min_p"], want_logprobs=True)
        return {"tokens": tokens, "logprobs": logprobs}
    if c["op"] == "decode":
        return _plain_decode(state)
    if c["op"] == "write":
        return _plain_write(state)
    if c["op"] == "copy":
        return _plain_copy(state)
    return _plain_sample(state)


def _plain_decode(s):
    q, cache, scale, lens = s["q"], s["cache"], s["scale"], s["lens"]
    B, Hq, Hkv = q.shape[0], q.shape[1], cache.shape[3]
    pos = torch.arange(s["longest"], device=q.device)
    blk, off = s["table"][:, pos // PAGE].long(), (pos % PAGE)[None, :]
    k = _rows(cache, (blk, 0, off)) * scale[blk, 0][..., None]                     # [B, L, Hkv, D]
    v = _rows(cache, (blk, 1, off)) * scale[blk, 1][..., None]
    there = (pos[None, :] < lens[:, None])[:, None, None, :]
    x = torch.einsum("bhgd,blhd->bhgl", q.float().view(B, Hkv, Hq // Hkv, D), k) * D ** -0.5
    x = x.masked_fill(~there, -math.inf)
    e = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-1e30))
    v = v * there[:, 0, 0, :, None, None]
    o = torch.einsum("bhgl,blhd->bhgd", e, v) / e.sum(-1, keepdim=True).clamp(min=1e-30)
    return o.reshape(B, Hq, D).to(torch.bfloat16)


def _plain_write(s):
    c, cache, scale, slots = s["case"], s["cache"], s["scale"], s["slots"]
    kind, new = c["kind"], torch.stack((s["k"], s["v"]), 1).float()                # [T, 2, Hkv, D]
    blk, off = slots // PAGE, slots % PAGE
    touched, of = torch.unique(blk, return_inverse=True)
    amax = torch.zeros(touched.numel(), 2, new.shape[2], device=new.device).index_reduce_(0, of, new.abs().amax(-1), "amax")
    anew = torch.zeros(touched.numel(), device=new.device).index_reduce_(0, of, (off == 0).float(), "amax")[:, None, None] > 0
    fits = torch.ldexp(torch.ones_like(amax), _exponent(amax, kind))
    before = scale[touched]
    now = torch.where(anew, fits, torch.maximum(before, fits))
    held = _rows(cache, touched)                                                    # [pages, 2, PAGE, Hkv, D]
    shrink = torch.where(anew, torch.ones_like(now), before / now)
    held = _round8(held * shrink[:, :, None, :, None], kind)
    held[of, :, off] = _round8(new / now[of][..., None], kind)
    cache.view(torch.uint8)[touched] = _bytes_of(held, kind).view(torch.uint8)
    scale[touched] = now
    pos = torch.arange(c["prefix"] + c["tokens"], device=slots.device)
    b = s["table"][pos // PAGE].long()
    k = (_rows(cache, (b, 0, pos % PAGE)) * scale[b, 0][..., None]).to(torch.bfloat16)
    v = (_rows(cache, (b, 1, pos % PAGE)) * scale[b, 1][..., None]).to(torch.bfloat16)
    return {"k": k, "v": v, "scale": scale}


def _plain_copy(s):
    at = torch.tensor(s["pairs"], device=s["caches"][0].device)
    return [cache.index_copy_(0, at[:, 1], cache[at[:, 0]]) for cache in s["caches"]]


def _plain_sample(s):
    # sums of up to 128 K weights and the borders between tokens need 64 bits
    V = s["case"]["vocab"]
    x = s["logits"][:, :V].double()
    t, u = s["temperature"].double()[:, None], s["u"].double()[:, None]
    greedy = t <= 0
    top = x.amax(1, keepdim=True)
    w = torch.exp((x - top) / torch.where(greedy, 1.0, t))
    w = torch.where(greedy, (x == top).double(), w)
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(V, device=x.device)[None, :]
    k = torch.where(greedy, 1, torch.where(s["top_k"][:, None] <= 0, V, s["top_k"][:, None]))
    ws_k = torch.where(rank < k, ws, 0.0)
    before = torch.cumsum(ws_k, 1) - ws_k
    p = s["top_p"].double()[:, None]
    keep = (rank < k) & ((rank == 0) | (p >= 1) | (before < p * ws_k.sum(1, keepdim=True))) & ((rank == 0) | (ws >= s["min_p"].double()[:, None]))
    kept = torch.zeros_like(x).scatter_(1, order, torch.where(keep, ws, 0.0))
    total = torch.cumsum(kept, 1)
    last = torch.where(kept > 0, rank, 0).amax(1)
    token = torch.minimum((total <= u * total[:, -1:]).sum(1), last)
    logprob = torch.log(kept.gather(1, token[:, None])[:, 0] / total[:, -1])
    return {"tokens": token, "logprobs": logprob.float()}


# ------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
    c = case
    if c["op"] == "decode":
        n = sum(_lengths(c))
        pages = sum(_pages(x) for x in _lengths(c))
        return {"bytes": n * 2.0 * c["kv_heads"] * D + pages * (8.0 * c["kv_heads"] + 4) + 4.0 * c["batch"] * c["heads"] * D, "flops": 4.0 * n * c["heads"] * D}
    if c["op"] == "write":
        row = 2.0 * c["kv_heads"] * D
        # new rows in 16 bits and out in 8, the whole sequence in 8 bits (the prefix read) and out in 16
        return {"bytes": c["tokens"] * 3 * row + c["prefix"] * row + (c["prefix"] + c["tokens"]) * 2 * row, "flops": 2.0 * c["tokens"] * row}
    if c["op"] == "copy":
        return {"bytes": c["layers"] * c["pairs"] * 2 * (2.0 * PAGE * c["kv_heads"] * D * 2), "flops": 0.0}
    n = c["rows"] * c["vocab"]
    return {"bytes": n * (2.0 if c["dtype"] == "bf16" else 4.0) + c["rows"] * 32.0, "flops": 4.0 * n}


# ------------------------------------------------------------------------------------------ the same in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = case
    if c["op"] == "decode":
        return _exact_decode(c, s)
    if c["op"] == "write":
        return _exact_write(c, s)
    if c["op"] == "copy":
        out = [t.clone() for t in s["caches"]]
        for was, t in zip(s["caches"], out):
            for a, b in s["pairs"]:
                t[b] = was[a]
        return out
    return _exact_sample(c, s)


def _exact_decode(c, s):
    out = torch.empty(c["batch"], c["heads"], D, dtype=torch.float64, device="cuda")
    group = c["heads"] // c["kv_heads"]
    values = s["cache"].float()
    for b, n in enumerate(_lengths(c)):
        pages = s["table"][b, :_pages(n)].long()
        kv = values[pages].double() * s["scale"][pages].double()[:, :, None, :, None]
        kv = kv.transpose(0, 1).reshape(2, -1, c["kv_heads"], D)[:, :n]
        for h in range(c["kv_heads"]):
            q = s["q"][b, h * group:(h + 1) * group].double()
            out[b, h * group:(h + 1) * group] = torch.softmax(q @ kv[0, :, h].T / math.sqrt(D), -1) @ kv[1, :, h]
    return out


def _exact_write(c, s):
    """Block by block: scales by comparison with every power of two, int8 and e4m3 by the nearest of the numbers that exist."""
    m = np.arange(8) / 8.0
    if c["kind"] == "e4m3":
        grid = np.concatenate([m * 2.0 ** -6] + [(1 + m) * 2.0 ** e for e in range(-6, 9)])
        grid = grid[grid <= 448.0]
    else:
        grid = np.arange(128.0)
    powers = 2.0 ** np.arange(-40, 41)

    def nearest(x):
        a = np.minimum(np.abs(x), grid[-1])
        hi = np.searchsorted(grid, a).clip(1, len(grid) - 1)
        lo = hi - 1
        up, down = grid[hi] - a, a - grid[lo]
        return np.sign(x) * np.where((up < down) | ((up == down) & (hi % 2 == 0)), grid[hi], grid[lo])   # ties: even mantissa

    held = s["cache"].float().cpu().numpy().astype(np.float64)
    scale = s["scale"].cpu().numpy().astype(np.float64)
    new = np.stack((s["k"].float().cpu().numpy(), s["v"].float().cpu().numpy()), 1).astype(np.float64)
    slots = s["slots"].cpu().numpy()
    for b in dict.fromkeys((slots // PAGE).tolist()):
        rows = np.nonzero(slots // PAGE == b)[0]
        off = slots[rows] % PAGE
        for j in range(2):
            amax = np.abs(new[rows, j]).max((0, 2))
            fit = powers[np.minimum(np.searchsorted(powers * grid[-1], amax), len(powers) - 1)]
            if 0 not in off:
                fit = np.maximum(fit, scale[b, j])
                held[b, j] = nearest(held[b, j] * (scale[b, j] / fit)[None, :, None])
            scale[b, j] = fit
            held[b, j, off] = nearest(new[rows, j] / fit[None, :, None])
    total = c["prefix"] + c["tokens"]
    pages = s["table"].cpu().numpy()
    values = (held[pages] * scale[pages][:, :, None, :, None]).transpose(1, 0, 2, 3, 4).reshape(2, -1, c["kv_heads"], D)[:, :total]
    return {"k": torch.from_numpy(values[0]), "v": torch.from_numpy(values[1]), "scale": torch.from_numpy(scale)}


def _exact_sample(c, s):
    V = c["vocab"]
    x = s["logits"][:, :V].float().cpu().numpy().astype(np.float64)
    par = [s[n].cpu().numpy().astype(np.float64) for n in ("temperature", "top_k", "top_p", "min_p", "u")]
    tokens, logprobs = np.zeros(c["rows"], np.int64), np.zeros(c["rows"])
    for r in range(c["rows"]):
        t, k, p, least, u = (float(a[r]) for a in par)
        if t <= 0:
            tokens[r] = int(np.argmax(x[r]))
            continue
        w = np.exp((x[r] - x[r].max()) / t)
        order = np.argsort(-x[r], kind="stable")
        if 0 < k < V:
            order = order[:int(k)]
        if p < 1:
            run_sum = np.cumsum(w[order])
            order = order[:int(np.searchsorted(run_sum, p * run_sum[-1])) + 1]
        order = np.sort(order[(w[order] >= least) | (np.arange(len(order)) == 0)])
        run_sum = np.cumsum(w[order])
        at = min(int(np.searchsorted(run_sum, u * run_sum[-1], side="right")), len(order) - 1)
        tokens[r], logprobs[r] = order[at], math.log(w[order[at]] / run_sum[-1])
    return {"tokens": torch.from_numpy(tokens), "logprobs": torch.from_numpy(logprobs)}
