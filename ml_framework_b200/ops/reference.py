"""Plain-PyTorch (fp32) statements of every native kernel.

They serve three purposes: the CPU execution path of the framework (so models, parallel
wrappers and the serving stack run and are tested without a GPU), the oracle that GPU tests
compare the CUDA kernels against, and executable documentation of the math.
"""
from __future__ import annotations

import math

import torch
import torch.nn.functional as F


def layer_norm_ref(x, gamma, beta, eps=1e-5):
    xf = x.float()
    mean = xf.mean(-1, keepdim=True)
    var = ((xf - mean) ** 2).mean(-1, keepdim=True)
    rstd = torch.rsqrt(var + eps)
    y = (xf - mean) * rstd * gamma.float() + (beta.float() if beta is not None else 0.0)
    return y, mean.squeeze(-1), rstd.squeeze(-1)


def rms_norm_ref(x, gamma, eps=1e-5):
    xf = x.float()
    rstd = torch.rsqrt((xf * xf).mean(-1, keepdim=True) + eps)
    return xf * rstd * gamma.float(), rstd.squeeze(-1)


def rope_ref(x: torch.Tensor, pos: torch.Tensor, theta: float, inverse: bool = False) -> torch.Tensor:
    """x [T, H, Dh], rotate-half convention: pairs (d, d + Dh/2)."""
    T, H, Dh = x.shape
    half = Dh // 2
    inv_freq = torch.exp(-math.log(theta) * (2.0 * torch.arange(half, device=x.device, dtype=torch.float32) / Dh))
    ang = pos.float()[:, None] * inv_freq[None, :]
    c, s = torch.cos(ang)[:, None, :], torch.sin(ang)[:, None, :]
    if inverse:
        s = -s
    xf = x.float()
    a, b = xf[..., :half], xf[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], dim=-1)


def swiglu_ref(gu: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    f = gu.float()
    if interleaved:
        g, u = f[..., 0::2], f[..., 1::2]
    else:
        Fh = f.shape[-1] // 2
        g, u = f[..., :Fh], f[..., Fh:]
    return F.silu(g) * u


def attention_ref(q, k, v, *, causal=True, scale=None, start_pos: int = 0):
    """q [B, Sq, Hq, D], k/v [B, Sk, Hkv, D] -> (out [B, Sq, Hq, D], lse [B, Hq, Sq]).

    With ``causal`` query i sees keys ``<= start_pos + i`` (start_pos = Sk - Sq for decode),
    the rule of StandardPagedAttentionKernel.ApplyCausalMask
    (src/MLFramework/Inference/PagedAttention/Kernels/StandardPagedAttentionKernel.cs:219-255).
    """
    B, Sq, Hq, D = q.shape
    Sk, Hkv = k.shape[1], k.shape[2]
    scale = scale if scale is not None else D ** -0.5
    rep = Hq // Hkv
    qf = q.float().permute(0, 2, 1, 3)
    kf = k.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    vf = v.float().permute(0, 2, 1, 3).repeat_interleave(rep, dim=1)
    s = torch.matmul(qf, kf.transpose(-1, -2)) * scale
    if causal:
        qi = torch.arange(Sq, device=q.device)[:, None] + start_pos
        kj = torch.arange(Sk, device=q.device)[None, :]
        s = s.masked_fill(kj > qi, float("-inf"))
    lse = torch.logsumexp(s, dim=-1)
    p = torch.softmax(s, dim=-1)
    o = torch.matmul(p, vf).permute(0, 2, 1, 3)
    return o, lse


def paged_attention_ref(q, kv_cache, block_table, seq_lens, *, scale=None, kv_scale=None):
    """Decode attention through a block table.

    q [B, Hq, D]; kv_cache [num_blocks, 2, block_size, Hkv, D]; block_table [B, max_blocks]
    (int32); seq_lens [B] = number of cached tokens including the current one. Returns [B, Hq, D].
    kv_scale [num_blocks, 2, Hkv]: the scales of an 8-bit cache. A sequence's own blocks are all that is converted.
    """
    B, Hq, D = q.shape
    bs = kv_cache.shape[2]
    outs = []
    for b in range(B):
        n = int(seq_lens[b])
        nb = (n + bs - 1) // bs
        blocks = block_table[b, :nb].long()
        pages = kv_values_ref(kv_cache[blocks], kv_scale[blocks] if kv_scale is not None else None)
        k = pages[:, 0].reshape(nb * bs, -1, D)[:n]
        v = pages[:, 1].reshape(nb * bs, -1, D)[:n]
        o, _ = attention_ref(q[b][None, None], k[None], v[None], causal=False, scale=scale)
        outs.append(o[0, 0])
    return torch.stack(outs)


# ------------------------------------------------------------------ paged cache in 8 bits
def q8_scale_ref(amax: torch.Tensor, dtype) -> torch.Tensor:
    """The smallest power of two, 2^-40 to 2^40, under which magnitudes up to ``amax`` fit ``dtype`` (448 or 127)."""
    frac, e = torch.frexp(amax.float())
    top, bits = (448 / 512, 9) if dtype == torch.float8_e4m3fn else (127 / 128, 7)
    e = torch.where(frac <= top, e - bits, e - bits + 1)
    e = torch.where(amax == 0, torch.full_like(e, -40), torch.where(torch.isinf(amax), torch.full_like(e, 40), e)).clamp(-40, 40)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float32), e)


def q8_round_ref(x: torch.Tensor, dtype) -> torch.Tensor:
    """Numbers in units of their scale rounded to 8 bits, ties to even; NaN stays in e4m3 and becomes 0 in int8."""
    if dtype == torch.float8_e4m3fn:
        return x.clamp(-448.0, 448.0).to(dtype)
    return torch.nan_to_num(x, nan=0.0).round().clamp(-127.0, 127.0).to(dtype)


def kv_values_ref(cache: torch.Tensor, scale: Optional[torch.Tensor]) -> torch.Tensor:
    """The values of cache blocks [n, 2, block_size, Hkv, D] (all of a cache, or some blocks with their scales) in fp32."""
    return cache.float() if scale is None else cache.float() * scale[:, :, None, :, None]


def kv_write_ref(cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, scale: Optional[torch.Tensor] = None):
    """k, v [T, Hkv, D] into cache slots (< 0 skips), in place. With ``scale`` (an 8-bit cache) the blocks' scales are settled first:
    a block whose first row is written takes the new rows' own, another one the larger of that and its old scale, to which
    the rows that it holds are rounded."""
    bs = cache.shape[2]
    ok = slots >= 0
    blk, off = slots[ok] // bs, slots[ok] % bs
    new = torch.stack((k[ok], v[ok]), 1)
    if scale is None:
        cache[blk, :, off] = new.to(cache.dtype)
        return
    new = new.float()
    for b in torch.unique(blk).tolist():
        at = blk == b
        amax = torch.nan_to_num(new[at].abs(), nan=0.0, posinf=float("inf")).amax((0, 3))
        now = q8_scale_ref(amax, cache.dtype)
        if not bool((off[at] == 0).any()):
            before = scale[b].clone()
            now = torch.maximum(now, before)
            grown = (before < now)[:, None, :, None]
            held = cache[b].float()
            cache[b] = q8_round_ref(torch.where(grown, held * (before / now)[:, None, :, None], held), cache.dtype)
        scale[b] = now
        cache[b][:, off[at]] = q8_round_ref(new[at] / now[None, :, :, None], cache.dtype).transpose(0, 1)


# ------------------------------------------------------------------ sampling
def sample_ref(logits: torch.Tensor, vocab: int, u: torch.Tensor, temperature: torch.Tensor, top_k: Optional[torch.Tensor] = None,
               top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None):
    """(tokens, logprobs) of ``native.sample_rows`` in 64 bits, by its definition."""
    x = logits[:, :vocab].double()
    x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
    rows, dev = x.shape[0], x.device
    t = temperature.double()[:, None].clamp(max=2.0 ** 90)
    greedy = ~(t >= 2.0 ** -90)
    top = x.amax(1, keepdim=True)
    first = (x == top).to(torch.int8).argmax(1)                     # of equal ones the lowest index
    w = torch.where(x == top, 1.0, torch.exp((x - top) / torch.where(greedy, 1.0, t)))
    w = torch.where(torch.isinf(x) & (x < 0), 0.0, w)
    _, order = torch.sort(x, dim=1, descending=True, stable=True)
    ws = w.gather(1, order)
    rank = torch.arange(vocab, device=dev)[None, :]
    k = torch.full((rows, 1), vocab, device=dev) if top_k is None else torch.where(top_k <= 0, vocab, top_k.long())[:, None]
    ws = torch.where(rank < k, ws, 0.0)
    keep = ws > 0
    if top_p is not None:
        p = top_p.double()[:, None]
        keep &= (p >= 1) | (torch.cumsum(ws, 1) - ws < p * ws.sum(1, keepdim=True)) | (rank == 0)
    if min_p is not None:
        keep &= (ws >= min_p.double()[:, None]) | (rank == 0)
    kept = torch.zeros_like(x).scatter_(1, order, torch.where(keep, ws, 0.0))
    run = torch.cumsum(kept, 1)
    last = torch.where(kept > 0, rank, 0).amax(1)
    token = torch.minimum((run <= u.double()[:, None] * run[:, -1:]).sum(1), last)
    logprob = torch.log(kept.gather(1, token[:, None])[:, 0] / run[:, -1])
    none = torch.isinf(top[:, 0]) & (top[:, 0] < 0)
    token = torch.where(greedy[:, 0], first, token)
    logprob = torch.where(greedy[:, 0], torch.zeros_like(logprob), logprob)
    return torch.where(none, torch.zeros_like(token), token), torch.where(none, torch.full_like(logprob, float("-inf")), logprob).float()


def adamw_ref(p, m, v, g, *, lr, beta1, beta2, eps, weight_decay, step, vmax=None):
    """One AdamW step in fp32, decay first then the Adam update
    (src/MLFramework/Optimizers/Adam.cs:167-213). Returns new (p, m, v[, vmax])."""
    m = beta1 * m + (1 - beta1) * g
    v = beta2 * v + (1 - beta2) * g * g
    bc1, bc2 = 1 - beta1 ** step, 1 - beta2 ** step
    vh = v
    if vmax is not None:
        vmax = torch.maximum(vmax, v)
        vh = vmax
    p = p - lr * weight_decay * p
    p = p - lr * (m / bc1) / (torch.sqrt(vh / bc2) + eps)
    return (p, m, v) if vmax is None else (p, m, v, vmax)


def cross_entropy_ref(logits: torch.Tensor, targets: torch.Tensor, vocab: int, grad_scale: float = 1.0):
    """Returns (loss_rows fp32, dlogits fp32 * grad_scale); target < 0 rows are ignored."""
    lf = logits.float()[:, :vocab]
    lse = torch.logsumexp(lf, dim=-1)
    valid = targets >= 0
    tg = targets.clamp(min=0)
    loss = (lse - lf.gather(1, tg[:, None]).squeeze(1)) * valid
    p = torch.softmax(lf, dim=-1)
    p[torch.arange(lf.shape[0]), tg] -= 1.0
    p = p * valid[:, None] * grad_scale
    d = torch.zeros(logits.shape, dtype=torch.float32, device=logits.device)
    d[:, :vocab] = p
    return loss, d
