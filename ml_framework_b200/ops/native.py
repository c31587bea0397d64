"""Thin, typed wrappers over the C ABI of ``libmlfb200.so`` (one Python function per kernel).

Every wrapper takes CUDA tensors, launches on the current stream and returns its outputs.
They fail loudly (``MlfError``) on a host-side problem; nothing here falls back to PyTorch.
The PyTorch statements of the same math, used on CPU tensors and as test oracles, live in
:mod:`ml_framework_b200.ops.reference`.
"""
from __future__ import annotations

import ctypes as C
from array import array
from functools import lru_cache
from itertools import chain
from operator import attrgetter
from typing import Optional, Sequence, Tuple

import torch

from .. import _lib

_BIN_OPS = {"add": 0, "sub": 1, "mul": 2, "div": 3, "max": 4, "min": 5}
_UN_OPS = {"relu": 0, "sigmoid": 1, "tanh": 2, "gelu": 3, "silu": 4, "exp": 5, "neg": 6, "sqrt": 7, "log": 8, "abs": 9}
_RED = {"sum": 0, "max": 1, "min": 2, "mean": 3}


def _L():
    return _lib.get()


def _st():
    return C.c_uint64(_lib.stream_handle())


def _p(t: Optional[torch.Tensor]):
    """Address of ``t``, which the caller has to hold until the launch is queued: a copy that nothing else holds is freed at
    once, and the next one may be put in its place."""
    return C.c_void_p(t.data_ptr()) if t is not None else None


def _dt(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return 0
    if t.dtype == torch.bfloat16:
        return 1
    raise TypeError(f"unsupported dtype {t.dtype}; kernels take float32 or bfloat16")


_scratch: dict = {}


def scratch(name: str, nbytes: int, device) -> torch.Tensor:
    """Per-device, per-purpose scratch buffer that only ever grows (uint8)."""
    key = (name, torch.device(device).index)
    buf = _scratch.get(key)
    if buf is None or buf.numel() < nbytes:
        buf = torch.empty(max(nbytes, 1 << 16), dtype=torch.uint8, device=device)
        _scratch[key] = buf
    return buf


# ------------------------------------------------------------------ element-wise / reductions
def ew_binary(op: str, a: torch.Tensor, b, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    a = a.contiguous()
    out = torch.empty_like(a) if out is None else out
    if isinstance(b, torch.Tensor):
        b = b.contiguous()
        assert b.shape == a.shape and b.dtype == a.dtype
        rc = _L().mlf_ew_binary(_p(out), _p(a), _p(b), C.c_float(0.0), C.c_longlong(a.numel()), _BIN_OPS[op], _dt(a), _st())
    else:
        rc = _L().mlf_ew_binary(_p(out), _p(a), None, C.c_float(float(b)), C.c_longlong(a.numel()), _BIN_OPS[op], _dt(a), _st())
    _lib.check(rc, "mlf_ew_binary")
    return out


def ew_unary(op: str, a: torch.Tensor, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    a = a.contiguous()
    out = torch.empty_like(a) if out is None else out
    _lib.check(_L().mlf_ew_unary(_p(out), _p(a), C.c_longlong(a.numel()), _UN_OPS[op], _dt(a), _st()), "mlf_ew_unary")
    return out


def fill_(t: torch.Tensor, value: float) -> torch.Tensor:
    assert t.is_contiguous()
    _lib.check(_L().mlf_fill(_p(t), C.c_float(value), C.c_longlong(t.numel()), _dt(t), _st()), "mlf_fill")
    return t


def reduce_all(op: str, a: torch.Tensor) -> torch.Tensor:
    a = a.contiguous()
    out = torch.empty((), dtype=torch.float32, device=a.device)
    sc = scratch("reduce", 4096, a.device)
    _lib.check(_L().mlf_reduce_all(_p(out), _p(a), C.c_longlong(a.numel()), _RED[op], _dt(a), _p(sc), _st()), "mlf_reduce_all")
    return out


# ------------------------------------------------------------------ norms
def norm_fwd(x: torch.Tensor, gamma: torch.Tensor, beta: Optional[torch.Tensor], eps: float, rms: bool,
             want_stats: bool = True, zero: Optional[torch.Tensor] = None):
    """``zero``: a contiguous buffer that the same launch clears (the output a following product accumulates into)."""
    D = x.shape[-1]
    x2 = x.reshape(-1, D)
    assert x2.is_contiguous() and x2.dtype == torch.bfloat16
    rows = x2.shape[0]
    y = torch.empty_like(x2)
    mean = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats and not rms else None
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if want_stats else None
    zbytes = 0
    if zero is not None:
        assert zero.is_contiguous() and zero.device == x.device
        zbytes = zero.numel() * zero.element_size()
    rc = _L().mlf_norm_fwd_zero(_p(x2), _p(gamma), _p(beta), _p(y), _p(mean), _p(rstd), rows, D, C.c_float(eps), int(rms),
                                _p(zero), C.c_longlong(zbytes), _st())
    _lib.check(rc, "mlf_norm_fwd")
    return y.view(x.shape), mean, rstd


def norm_bwd(x: torch.Tensor, dy: torch.Tensor, gamma: torch.Tensor, mean, rstd, rms: bool,
             dgamma_out: Optional[torch.Tensor] = None, dbeta_out: Optional[torch.Tensor] = None,
             accumulate: bool = False, dx_add: Optional[torch.Tensor] = None, accumulate_beta: Optional[bool] = None):
    """``dx_add`` (same shape as x) is added to the returned dx inside the kernel: the gradient of a skip
    connection that branched off x. ``accumulate`` adds the gradients of gamma and beta to their buffers (of one type),
    ``accumulate_beta`` decides for beta's alone."""
    D = x.shape[-1]
    x2, dy2 = x.reshape(-1, D), dy.reshape(-1, D)
    assert x2.is_contiguous() and dy2.is_contiguous()
    add2 = None
    if dx_add is not None:
        add2 = dx_add.reshape(-1, D)
        assert add2.is_contiguous() and add2.dtype == x2.dtype and add2.shape == x2.shape
    rows = x2.shape[0]
    dx = torch.empty_like(x2)
    grad_dtype = dgamma_out.dtype if dgamma_out is not None else dbeta_out.dtype if dbeta_out is not None and not rms else gamma.dtype
    dgamma = dgamma_out if dgamma_out is not None else torch.empty(D, dtype=grad_dtype, device=x.device)
    dbeta = None
    if not rms:
        dbeta = dbeta_out if dbeta_out is not None else torch.empty(D, dtype=grad_dtype, device=x.device)
        assert dbeta.dtype == grad_dtype
    L = _L()
    L.mlf_norm_bwd_scratch_elems.restype = C.c_longlong
    n = L.mlf_norm_bwd_scratch_elems(rows, D)
    part = scratch("norm_bwd", n * 4, x.device)
    rc = L.mlf_norm_bwd_add(_p(x2), _p(dy2), _p(gamma), _p(mean), _p(rstd), _p(dx), _p(dgamma), _p(dbeta), _p(part),
                            rows, D, int(rms), int(grad_dtype == torch.float32), int(accumulate),
                            int(accumulate if accumulate_beta is None else accumulate_beta), _p(add2), _st())
    _lib.check(rc, "mlf_norm_bwd_add")
    return dx.view(x.shape), dgamma, dbeta


# ------------------------------------------------------------------ activations
def gelu_bwd(dy: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    dx = torch.empty_like(x)
    dy, x = dy.contiguous(), x.contiguous()
    _lib.check(_L().mlf_gelu_bwd(_p(dx), _p(dy), _p(x), C.c_longlong(x.numel()), _st()), "mlf_gelu_bwd")
    return dx


def swiglu_fwd(gu: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    F = gu.shape[-1] // 2
    g2 = gu.reshape(-1, 2 * F)
    out = torch.empty(g2.shape[0], F, dtype=gu.dtype, device=gu.device)
    _lib.check(_L().mlf_swiglu_fwd(_p(out), _p(g2), C.c_longlong(g2.shape[0]), F, int(interleaved), _st()), "mlf_swiglu_fwd")
    return out.view(*gu.shape[:-1], F)


def swiglu_bwd(dout: torch.Tensor, gu: torch.Tensor, interleaved: bool = False) -> torch.Tensor:
    F = gu.shape[-1] // 2
    g2 = gu.reshape(-1, 2 * F)
    dgu = torch.empty_like(g2)
    dout = dout.reshape(-1, F).contiguous()
    _lib.check(_L().mlf_swiglu_bwd(_p(dgu), _p(dout), _p(g2), C.c_longlong(g2.shape[0]), F,
                                   int(interleaved), _st()), "mlf_swiglu_bwd")
    return dgu.view(gu.shape)


def colsum_scratch(M: int, widths, device) -> torch.Tensor:
    """Scratch for column sums of matrices of M rows: launches over ``widths`` columns, of one matrix or (a pair) of two."""
    L = _L()
    L.mlf_colsum2_scratch_bytes.restype = C.c_longlong
    need = max(int(L.mlf_colsum2_scratch_bytes(M, *(n if isinstance(n, tuple) else (n, 0)))) for n in widths)
    key = ("colsum0", device.index)
    sc = _scratch.get(key)
    if sc is None or sc.numel() < need:                  # zero-filled once: the kernel keeps its counters at zero
        sc = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=device)
        _scratch[key] = sc
    return sc


def colsum(dy: torch.Tensor, out: Optional[torch.Tensor] = None, accumulate: bool = False) -> torch.Tensor:
    """bf16 column sums of a 2-D bf16 matrix (bias gradient)."""
    assert dy.dim() == 2 and dy.stride(1) == 1
    M, N = dy.shape
    out = torch.empty(N, dtype=torch.bfloat16, device=dy.device) if out is None else out
    L = _L()
    sc = colsum_scratch(M, (N,), dy.device)
    _lib.check(L.mlf_colsum(_p(out), _p(dy), M, N, C.c_longlong(dy.stride(0)), _p(sc), int(accumulate), _st()), "mlf_colsum")
    return out


def embedding_fwd(ids: torch.Tensor, wte: torch.Tensor, pos: Optional[torch.Tensor] = None,
                  wpe: Optional[torch.Tensor] = None) -> torch.Tensor:
    T = ids.numel()
    D = wte.shape[1]
    out = torch.empty(T, D, dtype=wte.dtype, device=wte.device)
    flat = ids.reshape(-1).contiguous()
    pos = pos.reshape(-1).contiguous() if pos is not None else None
    rc = _L().mlf_embedding_fwd(_p(out), _p(flat), _p(pos), _p(wte), _p(wpe), C.c_longlong(T), D, wte.shape[0], wpe.shape[0] if wpe is not None else 0, _st())
    _lib.check(rc, "mlf_embedding_fwd")
    return out.view(*ids.shape, D)


def embedding_bwd(dout: torch.Tensor, ids: torch.Tensor, vocab: int, dw_fp32: Optional[torch.Tensor] = None) -> torch.Tensor:
    D = dout.shape[-1]
    T = ids.numel()
    if dw_fp32 is None:
        dw_fp32 = torch.zeros(vocab, D, dtype=torch.float32, device=dout.device)
    dout, ids = dout.reshape(T, D).contiguous(), ids.reshape(-1).contiguous()
    rc = _L().mlf_embedding_bwd(_p(dw_fp32), _p(dout), _p(ids), C.c_longlong(T), D, vocab, _st())
    _lib.check(rc, "mlf_embedding_bwd")
    return dw_fp32


def embedding_grad(dout: torch.Tensor, ids: torch.Tensor, out: torch.Tensor, accumulate: bool = False) -> torch.Tensor:
    """out[v] (+)= sum of dout's rows with id v, summed in fp32 and rounded once. ``out``: contiguous bf16 [vocab, D],
    16-byte aligned."""
    vocab, D = out.shape
    T = ids.numel()
    L = _L()
    L.mlf_embedding_grad_scratch_bytes.restype = C.c_longlong
    scratch = torch.empty(L.mlf_embedding_grad_scratch_bytes(C.c_longlong(T), D, vocab), dtype=torch.uint8, device=dout.device)
    dout, ids = dout.reshape(T, D).contiguous(), ids.reshape(-1).contiguous()
    rc = L.mlf_embedding_grad(_p(out), _p(dout), _p(ids), _p(scratch), C.c_longlong(T), D, vocab, int(accumulate), _st())
    _lib.check(rc, "mlf_embedding_grad")
    return out


def cast_f32_to_bf16(src: torch.Tensor, out: torch.Tensor, accumulate: bool = False) -> torch.Tensor:
    _lib.check(_L().mlf_cast_f32_to_bf16(_p(out), _p(src), C.c_longlong(src.numel()), int(accumulate), _st()), "mlf_cast")
    return out


def rope_(x: torch.Tensor, pos: torch.Tensor, theta: float, inverse: bool = False) -> torch.Tensor:
    """In-place rotary embedding on ``x`` [T, H, Dh] (may be a strided view over a packed row)."""
    T, H, Dh = x.shape
    assert x.stride(2) == 1 and x.stride(1) == Dh
    pos = pos.contiguous()
    rc = _L().mlf_rope(_p(x), _p(pos), C.c_longlong(T), H, Dh, C.c_longlong(x.stride(0)), C.c_float(theta),
                       int(inverse), _st())
    _lib.check(rc, "mlf_rope")
    return x


def rope_qkv(qkv: torch.Tensor, pos: torch.Tensor, Hq: int, Hkv: int, theta: float, inverse: bool = False,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rotary embedding of the query and key heads of packed rows [T, (Hq + 2 Hkv) * 128] into ``out`` (a new tensor by
    default, ``qkv`` itself for in place); value heads are copied. Rows must be 16-byte aligned."""
    assert qkv.dim() == 2 and qkv.stride(1) == 1 and qkv.shape[1] == (Hq + 2 * Hkv) * 128 and qkv.dtype == torch.bfloat16
    assert pos.dtype == torch.int64 and pos.numel() == qkv.shape[0]
    if out is None:
        out = torch.empty(qkv.shape, dtype=qkv.dtype, device=qkv.device)
    assert out.shape == qkv.shape and out.dtype == qkv.dtype and out.stride(1) == 1
    pos = pos.contiguous()
    rc = _L().mlf_rope_qkv(_p(out), _p(qkv), _p(pos), C.c_longlong(qkv.shape[0]), Hq, Hkv, C.c_longlong(out.stride(0)),
                           C.c_longlong(qkv.stride(0)), C.c_float(theta), int(inverse), _st())
    _lib.check(rc, "mlf_rope_qkv")
    return out


# ------------------------------------------------------------------ optimizer / AMP / loss
def adamw_(master, m, v, grad, param_out, *, lr, beta1, beta2, eps, weight_decay, step, grad_scale=1.0,
           inv_scale: Optional[torch.Tensor] = None, found_inf: Optional[torch.Tensor] = None, vmax=None):
    n = master.numel()
    rc = _L().mlf_adamw(_p(master), _p(m), _p(v), _p(vmax), _p(grad), _dt(grad), _p(param_out), C.c_longlong(n),
                        C.c_float(lr), C.c_float(beta1), C.c_float(beta2), C.c_float(eps), C.c_float(weight_decay),
                        int(step), C.c_float(grad_scale), _p(inv_scale), _p(found_inf), _st())
    _lib.check(rc, "mlf_adamw")


def sgd_(master, mom, grad, param_out, *, lr, momentum=0.0, weight_decay=0.0, grad_scale=1.0, inv_scale=None, found_inf=None):
    rc = _L().mlf_sgd(_p(master), _p(mom), _p(grad), _dt(grad), _p(param_out), C.c_longlong(master.numel()), C.c_float(lr),
                      C.c_float(momentum), C.c_float(weight_decay), C.c_float(grad_scale), _p(inv_scale), _p(found_inf), _st())
    _lib.check(rc, "mlf_sgd")


def amp_unscale_check_(grad, found_inf: torch.Tensor, *, inv_scale: Optional[torch.Tensor] = None, inv_scale_host: float = 1.0,
                       sumsq: Optional[torch.Tensor] = None, write_back: bool = True):
    rc = _L().mlf_amp_unscale_check(_p(grad), _dt(grad), C.c_longlong(grad.numel()), _p(inv_scale), C.c_float(inv_scale_host),
                                    _p(found_inf), _p(sumsq), int(write_back), _st())
    _lib.check(rc, "mlf_amp_unscale_check")


def scaler_update_(scale: torch.Tensor, tracker: torch.Tensor, found_inf: torch.Tensor, *, growth, backoff, interval,
                   min_scale, max_scale, skipped: Optional[torch.Tensor] = None):
    rc = _L().mlf_scaler_update(_p(scale), _p(tracker), _p(found_inf), C.c_float(growth), C.c_float(backoff), int(interval),
                                C.c_float(min_scale), C.c_float(max_scale), _p(skipped), _st())
    _lib.check(rc, "mlf_scaler_update")


def clip_scale_(grad, sumsq: torch.Tensor, max_norm: float, eps: float = 1e-6):
    rc = _L().mlf_clip_scale(_p(grad), _dt(grad), C.c_longlong(grad.numel()), _p(sumsq), C.c_float(max_norm), C.c_float(eps), _st())
    _lib.check(rc, "mlf_clip_scale")


def cross_entropy_(logits: torch.Tensor, targets: torch.Tensor, vocab: int, *, grad_scale: float = 1.0,
                   grad_scale_dev: Optional[torch.Tensor] = None, loss_weight: float = 1.0):
    """Overwrites ``logits`` [T, ld] with d(loss)/d(logits) * grad_scale; returns (loss_rows, loss_sum)."""
    assert logits.dim() == 2 and logits.stride(1) == 1 and logits.dtype == torch.bfloat16
    T = logits.shape[0]
    loss_rows = torch.empty(T, dtype=torch.float32, device=logits.device)
    loss_sum = torch.zeros((), dtype=torch.float32, device=logits.device)
    targets = targets.contiguous()
    rc = _L().mlf_cross_entropy(_p(logits), _p(targets), _p(loss_rows), _p(loss_sum), T, vocab,
                                C.c_longlong(logits.stride(0)), C.c_float(grad_scale), _p(grad_scale_dev),
                                C.c_float(loss_weight), _st())
    _lib.check(rc, "mlf_cross_entropy")
    return loss_rows, loss_sum


# ------------------------------------------------------------------ attention
def flash_fwd(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, B: int, S: int, *, causal: bool = True,
              scale: Optional[float] = None, want_lse: bool = True):
    """q [B*S, Hq, 128], k/v [B*S, Hkv, 128] (views with unit stride over heads*128)."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    assert D == 128 and T == B * S
    for t in (q, k, v):
        assert t.stride(2) == 1 and t.stride(1) == D and t.dtype == torch.bfloat16
    out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=q.device)
    lse = torch.empty(B, Hq, S, dtype=torch.float32, device=q.device) if want_lse else None
    scale = scale if scale is not None else D ** -0.5
    rc = _L().mlf_flash_fwd(_p(q), _p(k), _p(v), _p(out), _p(lse), B, S, Hq, Hkv, C.c_longlong(q.stride(0)),
                            C.c_longlong(k.stride(0)), C.c_longlong(v.stride(0)), C.c_longlong(Hq * D), C.c_float(scale),
                            int(causal), _st())
    _lib.check(rc, "mlf_flash_fwd")
    return out, lse


def flash_fwd_prefix(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, B: int, Sq: int, Skv: int, *, causal: bool = True,
                     scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the LAST ``Sq`` positions of each sequence over all ``Skv`` keys / values (a prompt chunk over
    its cached prefix plus itself). q [B*Sq, Hq, 128]; k, v [B*Skv, Hkv, 128]; token stride arbitrary."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    assert D == 128 and T == B * Sq and k.shape[0] == B * Skv and v.shape[0] == B * Skv and Skv >= Sq
    for t in (q, k, v):
        assert t.stride(2) == 1 and t.stride(1) == D and t.dtype == torch.bfloat16
    out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=q.device)
    scale = scale if scale is not None else D ** -0.5
    rc = _L().mlf_flash_fwd_prefix(_p(q), _p(k), _p(v), _p(out), None, B, Sq, Skv, Hq, Hkv, C.c_longlong(q.stride(0)),
                                   C.c_longlong(k.stride(0)), C.c_longlong(v.stride(0)), C.c_longlong(Hq * D), C.c_float(scale),
                                   int(causal), _st())
    _lib.check(rc, "mlf_flash_fwd_prefix")
    return out


def flash_fwd_paged(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, B: int, Sq: int, Skv: int, *,
                    causal: bool = True, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of the LAST ``Sq`` positions of each of ``B`` sequences over their ``Skv`` cached tokens, keys and
    values read page by page through ``block_table`` inside the kernel (the chunk's own K / V must already be in the
    cache). q [B*Sq, Hq, 128]; kv_cache [num_blocks, 2, 16, Hkv, 128] bf16; block_table int32 [B, max_blocks]."""
    T, Hq, D = q.shape
    nb, two, bs, Hkv, Dc = kv_cache.shape
    assert D == 128 and Dc == 128 and two == 2 and T == B * Sq and Skv >= Sq
    assert q.stride(2) == 1 and q.stride(1) == D and q.dtype == torch.bfloat16 and kv_cache.dtype == torch.bfloat16
    assert kv_cache.is_contiguous() and block_table.dtype == torch.int32 and block_table.dim() == 2 and block_table.shape[0] == B
    table = block_table.contiguous()
    out = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=q.device)
    scale = scale if scale is not None else D ** -0.5
    rc = _L().mlf_flash_fwd_paged(_p(q), _p(kv_cache), _p(table), _p(out), None, B, Sq, Skv, Hq, Hkv, C.c_longlong(q.stride(0)),
                                  C.c_longlong(Hq * D), int(nb), int(bs), int(table.shape[1]), C.c_float(scale), int(causal), _st())
    _lib.check(rc, "mlf_flash_fwd_paged")
    return out


def flash_bwd(q, k, v, o, dout, lse, B: int, S: int, *, causal: bool = True, scale: Optional[float] = None,
              dq: Optional[torch.Tensor] = None, dk: Optional[torch.Tensor] = None, dv: Optional[torch.Tensor] = None):
    """Gradients of :func:`flash_fwd`. ``dq/dk/dv`` may be views into a packed dQKV buffer."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    assert D == 128 and T == B * S
    dout = dout if (dout.stride(2) == 1 and dout.stride(1) == D) else dout.contiguous()
    for t in (q, k, v, o, dout):
        assert t.stride(2) == 1 and t.stride(1) == D and t.dtype == torch.bfloat16
    dq = torch.empty(T, Hq, D, dtype=torch.bfloat16, device=q.device) if dq is None else dq
    dk = torch.empty(T, Hkv, D, dtype=torch.bfloat16, device=q.device) if dk is None else dk
    dv = torch.empty(T, Hkv, D, dtype=torch.bfloat16, device=q.device) if dv is None else dv
    scale = scale if scale is not None else D ** -0.5
    L = _L()
    L.mlf_flash_bwd_scratch_bytes.restype = C.c_longlong
    sc = scratch("flash_bwd", L.mlf_flash_bwd_scratch_bytes(B, S, Hq), q.device)
    ll = C.c_longlong
    rc = L.mlf_flash_bwd(_p(q), _p(k), _p(v), _p(o), _p(dout), _p(lse), _p(dq), _p(dk), _p(dv), _p(sc), B, S, Hq, Hkv,
                         ll(q.stride(0)), ll(k.stride(0)), ll(v.stride(0)), ll(o.stride(0)), ll(dout.stride(0)),
                         ll(dq.stride(0)), ll(dk.stride(0)), ll(dv.stride(0)), C.c_float(scale), int(causal), _st())
    _lib.check(rc, "mlf_flash_bwd")
    return dq, dk, dv


# ------------------------------------------------------------------ paged attention / KV cache
_Q8 = {torch.float8_e4m3fn: 0, torch.int8: 1}
_TYPES = {"p": C.c_void_p, "l": C.c_longlong, "i": C.c_int, "f": C.c_float, "u": C.c_uint64}


def _function(name: str, types: str):
    """Entry ``name`` of the library with its argument types, one letter each: plain numbers are then converted by the call itself,
    which takes a quarter of the time that an object for each of twenty arguments took (decode step of one sequence: 4 us)."""
    f = getattr(_L(), name)
    if f.argtypes is None:
        f.argtypes = [_TYPES[c] for c in types]
    return f


def _at(t: Optional[torch.Tensor]) -> Optional[int]:
    return t.data_ptr() if t is not None else None


def _stream(device_index: int) -> int:
    return torch._C._cuda_getCurrentRawStream(device_index)


def _on_current_device(what: str, *tensors: Optional[torch.Tensor]) -> int:
    """Launches go to the current device's stream: tensors of another device, or of the host, are refused. The device's index."""
    here = torch._C._cuda_getDevice() if torch.cuda.is_initialized() else 0
    for t in tensors:
        if t is not None and t.get_device() != here:
            raise ValueError(f"{what}: a tensor is on {t.device}, the kernel runs on the current CUDA device")
    return here


def _q8_cache(what: str, kv_cache: torch.Tensor, kv_scale: Optional[torch.Tensor]) -> Tuple[int, int, int, int]:
    """Format, num_blocks, block_size and Hkv of an 8-bit cache [num_blocks, 2, block_size, Hkv, 128] with its scales [num_blocks, 2, Hkv]."""
    fmt = _Q8.get(kv_cache.dtype)
    if fmt is None:
        raise TypeError(f"{what}: scales belong to a cache of torch.float8_e4m3fn or torch.int8, not {kv_cache.dtype}")
    shape = kv_cache.shape
    nb, two, bs, Hkv, D = shape if len(shape) == 5 else (0,) * 5
    if two != 2 or D != 128 or not kv_cache.is_contiguous():
        raise ValueError(f"{what}: the cache must be contiguous [num_blocks, 2, block_size, kv_heads, 128], got {tuple(shape)}")
    if kv_scale is None:
        raise ValueError(f"{what}: a cache of {kv_cache.dtype} needs kv_scale")
    if kv_scale.shape != (nb, 2, Hkv) or kv_scale.dtype != torch.float32 or not kv_scale.is_contiguous():
        raise ValueError(f"{what}: kv_scale must be contiguous float32 {(nb, 2, Hkv)}, got {kv_scale.dtype} {tuple(kv_scale.shape)}")
    return fmt, nb, bs, Hkv


def _index(what: str, name: str, t: torch.Tensor, dtype, *shape: int) -> torch.Tensor:
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{what}: {name} must be {dtype} {shape}, got {t.dtype} {tuple(t.shape)}")
    return t.contiguous()


def _heads(what: str, name: str, t: torch.Tensor, H: Optional[int] = None) -> torch.Tensor:
    """bf16 [T, H, 128] whose tokens are whole rows at any pitch."""
    shape = t.shape
    if len(shape) != 3 or shape[2] != 128 or (H is not None and shape[1] != H) or t.dtype != torch.bfloat16:
        raise ValueError(f"{what}: {name} must be bfloat16 [tokens, {'heads' if H is None else H}, 128], got {t.dtype} {tuple(shape)}")
    _, head, one = t.stride()
    return t if one == 1 and (head == 128 or shape[1] == 1) else t.contiguous()


def _aligned_rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` with rows that start on 16 bytes: itself where they do."""
    return t if t.data_ptr() % 16 == 0 and t.stride(0) % 8 == 0 else t.clone(memory_format=torch.contiguous_format)


@lru_cache(maxsize=None)
def _sm_count(device_index: int) -> int:
    """SMs of the current device, whose index the caller passes."""
    return int(_L().mlf_sm_count())


def _decode_split(pairs: int, max_seq_len: int, sms: int) -> int:
    """Tokens per split of the decode kernel for ``pairs`` (sequence, KV head) pairs on ``sms`` SMs, three CTAs of it on
    each. As many splits as keep all CTAs resident at once, none when the pairs alone fill the GPU: CTAs of a second round
    start when the short sequences of the first end, and a split costs its start and the merge launch. At least 128 tokens
    per split. (A captured decode step has one split for all lengths of its bucket, whose end is its ``max_seq_len``: 13 x 2500
    run as 16 x 4096, in 3 splits.) us at the longest of 8 KV heads' sequences, lengths from half of it on: 13 x 2500 4 splits 26 (8: 29);
    48 x 1024 none 35 (3: 45); 8 x 4000 6 splits 28 (11: 34).

    A split of more than 1400 tokens takes long enough for its CTA to be alone at the end, above all when one sequence is
    much longer than the others: then what fits two rounds, or three, of resident CTAs (just above a whole number of rounds
    the last one is nearly empty: 16 x 4096 in 3 / 4 / 6 / 7 splits 47 / 58 / 49 / 53). Up to 2048 tokens, pairs that fill two
    thirds of the first round stay whole (40 x 2048 1 / 2 / 3 splits 53 / 57 / 56; 36 x 1500 1 / 3 39 / 38). Counts on both
    sides: 28 x 2048 1 / 3 / 4 splits 46 / 41 / 40, 32 x 4096 1 / 3 / 4 / 5 96 / 82 / 86 / 82, 40 x 4096 1 / 3 / 4
    101 / 103 / 95, 48 x 4096 1 / 3 109 / 112, 64 x 4096 1 / 2 163 / 148; one sequence of 4000 beside others of 300: 20 in
    2 / 5 / 6 splits 39 / 25 / 23, 32 in 1 / 3 / 5 66 / 34 / 28, 48 in 1 / 3 67 / 39, 64 in 1 / 2 73 / 52."""
    splits = most = max(1, -(-max_seq_len // 128))
    for rounds in (1, 2, 3):
        splits = min(max(1, 3 * sms * rounds // pairs), most)
        if max_seq_len <= 1400 * splits or (2 * sms <= pairs <= 3 * sms and max_seq_len <= 2048):
            break
    return -(-max_seq_len // splits)


@lru_cache(maxsize=4096)
def _decode_splits_q8(pairs: int, max_seq_len: int, sms: int, per_sm: int = 3, smaller: bool = True) -> int:
    """Splits of the 8-bit decode kernel for ``pairs`` (sequence, KV head) pairs on ``sms`` SMs: one round of three CTAs
    (``per_sm``: two for more than eight heads a group) on each, of which every one has 128 tokens at least, 256 (all that its warps fetch at once) where that makes more than eight splits,
    and 96 splits at most; none up to 384 tokens, where the merge costs more than it saves. Two of 1500 tokens or more also where
    that makes one round of four ``smaller`` CTAs out of one of three that is two thirds full at most. us with 8 KV heads: 1 x 200 none 4.7
    (2: 5.5); 1 x 700 6 splits 5.3 (1: 8.6, 3: 6.5); 1 x 4000 16 8.6 (8: 9.0, 11: 10.4, 32: 10.1); 8 x 4000 6 18 (2: 31, 4: 21, 16: 24);
    13 x 2500 4 18 (1: 34, 3: 21, 5: 21); 16 x 4096 3 29 (1: 54, 2: 35, 4: 31); 48 x 4096 none 70 (2: 73); 4 x 60001 13 87 (8: 107,
    16: 86); 29 x 1500 2 25 (1: 27), 32 x 4096 2 51 (1: 60), 32 x 16384 2 177 (1: 217), 32 x 1000 none 20 (2: 20), 36 x 4096 2 58 (1: 61);
    one KV head, 1 x 60000 96 20 (32: 22, 64: 19, 200: 23). Groups of 16: 13 x 2500 of 4 heads 5 18 (4: 20, 6: 33, 8: 30), 32 x 4096 2 40 (1: 56,
    3: 57), 64 x 2000 none 34 (2: 47)."""
    most = 1 if max_seq_len <= 384 else max(min(8, -(-max_seq_len // 128)), min(96, -(-max_seq_len // 256)))
    if smaller and 3 * sms < 2 * pairs <= 4 * sms and max_seq_len >= 1500:
        return 2
    return max(1, min(per_sm * sms // pairs, most))


def _decode_q8(what: str, q: torch.Tensor, ldq: int, Hq: int, kv_cache, kv_scale, block_table, seq_lens, slots, max_seq_len: int, scale, split_tokens: int,
               theta: float, inputs_static: bool) -> torch.Tensor:
    """Attention of :func:`paged_decode` (``slots`` None) and :func:`paged_decode_rope` over an 8-bit cache."""
    fmt, nb, bs, Hkv = _q8_cache(what, kv_cache, kv_scale)
    B, rows = q.shape[0], block_table.shape
    if Hkv == 0 or Hq % Hkv or not 0 < Hq // Hkv <= 16:
        raise ValueError(f"{what}: {Hq} query heads over {Hkv} KV heads (groups of 1 to 16)")
    if block_table.dtype != torch.int32 or len(rows) != 2 or rows[0] != B:
        raise ValueError(f"{what}: block_table must be int32 [{B}, max_blocks], got {block_table.dtype} {tuple(rows)}")
    table, lens = block_table.contiguous(), _index(what, "seq_lens", seq_lens, torch.int32, B)
    slots = _index(what, "slots", slots, torch.int64, B) if slots is not None else None
    dev = _on_current_device(what, q, kv_cache, kv_scale, table, lens, slots)
    out = q.new_empty((B, Hq, 128))
    if B == 0:
        return out
    if rows[1] == 0:
        return out.zero_()
    sms, per_sm = _sm_count(dev), 3 if Hq // Hkv <= 8 else 2
    if split_tokens <= 0:
        splits = _decode_splits_q8(B * Hkv, max_seq_len, sms, per_sm, per_sm == 3 and bs % 16 == 0)
    else:
        st = (max(split_tokens, 128) + 127) // 128 * 128
        splits = max(1, (max_seq_len + st - 1) // st)
    # maximum, sum and output of each split; up to eight that are resident at once are merged within the launch
    within = splits <= 8 and (splits == 1 or B * Hkv * splits <= per_sm * sms)
    ws = None if within else torch.empty(B * Hq * splits * 130, dtype=torch.float32, device=q.device)
    rc = _function("mlf_paged_decode_q8", "plppipppppliiiiiiiiffiu")(
        q.data_ptr(), ldq, kv_cache.data_ptr(), kv_scale.data_ptr(), fmt, table.data_ptr(), lens.data_ptr(), _at(slots), out.data_ptr(), _at(ws),
        0 if ws is None else ws.numel(), B, Hq, Hkv, bs, rows[1], nb, max_seq_len, splits,
        scale if scale is not None else 128 ** -0.5, theta, int(inputs_static), _stream(dev))
    _lib.check(rc, "mlf_paged_decode_q8")
    return out


def paged_decode(q: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor,
                 max_seq_len: int, *, scale: Optional[float] = None, split_tokens: int = 512, fused_merge: bool = False,
                 kv_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One query token per sequence against its paged KV cache.

    q [B, Hq, 128]; kv_cache [num_blocks, 2, block_size, Hkv, 128]; block_table int32 [B, max_blocks];
    seq_lens int32 [B] (cached tokens including the current one). ``max_seq_len`` (host int, an upper
    bound of seq_lens) fixes the number of splits so the launch shape does not depend on device data;
    ``split_tokens`` <= 0 picks the split count from the batch size (enough CTAs to fill the GPU).
    ``fused_merge`` lets the last split of each (sequence, kv head) merge the splits inside the same launch instead of
    a second small kernel; it measured slower (57 us against 48 us at batch 64, 576 cached tokens), hence off.

    An 8-bit cache (float8_e4m3fn or int8) comes with ``kv_scale``, float32 [num_blocks, 2, Hkv]: a value is its number times the
    scale of its block, side (K, V) and head. Scales from 2^-60 to 2^60, not powers of two alone; groups of 1 to 16 query heads per KV
    head; the splits are a whole number of blocks each, and ``fused_merge`` changes nothing. A sequence of length 0 gives zeros.
    """
    if kv_scale is not None or kv_cache.dtype in _Q8:
        q = _heads("paged_decode", "q", q)
        if q.data_ptr() % 4 or q.stride(0) % 2:
            q = q.clone(memory_format=torch.contiguous_format)
        return _decode_q8("paged_decode", q, q.stride(0), q.shape[1], kv_cache, kv_scale, block_table, seq_lens, None, int(max_seq_len), scale, split_tokens, 0.0, False)
    B, Hq, D = q.shape
    nb, two, bs, Hkv, D2 = kv_cache.shape
    assert D == 128 and D2 == 128 and two == 2 and kv_cache.is_contiguous()
    assert q.stride(2) == 1 and q.stride(1) == D and q.dtype == torch.bfloat16      # sequence pitch (stride 0) is free
    out = torch.empty(B, Hq, D, dtype=q.dtype, device=q.device)
    L = _L()
    L.mlf_paged_decode_ws_elems.restype = C.c_longlong
    if split_tokens <= 0:
        split_tokens = _decode_split(B * Hkv, max_seq_len, _sm_count(torch._C._cuda_getDevice()))
    st = (max(split_tokens, 128) + 127) // 128 * 128
    splits = max(1, (max_seq_len + st - 1) // st)
    ws = scratch("paged_decode", L.mlf_paged_decode_ws_elems(B, Hq, splits) * 4, q.device) if splits > 1 else None
    scale = scale if scale is not None else D ** -0.5
    ctr = None
    if splits > 1 and fused_merge:        # finished-split counters: zero at creation, left zero by every launch
        key = ("paged_decode_ctr", q.device.index)
        ctr = _scratch.get(key)
        if ctr is None or ctr.numel() < B * Hkv:
            ctr = torch.zeros(max(B * Hkv, 4096), dtype=torch.int32, device=q.device)
            _scratch[key] = ctr
    rc = L.mlf_paged_decode_ld(_p(q), C.c_longlong(q.stride(0)), _p(kv_cache), _p(block_table), _p(seq_lens), _p(out), _p(ws), _p(ctr), B, Hq, Hkv,
                               bs, block_table.shape[1], nb, int(max_seq_len), st, C.c_float(scale), _st())
    _lib.check(rc, "mlf_paged_decode_ld")
    return out


def paged_decode_rope(qkv: torch.Tensor, kv_cache: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor, slots: torch.Tensor,
                      Hq: int, Hkv: int, max_seq_len: int, theta: float, *, scale: Optional[float] = None, split_tokens: int = 0, inputs_static: bool = False,
                      kv_scale: Optional[torch.Tensor] = None) -> torch.Tensor:
    """:func:`rope_kv_write_` at positions ``seq_lens - 1`` followed by :func:`paged_decode` in one launch: ``qkv``
    [B, (Hq + 2 Hkv) * 128] holds the unrotated projection of each sequence's newest token, which ``seq_lens`` counts;
    its key and value go to cache slot ``slots`` (int64, < 0 skips the write). ``qkv`` is left as it is. ``inputs_static``:
    neither the last launch without programmatic overlap nor any launch after it writes ``block_table``, ``seq_lens`` or the
    cached rows of earlier tokens, which may then be read ahead of the kernels before this one.

    With ``kv_scale`` (an 8-bit cache, see :func:`paged_decode`) the new rows are rounded to 8 bits as :func:`kv_cache_write` does
    and attended to as they are then held; ``inputs_static`` speaks of the scales too. A slot is the place of the sequence's newest
    token by its block table, in a block that no other sequence reads (a shared one is copied first): the block's scale may grow."""
    B = qkv.shape[0]
    if kv_scale is not None or kv_cache.dtype in _Q8:
        what = "paged_decode_rope"
        if qkv.dim() != 2 or qkv.dtype != torch.bfloat16 or qkv.shape[1] != (Hq + 2 * Hkv) * 128 or qkv.stride(1) != 1 or kv_cache.shape[3] != Hkv:
            raise ValueError(f"{what}: qkv must be bfloat16 [B, ({Hq} + 2 * {Hkv}) * 128] beside a cache of {Hkv} heads, got {qkv.dtype} {tuple(qkv.shape)}")
        if qkv.data_ptr() % 8 or qkv.stride(0) % 4 or not theta > 0:
            raise ValueError(f"{what}: rows must be 8-byte aligned and theta positive")
        if inputs_static and not (seq_lens.is_contiguous() and block_table.is_contiguous() and slots.is_contiguous()):
            raise ValueError(f"{what}: inputs_static needs contiguous block_table, seq_lens and slots")      # a copy here would write them
        return _decode_q8(what, qkv, qkv.stride(0), Hq, kv_cache, kv_scale, block_table, seq_lens, slots, int(max_seq_len), scale, split_tokens, theta, inputs_static)
    nb, two, bs, Hc, D = kv_cache.shape
    assert D == 128 and two == 2 and Hc == Hkv and kv_cache.is_contiguous() and qkv.shape[1] == (Hq + 2 * Hkv) * D
    assert qkv.stride(1) == 1 and qkv.dtype == torch.bfloat16 and kv_cache.dtype == torch.bfloat16 and slots.dtype == torch.int64
    assert block_table.dtype == torch.int32 and block_table.is_contiguous() and seq_lens.dtype == torch.int32
    assert not inputs_static or (seq_lens.is_contiguous() and slots.is_contiguous())      # a copy here would write them
    out = torch.empty(B, Hq, D, dtype=qkv.dtype, device=qkv.device)
    L = _L()
    L.mlf_paged_decode_ws_elems.restype = C.c_longlong
    if split_tokens <= 0:
        split_tokens = _decode_split(B * Hkv, max_seq_len, _sm_count(torch._C._cuda_getDevice()))
    st = (max(split_tokens, 128) + 127) // 128 * 128
    splits = max(1, (max_seq_len + st - 1) // st)
    ws = torch.empty(int(L.mlf_paged_decode_ws_elems(B, Hq, splits)), dtype=torch.float32, device=qkv.device) if splits > 1 else None
    seq_lens, slots = seq_lens.contiguous(), slots.contiguous()
    rc = L.mlf_paged_decode_rope(_p(qkv), C.c_longlong(qkv.stride(0)), _p(kv_cache), _p(block_table), _p(seq_lens), _p(slots), _p(out), _p(ws), B, Hq, Hkv, bs,
                                 block_table.shape[1], nb, int(max_seq_len), st, C.c_float(scale if scale is not None else D ** -0.5), C.c_float(theta), int(inputs_static), _st())
    _lib.check(rc, "mlf_paged_decode_rope")
    return out


def _write_q8(dev: int, kv_cache, kv_scale, layout: Tuple[int, int, int, int], k: int, v: int, slots: torch.Tensor, T: int, ldk: int, ldv: int):
    """T rows at the addresses ``k`` and ``v``, checked by the callers."""
    fmt, nb, bs, Hkv = layout
    where = kv_cache.new_empty(nb * bs, dtype=torch.int32) if T > 2048 or bs > 64 else None
    rc = _function("mlf_kv_write_q8", "ppippppliiillu")(kv_cache.data_ptr(), kv_scale.data_ptr(), fmt, k, v, slots.data_ptr(), _at(where), T, Hkv, bs, nb,
                                                        ldk, ldv, _stream(dev))
    _lib.check(rc, "mlf_kv_write_q8")


def kv_cache_write(kv_cache: torch.Tensor, k: torch.Tensor, v: torch.Tensor, slots: torch.Tensor, kv_scale: Optional[torch.Tensor] = None):
    """Scatter k, v [T, Hkv, 128] into cache slots (slot = block * block_size + offset; < 0 skips).

    With ``kv_scale`` (an 8-bit cache, see :func:`paged_decode`) rows are rounded to numbers of 8 bits, ties to even, under one scale for
    each block, side and head: the smallest power of two, from 2^-40 to 2^40, under which the largest magnitude fits (448 for e4m3,
    127 for int8; larger values than 2^40 allows become the largest number). A call that writes a block's first row starts
    the block anew: rows of it that the call does not write lose their meaning. A call that writes later rows only keeps the
    larger of the block's scale and their own, and rounds the rows that the block holds to it. Rows of one block may
    stand anywhere in the list; a slot given twice keeps one of its rows, whole. NaN stays NaN in e4m3 and becomes 0 in int8."""
    if kv_scale is not None or kv_cache.dtype in _Q8:
        what = "kv_cache_write"
        fmt, nb, bs, Hkv = _q8_cache(what, kv_cache, kv_scale)
        k, v = _aligned_rows(_heads(what, "k", k, Hkv)), _aligned_rows(_heads(what, "v", v, Hkv))
        T = k.shape[0]
        if v.shape[0] != T:
            raise ValueError(f"{what}: {T} keys and {v.shape[0]} values")
        slots = _index(what, "slots", slots, torch.int64, T)
        dev = _on_current_device(what, kv_cache, kv_scale, k, v, slots)
        if T > 0 and kv_cache.numel() > 0:
            _write_q8(dev, kv_cache, kv_scale, (fmt, nb, bs, Hkv), k.data_ptr(), v.data_ptr(), slots, T, k.stride(0), v.stride(0))
        return
    nb, _, bs, Hkv, D = kv_cache.shape
    T = k.shape[0]
    assert k.stride(2) == 1 and k.stride(1) == D and v.stride(2) == 1 and v.stride(1) == D
    slots = slots.contiguous()
    rc = _L().mlf_kv_cache_write(_p(kv_cache), _p(k), _p(v), _p(slots), C.c_longlong(T), Hkv, bs, nb,
                                 C.c_longlong(k.stride(0)), C.c_longlong(v.stride(0)), _st())
    _lib.check(rc, "mlf_kv_cache_write")


def rope_kv_write_(qkv: torch.Tensor, pos: torch.Tensor, slots: torch.Tensor, kv_cache: torch.Tensor, Hq: int, Hkv: int, theta: float,
                   kv_scale: Optional[torch.Tensor] = None):
    """In place on packed ``qkv`` [T, (Hq + 2 Hkv) * 128]: rotary embedding of the query and key heads; the rotated
    keys and the values are also written to their cache slots (one launch). With ``kv_scale`` (an 8-bit cache) the write is
    :func:`kv_cache_write`'s, in launches of its own, and rows must be 16-byte aligned."""
    if kv_scale is not None or kv_cache.dtype in _Q8:
        what = "rope_kv_write_"
        layout = _q8_cache(what, kv_cache, kv_scale)
        T = qkv.shape[0]
        if qkv.dim() != 2 or qkv.dtype != torch.bfloat16 or qkv.shape[1] != (Hq + 2 * Hkv) * 128 or qkv.stride(1) != 1 or layout[3] != Hkv:
            raise ValueError(f"{what}: qkv must be bfloat16 [T, ({Hq} + 2 * {Hkv}) * 128] beside a cache of {Hkv} heads, got {qkv.dtype} {tuple(qkv.shape)}")
        if qkv.data_ptr() % 16 or qkv.stride(0) % 8:
            raise ValueError(f"{what}: rows must be 16-byte aligned")
        pos, slots = _index(what, "pos", pos, torch.int64, T), _index(what, "slots", slots, torch.int64, T)
        dev = _on_current_device(what, qkv, pos, slots, kv_cache, kv_scale)
        if T == 0:
            return qkv
        rope_qkv(qkv, pos, Hq, Hkv, theta, out=qkv)
        if kv_cache.numel() > 0:
            k = qkv.data_ptr() + Hq * 256
            _write_q8(dev, kv_cache, kv_scale, layout, k, k + Hkv * 256, slots, T, qkv.stride(0), qkv.stride(0))
        return qkv
    nb, _, bs, Hc, D = kv_cache.shape
    assert D == 128 and Hc == Hkv and qkv.dim() == 2 and qkv.stride(1) == 1 and qkv.shape[1] == (Hq + 2 * Hkv) * 128
    assert qkv.dtype == torch.bfloat16 and pos.dtype == torch.int64 and slots.dtype == torch.int64
    pos, slots = pos.contiguous(), slots.contiguous()
    rc = _L().mlf_rope_kv_write(_p(qkv), C.c_longlong(qkv.stride(0)), _p(pos), _p(slots), _p(kv_cache),
                                C.c_longlong(qkv.shape[0]), Hq, Hkv, bs, nb, C.c_float(theta), _st())
    _lib.check(rc, "mlf_rope_kv_write")
    return qkv


def kv_gather(kv_cache: torch.Tensor, block_table_row: torch.Tensor, length: int, kv_scale: Optional[torch.Tensor] = None):
    """Contiguous (k, v) [length, Hkv, 128] of one sequence from its pages; in bf16 the values of an 8-bit cache (``kv_scale``)."""
    if kv_scale is not None or kv_cache.dtype in _Q8:
        what = "kv_gather"
        fmt, nb, bs, Hkv = _q8_cache(what, kv_cache, kv_scale)
        length, entries = int(length), block_table_row.numel()
        row = _index(what, "block_table_row", block_table_row, torch.int32, entries)
        if not 0 <= length <= entries * bs:
            raise ValueError(f"{what}: {length} tokens, {entries} block-table entries of {bs}")
        dev = _on_current_device(what, kv_cache, kv_scale, row)
        k = kv_cache.new_empty((length, Hkv, 128), dtype=torch.bfloat16)
        v = torch.empty_like(k)
        if length:
            rc = _function("mlf_kv_gather_q8", "ppipiiiiippu")(
                kv_cache.data_ptr(), kv_scale.data_ptr(), fmt, row.data_ptr(), entries, length, Hkv, bs, nb, k.data_ptr(), v.data_ptr(), _stream(dev))
            _lib.check(rc, "mlf_kv_gather_q8")
        return k, v
    nb, _, bs, Hkv, D = kv_cache.shape
    k = torch.empty(length, Hkv, D, dtype=kv_cache.dtype, device=kv_cache.device)
    v = torch.empty_like(k)
    row = block_table_row.contiguous()
    rc = _L().mlf_kv_gather(_p(kv_cache), _p(row), int(row.numel()), int(length), Hkv, bs, nb, _p(k), _p(v), _st())
    _lib.check(rc, "mlf_kv_gather")
    return k, v


def kv_copy_blocks_(tensors: Sequence[torch.Tensor], pairs: Sequence[Tuple[int, int]]):
    """``t[dst] = t[src]`` for every tensor (a layer's cache, or its scales; any type, ``[num_blocks, ...]`` alike) and every
    (src, dst) of ``pairs``, in one launch for up to 64 tensors and 384 pairs. The pairs are host numbers. A block is written once
    at most and none is both read and written, so that no order of the copies matters; anything else is refused."""
    tensors = list(tensors)
    flat = array("i", chain.from_iterable(pairs))
    if not set(map(len, pairs)) <= {2}:
        raise ValueError("kv_copy_blocks_: pairs must be (source, destination) block numbers")
    if not tensors or not flat:
        return
    # one property of all tensors after the other: a third of the time of all properties of one tensor after the other
    T = torch.Tensor
    sizes = array("q", map(attrgetter("nbytes"), tensors))
    nb = tensors[0].size(0) if tensors[0].dim() else 0
    if 0 in sizes or not all(map(T.is_contiguous, tensors)) or any(len(s) == 0 or s[0] != nb for s in set(map(attrgetter("shape"), tensors))):
        raise ValueError(f"kv_copy_blocks_: tensors must be contiguous with the same number of blocks, got {[tuple(t.shape) for t in tensors]}")
    dev = _on_current_device("kv_copy_blocks_", tensors[0])
    if set(map(T.get_device, tensors)) != {dev}:
        _on_current_device("kv_copy_blocks_", *tensors)
    bases = array("Q", map(T.data_ptr, tensors))
    rc = _function("mlf_kv_copy_blocks", "ppipiiu")(bases.buffer_info()[0], sizes.buffer_info()[0], len(tensors), flat.buffer_info()[0], len(pairs), nb, _stream(dev))
    _lib.check(rc, "mlf_kv_copy_blocks")


def argmax_rows(logits: torch.Tensor, vocab: int) -> torch.Tensor:
    """Greedy sampling: int64 argmax over the first ``vocab`` columns of bf16 ``logits`` [rows, ld]."""
    assert logits.dim() == 2 and logits.stride(1) == 1 and logits.dtype == torch.bfloat16
    out = torch.empty(logits.shape[0], dtype=torch.int64, device=logits.device)
    rc = _L().mlf_argmax_rows(_p(logits), C.c_longlong(logits.shape[0]), C.c_longlong(logits.stride(0)), int(vocab), _p(out), _st())
    _lib.check(rc, "mlf_argmax_rows")
    return out


def sample_rows(logits: torch.Tensor, vocab: int, u: torch.Tensor, temperature: torch.Tensor, top_k: Optional[torch.Tensor] = None,
                top_p: Optional[torch.Tensor] = None, min_p: Optional[torch.Tensor] = None, want_logprobs: bool = False):
    """Next tokens (int64 [rows]) from the first ``vocab`` columns (up to 2^20) of ``logits`` [rows, ld], bf16 or fp32, each row with settings of its own:
    ``temperature`` (float32; below 2^-90: the largest logit; at most 2^90), ``top_k`` (int32; 0 or less: no limit), ``top_p`` (1 or more: no limit) and
    ``min_p`` (0 or less: no limit; float32 each). ``u``: a random number of [0, 1) per row, float32.

    With w_i = exp((x_i - max x) / temperature), in the order of x (of equal ones the lower index first): the first top_k tokens
    are kept; of these the shortest prefix whose weights reach top_p of theirs; of these those with w_i >= min_p; the first one in any
    case. The token is the first one, by index, at which the running sum of the kept weights exceeds u times their total. A row gives the same token
    whatever stands in the other rows. Weights are multiples of 2^-40 of the largest: a border between two tokens lies within 2^-28 +
    vocab * 2^-41 of the total from its place, and what weighs less than 2^-41 is never drawn. NaN counts as -inf; a row without any other logit gives token 0. With
    ``want_logprobs``: (tokens, logprobs), float32 [rows], the logarithm of the token's probability among the kept ones (0 for
    the largest logit alone, -inf for a row of -inf)."""
    what, vocab = "sample_rows", int(vocab)
    if logits.dim() != 2 or logits.dtype not in (torch.bfloat16, torch.float32) or not 0 < vocab <= logits.shape[1]:
        raise ValueError(f"{what}: logits must be bfloat16 or float32 [rows, at least {vocab}], got {logits.dtype} {tuple(logits.shape)}")
    rows = logits.shape[0]
    if logits.stride(1) != 1:
        logits = logits.contiguous()
    u, temperature = _index(what, "u", u, torch.float32, rows), _index(what, "temperature", temperature, torch.float32, rows)
    top_k = _index(what, "top_k", top_k, torch.int32, rows) if top_k is not None else None
    top_p = _index(what, "top_p", top_p, torch.float32, rows) if top_p is not None else None
    min_p = _index(what, "min_p", min_p, torch.float32, rows) if min_p is not None else None
    dev = _on_current_device(what, logits, u, temperature, top_k, top_p, min_p)
    tokens = torch.empty(rows, dtype=torch.int64, device=logits.device)
    logprobs = torch.empty(rows, dtype=torch.float32, device=logits.device) if want_logprobs else None
    rc = _function("mlf_sample_rows", "pillipppppppu")(
        logits.data_ptr(), int(logits.dtype == torch.float32), rows, logits.stride(0), vocab, u.data_ptr(), temperature.data_ptr(), _at(top_k),
        _at(top_p), _at(min_p), tokens.data_ptr(), _at(logprobs), _stream(dev))
    _lib.check(rc, "mlf_sample_rows")
    return (tokens, logprobs) if want_logprobs else tokens
