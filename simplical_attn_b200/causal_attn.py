"""Ordinary causal attention, for the layers between a model's 2-simplicial ones.

    logits_ij = scale * Q_i . K_j     over keys j <= i + (keys - queries) of i's sequence
    O_i = sum_j softmax_j(logits_i) V_j

One call serves whole prompts, a chunk of a prompt over the keys before it, single tokens (the last query of a sequence sees
all its keys) and packed sequences of different lengths, with grouped heads.  A query that sees no key, or whose scores are
all -inf, has O = 0.
The layout is the 2-simplicial operator's: [batch, seq_len, heads, head_dim], or packed [rows, heads, head_dim].
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _abi
from . import simplicial_attn as _host
from .simplicial_attn import _ALGOS, _DTYPES, _native, _ptr, _unit_inner
from .rotary import _row_strides


def _check(q, k, v, cu_q, cu_k):
    if not q.is_cuda:
        raise RuntimeError("simplical_attn_b200 runs on CUDA tensors only; there is no CPU path")
    if q.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {q.dtype}")
    packed = cu_q is not None
    if q.dim() != (3 if packed else 4):
        raise ValueError("q must be [batch, seq_len, num_heads, head_dim], or packed [rows, num_heads, head_dim] with cu_q")
    for name, t in (("k", k), ("v", v)):
        if t.dtype != q.dtype or t.device != q.device:
            raise TypeError(f"{name} must match q's dtype and device")
        if t.dim() != q.dim() or t.shape != k.shape or t.shape[-1] != q.shape[-1] or (not packed and t.shape[0] != q.shape[0]):
            raise ValueError(f"{name} must be [batch, key_len, kv_heads, head_dim] (packed: [rows, kv_heads, head_dim]), got {tuple(t.shape)}")
    if k.shape[-2] == 0 or q.shape[-2] == 0 or q.shape[-2] % k.shape[-2] != 0:
        raise ValueError("K and V must have a head count that divides the query head count")
    if q.shape[-1] == 0:
        raise ValueError("head_dim must be positive")
    if not packed:
        if cu_k is not None:
            raise ValueError("cu_k without cu_q")
        return
    for name, cu in (("cu_q", cu_q), ("cu_k", cu_k)):
        if cu.dtype != torch.int32 or cu.device != q.device:
            raise TypeError(f"{name} must be int32 on q's device")
        if cu.dim() != 1 or cu.shape[0] < 2 or cu.shape != cu_q.shape or not cu.is_contiguous():
            raise ValueError(f"{name} must be contiguous [sequences + 1] with at least one sequence, as many as cu_q has")


def _starts_of_keys(q, k, cu_q, cu_k):
    """`cu_k`, which defaults to `cu_q` where the tensors have the same rows."""
    if cu_k is not None or cu_q is None:
        return cu_k
    if k.shape[:1] != q.shape[:1]:
        raise ValueError("without cu_k, k and v must have q's rows")
    return cu_q


def _params(q, k, v, o, cu_q, scale, max_q, max_k, algo):
    p = _abi.CausalParams()
    packed = cu_q is not None
    p.B = 1 if packed else q.shape[0]
    p.Nq, p.Nk, p.H, p.Hkv, p.D = q.shape[-3], k.shape[-3], q.shape[-2], k.shape[-2], q.shape[-1]
    p.sequences = cu_q.shape[0] - 1 if packed else 0
    p.max_q, p.max_k = max_q, max_k
    p.dtype, p.algo, p.scale = _DTYPES[q.dtype], _ALGOS[algo], scale
    p.q, p.k, p.v, p.o = (_row_strides(t) for t in (q, k, v, o))
    return p


def _with_status(size, device):
    """A workspace of `size` bytes behind 256 for the status word."""
    return _host._workspace(256 + size, device)


def causal_attention_fwd(q, k, v, scale, cu_q=None, cu_k=None, max_q=0, max_k=0, algo=None, low=False):
    """Forward launch: (O, LSE), LSE fp32 [B, H, N] (packed: [H, rows]).  With `low` also what rounding took from a 16-bit O
    (None for fp32), which the backward forms sum dO O with: without it dQ and dK are about 5 % less exact."""
    algo = algo or _host.default_algo
    cu_k = _starts_of_keys(q, k, cu_q, cu_k)
    if _host._status_watch.active:
        _host._status_watch.poll(q.device)
    native = _native()
    if native is not None:
        out = native.causal_forward(q, k, v, cu_q, cu_k, scale, max_q, max_k, _ALGOS[algo], low)
        if out is not None:
            if _host.debug_device_status:
                _host._status_watch.flush(q.device)
            return out if low else out[:2]
    _check(q, k, v, cu_q, cu_k)
    lib = _abi.load()
    q, k, v = (_unit_inner(t) for t in (q, k, v))
    with torch.cuda.device(q.device):
        o = torch.empty_like(q)
        lse = torch.empty((*q.shape[:-3], q.shape[-2], q.shape[-3]), device=q.device, dtype=torch.float32)
        if q.numel() == 0 or k.numel() == 0:
            return (o.zero_(), lse.fill_(-math.inf)) + ((None,) if low else ())
        o_low = torch.empty_like(o) if low and q.dtype != torch.float32 else None
        p = _params(q, k, v, o, cu_q, scale, max_q, max_k, algo)
        ws = _with_status(lib.sa_causal_forward_workspace_size(ctypes.byref(p)), q.device)
        sh = torch.cuda.current_stream().cuda_stream
        rc = lib.sa_causal_forward(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(o_low), _ptr(lse), _ptr(cu_q), _ptr(cu_k),
                                   ws.data_ptr() + 256, ws.numel() - 256, _ptr(ws), ctypes.c_void_p(sh))
        _abi.check("sa_causal_forward", rc)
        _host._status(lib, ws, "sa_causal_forward", sh)
    return (o, lse, o_low) if low else (o, lse)


def causal_attention_bwd(q, k, v, o, lse, d_o, scale, cu_q=None, cu_k=None, max_q=0, max_k=0, need=(True, True, True), algo=None, o_low=None):
    """Backward launches: (dq, dk, dv), `None` where `need[i]` is false."""
    algo = algo or _host.default_algo
    cu_k = _starts_of_keys(q, k, cu_q, cu_k)
    if _host._status_watch.active:
        _host._status_watch.poll(q.device)
    native = _native()
    if native is not None:
        bits = sum(1 << i for i, n in enumerate(need) if n)
        grads = native.causal_backward(q, k, v, o, lse, d_o, o_low, cu_q, cu_k, scale, max_q, max_k, _ALGOS[algo], bits)
        if grads is not None:
            if _host.debug_device_status:
                _host._status_watch.flush(q.device)
            return grads
    _check(q, k, v, cu_q, cu_k)
    for t in (o, d_o):
        if t.dtype != q.dtype or t.device != q.device:
            raise TypeError("o and its gradient must match q's dtype and device")
        if t.shape != q.shape:
            raise ValueError("o and its gradient must have q's shape")
    if lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous() or lse.shape != (*q.shape[:-3], q.shape[-2], q.shape[-3]):
        raise ValueError("lse must be the forward's")
    if o_low is not None and (o_low.shape != o.shape or o_low.stride() != o.stride() or o_low.dtype != o.dtype or o_low.device != o.device):
        raise ValueError("o_low must be the forward's")
    lib = _abi.load()
    q, k, v, o, d_o = (_unit_inner(t) for t in (q, k, v, o, d_o))
    with torch.cuda.device(q.device):
        if q.numel() == 0 or k.numel() == 0:
            return tuple(torch.zeros_like(t) if n else None for t, n in zip((q, k, v), need))
        grads = [torch.empty_like(t) if n else None for t, n in zip((q, k, v), need)]
        p = _params(q, k, v, o, cu_q, scale, max_q, max_k, algo)
        p.d_o = _row_strides(d_o)
        p.dq, p.dk, p.dv = (_abi.Strides(0, 0, 0) if g is None else _row_strides(g) for g in grads)
        ws = _with_status(lib.sa_causal_backward_workspace_size(ctypes.byref(p)), q.device)
        sh = torch.cuda.current_stream().cuda_stream
        rc = lib.sa_causal_backward(ctypes.byref(p), _ptr(q), _ptr(k), _ptr(v), _ptr(o), _ptr(o_low), _ptr(lse), _ptr(d_o), *[_ptr(g) for g in grads],
                                    _ptr(cu_q), _ptr(cu_k), ws.data_ptr() + 256, ws.numel() - 256, _ptr(ws), ctypes.c_void_p(sh))
        _abi.check("sa_causal_backward", rc)
        _host._status(lib, ws, "sa_causal_backward", sh)
    return tuple(grads)


class CausalAttentionFunction(torch.autograd.Function):
    """The history of calls that are not plain (traces, functorch transforms, tensor subclasses)."""

    @staticmethod
    def forward(ctx, q, k, v, cu_q, cu_k, scale, max_q, max_k):
        o, lse, o_low = causal_attention_fwd(q, k, v, scale, cu_q, cu_k, max_q, max_k, None, True)
        ctx.save_for_backward(q, k, v, o, lse, o_low, cu_q, cu_k)
        ctx.cfg = (scale, max_q, max_k)
        ctx.mark_non_differentiable(lse)
        return o, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad_output, _):
        q, k, v, o, lse, o_low, cu_q, cu_k = ctx.saved_tensors
        scale, max_q, max_k = ctx.cfg
        need = tuple(bool(n) for n in ctx.needs_input_grad[:3])
        return causal_attention_bwd(q, k, v, o, lse, grad_output, scale, cu_q, cu_k, max_q, max_k, need, o_low=o_low) + (None,) * 5


def causal_attention(q, k, v, scale: Optional[float] = None, *, cu_q: Optional[torch.Tensor] = None,
                     cu_k: Optional[torch.Tensor] = None, max_q: Optional[int] = None, max_k: Optional[int] = None,
                     return_lse: bool = False):
    """O of causal attention, in q's shape; with `return_lse` also the rows' log sum exp (fp32 [B, H, N], packed [H, rows]),
    which carries no gradient.  `scale` defaults to 1/sqrt(head_dim).

    Batched: q [B, N, H, D], k and v [B, M, Hkv, D], H a multiple of Hkv; every batch element is a sequence of N queries and
    M keys.  Packed: q [rows, H, D], k and v [rows, Hkv, D], and int32 device tensors `cu_q`, `cu_k` [sequences + 1] that say
    where sequences start, in order (`cu_k` defaults to `cu_q`): sequence s is rows cu[s] to cu[s + 1].  They are read on the
    device, so a captured call follows what they hold at replay.  `max_q` and `max_k` bound the sequences' lengths; they choose
    kernels and launch shapes, not results.  Rows outside every sequence have O = 0 and zero gradients.

    bf16 and fp16 with a head dim of at most 128 that is a multiple of 8 run on tensor cores; other head dims up to 256, fp32,
    unaligned strides and a scale that is not positive on the CUDA cores.  A few queries over many keys (`max_q` times the
    heads of a K/V head at most 32) have kernels of their own: packed single tokens want `max_q=1`.

    What lies in keys that a query does not see, in rows outside the sequences and in other sequences does not reach a result,
    NaN and infinities included.  The gradients keep to that between sequences; within one, an element that is not finite may reach
    gradients across the mask, at most 254 rows away.  They are written without atomics: equal calls give equal bits.  There is no
    second derivative.  For 16-bit tensors a call with a history keeps, beside Q, K, V, O and the LSE, what rounding took from O: one more
    tensor of O's size until its backward pass.  A backward pass is captured into a graph under torch's own condition, that no eager graph of the same leaves is
    alive.
    """
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() and q.shape[-1] else 1.0
    max_q, max_k = max_q or 0, max_k or 0
    if max_q < 0 or max_k < 0:
        raise ValueError("max_q and max_k must not be negative")
    cu_k = _starts_of_keys(q, k, cu_q, cu_k)
    native = None if _host.debug_device_status else _native()
    if native is not None:
        if _host._status_watch.active:
            _host._status_watch.poll(q.device)
        r = native.causal_attention(q, k, v, cu_q, cu_k, scale, max_q, max_k, _ALGOS[_host.default_algo])
        if r is not None:
            return r if return_lse else r[0]
    r = CausalAttentionFunction.apply(q, k, v, cu_q, cu_k, scale, max_q, max_k)
    return r if return_lse else r[0]
