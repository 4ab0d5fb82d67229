"""Rotary positions: the step between a layer's projections and its attention.

Every pair (x, y) of the rotated part of a head is turned by its row's position times the pair's frequency,

    (x, y) -> magnitude * (x cos t - y sin t,  y cos t + x sin t),     t = position * frequencies[i],

the pairs being (i, i + rotary_dim / 2), or (2i, 2i + 1) with `interleaved`; elements from rotary_dim on stay as they are.
One kernel turns up to four tensors (Q and K, or the Q, K1 and K2 of a 2-simplicial layer) with different head counts, read
where a fused projection left them.  Angles are formed in 64 bits from the position itself: no table, any position.  The
gradient is the rotation by the negative angle.

The scores of ordinary attention then depend on the distance of two rows only.  The 2-simplicial scores are products of
three rows and have no such invariance: there a rotation makes them depend on the positions themselves.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Sequence, Union

import torch

from . import _abi
from .simplicial_attn import _DTYPES, _native, _unit_inner

MAX_TENSORS = 4


def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: Optional[str] = None, factor: float = 1.0,
                       original_length: Optional[int] = None, low_turns: float = 1.0, high_turns: float = 32.0,
                       device=None) -> torch.Tensor:
    """float64 [rotary_dim / 2] frequencies in radians per position, base ** (-2i / rotary_dim), scaled for contexts `factor`
    times as long as the `original_length` a model was trained on:

    "linear"  every frequency is divided by `factor` (positions are interpolated);
    "base"    the base grows by factor ** (rotary_dim / (rotary_dim - 2)), so that the lowest frequency is divided by `factor`;
    "parts"   a frequency that makes fewer than `low_turns` turns in the original length is divided by `factor`, one with more
              than `high_turns` stays, in between the share that stays grows linearly with the turns.
    """
    if rotary_dim < 2 or rotary_dim % 2 != 0:
        raise ValueError(f"rotary_dim must be even and positive, got {rotary_dim}")
    if not (base > 0 and factor > 0 and math.isfinite(base) and math.isfinite(factor)):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    if scaling == "base":
        if rotary_dim == 2:
            raise ValueError('scaling "base" needs a rotary_dim of at least 4')
        base = base * factor ** (rotary_dim / (rotary_dim - 2))
    f = [base ** (-2.0 * i / rotary_dim) for i in range(rotary_dim // 2)]
    if scaling == "linear":
        f = [x / factor for x in f]
    elif scaling == "parts":
        if not original_length or original_length < 1:
            raise ValueError('scaling "parts" needs the original_length')
        if not high_turns > low_turns:
            raise ValueError("high_turns must be above low_turns")
        keep = [min(max((x * original_length / (2 * math.pi) - low_turns) / (high_turns - low_turns), 0.0), 1.0) for x in f]
        f = [x * (k + (1 - k) / factor) for x, k in zip(f, keep)]
    elif scaling not in (None, "base"):
        raise ValueError(f"unknown scaling {scaling!r}: None, 'linear', 'base' or 'parts'")
    return torch.tensor(f, dtype=torch.float64, device=device)


def _row_strides(t: torch.Tensor) -> _abi.Strides:
    return _abi.Strides(*t.stride()[:3]) if t.dim() == 4 else _abi.Strides(0, t.stride(0), t.stride(1))


def _call(xs, frequencies, positions, offset, interleaved, magnitude, inverse):
    """The call through ctypes: into new tensors, without a history (what the binding does for plain calls)."""
    x = xs[0]
    if not 1 <= len(xs) <= MAX_TENSORS:
        raise ValueError(f"rotary_positions takes one to four tensors, got {len(xs)}")
    if not x.is_cuda:
        raise RuntimeError("simplical_attn_b200 runs on CUDA tensors only; there is no CPU path")
    if x.dtype not in _DTYPES:
        raise TypeError(f"unsupported dtype {x.dtype}")
    for t in xs:
        if t.dtype != x.dtype or t.device != x.device:
            raise TypeError("the tensors must share dtype and device")
        if t.dim() not in (3, 4) or t.dim() != x.dim() or t.shape[:-2] != x.shape[:-2] or t.shape[-1] != x.shape[-1]:
            raise ValueError(f"the tensors must share every extent but the heads, got {tuple(x.shape)} and {tuple(t.shape)}")
    if frequencies.device != x.device or frequencies.dtype not in (torch.float32, torch.float64):
        raise TypeError("frequencies must be float32 or float64 on the tensors' device")
    if frequencies.dim() != 1 or not 2 <= 2 * frequencies.shape[0] <= x.shape[-1]:
        raise ValueError(f"frequencies must be [rotary_dim / 2] with 2 <= rotary_dim <= head_dim, got {tuple(frequencies.shape)}")
    if positions is not None:
        if positions.device != x.device or positions.dtype not in (torch.int32, torch.int64):
            raise TypeError("positions must be int32 or int64 on the tensors' device")
        if positions.shape != x.shape[-3:-2] and not (x.dim() == 4 and positions.shape == x.shape[:2]):
            raise ValueError(f"positions must be one per row, or [batch, seq_len], got {tuple(positions.shape)} for {tuple(x.shape)}")
    xs = [_unit_inner(t) for t in xs]
    frequencies = frequencies.contiguous()
    with torch.cuda.device(x.device):
        outs = [torch.empty_like(t) for t in xs]
        work = [(t, o) for t, o in zip(xs, outs) if t.numel() != 0]
        if not work:
            return outs
        p = _abi.RotaryParams()
        p.tensors = len(work)
        p.B, p.N, p.D = (x.shape[0] if x.dim() == 4 else 1), x.shape[-3], x.shape[-1]
        p.rotary_dim = 2 * frequencies.shape[0]
        p.interleaved, p.inverse = int(interleaved), int(inverse)
        p.dtype = _DTYPES[x.dtype]
        p.frequency_bits = 64 if frequencies.dtype == torch.float64 else 32
        p.offset, p.magnitude = int(offset), float(magnitude)
        if positions is not None:
            p.position_bits = 64 if positions.dtype == torch.int64 else 32
            p.position_b = positions.stride(0) if positions.dim() == 2 else 0
            p.position_n = positions.stride(-1)
        src, dst = (ctypes.c_void_p * MAX_TENSORS)(), (ctypes.c_void_p * MAX_TENSORS)()
        for i, (t, o) in enumerate(work):
            p.heads[i] = t.shape[-2]
            getattr(p, "in")[i], p.out[i] = _row_strides(t), _row_strides(o)
            src[i], dst[i] = t.data_ptr(), o.data_ptr()
        rc = _abi.load().sa_rotary(ctypes.byref(p), src, dst, 0 if positions is None else positions.data_ptr(), frequencies.data_ptr(),
                                   torch.cuda.current_stream().cuda_stream)
        _abi.check("sa_rotary", rc)
    return outs


class RotaryPositionsFunction(torch.autograd.Function):
    """The history of calls that are not plain (traces, functorch transforms, tensor subclasses)."""

    @staticmethod
    def forward(ctx, frequencies, positions, offset, interleaved, magnitude, inverse, *xs):
        ctx.save_for_backward(frequencies, positions)
        ctx.cfg = (offset, interleaved, magnitude, inverse)
        ctx.set_materialize_grads(False)
        return tuple(_call(xs, frequencies, positions, offset, interleaved, magnitude, inverse))

    @staticmethod
    def backward(ctx, *grads):
        frequencies, positions = ctx.saved_tensors
        offset, interleaved, magnitude, inverse = ctx.cfg
        of = [i for i, g in enumerate(grads) if g is not None and ctx.needs_input_grad[6 + i]]
        out = [None] * len(grads)
        if of:
            for i, g in zip(of, _rotate(tuple(grads[i] for i in of), frequencies, positions, offset, interleaved, magnitude, not inverse)):
                out[i] = g
        return (None,) * 6 + tuple(out)


def _rotate(xs, frequencies, positions, offset, interleaved, magnitude, inverse, out=None):
    native = _native()
    if native is not None:
        r = native.rotary(xs, out, frequencies, positions, offset, interleaved, magnitude, inverse)
        if r is not None:
            return r
    if not all(isinstance(t, torch.Tensor) for t in xs):
        raise TypeError("rotary_positions takes a tensor or a sequence of one to four tensors")
    if torch.is_grad_enabled() and frequencies.requires_grad:
        raise ValueError("there is no gradient for the frequencies")
    if out is not None:
        raise RuntimeError("rotary_positions with out= takes plain tensors, and needs the native binding")
    return RotaryPositionsFunction.apply(frequencies, positions, offset, interleaved, magnitude, inverse, *xs)


def rotary_positions(tensors: Union[torch.Tensor, Sequence[torch.Tensor]], frequencies: torch.Tensor,
                     positions: Optional[torch.Tensor] = None, *, offset: int = 0, interleaved: bool = False,
                     magnitude: float = 1.0, inverse: bool = False, out=None):
    """Rotates one to four tensors [B, N, heads, D] (or packed [T, heads, D]) that share every extent but the heads.

    `frequencies`: float32 or float64 [rotary_dim / 2] radians per position (`rotary_frequencies`), rotary_dim at most 2048.  `positions`: int32 or
    int64, one per row ([N], or [T] of packed rows) or [B, N]; None: rows count from 0.  `offset` is added to either.
    `magnitude` scales the rotated part; `inverse` turns back.  Returns a tensor for a tensor, else a tuple.

    `out` (a tensor, or as many as `tensors`) takes the results; an output may be its input itself, which then is turned in
    place, and must not overlap it otherwise.  Such a call records no gradient and refuses tensors that require one; it needs the
    native binding and plain tensors (no trace, no functorch transform, no subclass).
    """
    one = isinstance(tensors, torch.Tensor)
    xs = (tensors,) if one else tuple(tensors)
    if not xs:
        raise TypeError("rotary_positions takes a tensor or a sequence of one to four tensors")
    if out is not None:
        out = (out,) if isinstance(out, torch.Tensor) else tuple(out)
    r = _rotate(xs, frequencies, positions, offset, interleaved, magnitude, inverse, out)
    return r[0] if one else r


class RotaryPositions(torch.nn.Module):
    """`rotary_positions` with its frequencies as a buffer (not part of the state_dict: they follow from the arguments, which
    are those of `rotary_frequencies`)."""

    def __init__(self, rotary_dim: int, base: float = 10000.0, interleaved: bool = False, scaling: Optional[str] = None,
                 factor: float = 1.0, original_length: Optional[int] = None, low_turns: float = 1.0, high_turns: float = 32.0,
                 magnitude: float = 1.0, device=None):
        super().__init__()
        self.rotary_dim = rotary_dim
        self.interleaved = interleaved
        self.magnitude = magnitude
        self._arguments = (rotary_dim, base, scaling, factor, original_length, low_turns, high_turns)
        self.register_buffer("frequencies", rotary_frequencies(*self._arguments, device), persistent=False)

    def _apply(self, fn, recurse=True):
        # The values are kept whatever becomes of the parameters: in 64 bits under a cast (`.to(dtype)`, `.half()`), as they are under
        # `.to_empty()`, which leaves memory unwritten, and from the arguments where they were on the meta device.
        kept = self.frequencies
        super()._apply(fn, recurse)
        device = self.frequencies.device
        self.frequencies = kept.to(device) if device.type == "meta" or not kept.is_meta else rotary_frequencies(*self._arguments, device)
        return self

    def forward(self, *tensors, positions: Optional[torch.Tensor] = None, offset: int = 0):
        r = rotary_positions(tensors, self.frequencies, positions, offset=offset, interleaved=self.interleaved, magnitude=self.magnitude)
        return r[0] if len(tensors) == 1 else r
