"""Rotary positions of queries and keys, with or without the norm of each head.

``rotary`` turns pairs of columns of each head by an angle that grows with the position
(Su et al., "RoFormer", 2021); ``norm_rotary`` takes the RMS norm of each head's row,
times a weight, in the same pass.  Both take the [B, L, H, d] (or [L, H, d]) tensors of
``masked_attention_via_map``, queries and keys in one launch, and are differentiable.
``rotary_frequencies`` gives the angles per position, scaled for contexts longer than
those a model was trained on.
"""
from __future__ import annotations

import ctypes
import math
import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._operands import DTYPES, launch_on, on_gpu, rows, stream

__all__ = ["rotary_frequencies", "rotary", "norm_rotary"]

LAYOUTS = {"half": 0, "interleaved": 1}
MAX_D = 512


def rotary_frequencies(dim: int, base: float = 10000.0, *, scaling: Optional[str] = None, factor: float = 1.0,
                       context: Optional[int] = None, fast: float = 32.0, slow: float = 1.0, device=None):
    """(inverse frequencies, float64 [dim / 2]; factor of cosines and sines, float).

    Pair i of ``dim`` columns turns by base^(-2 i / dim) per position.  ``scaling`` fits
    a context ``factor`` times longer:

    None      as they are;
    "linear"  all divided by factor (positions are interpolated);
    "ntk"     base times factor^(dim / (dim - 2)): the slowest pair is divided by factor,
              the fastest kept;
    "parts"   pairs that turn fewer than ``slow`` times over the original ``context``
              are divided by factor, those that turn more than ``fast`` times kept, in
              between a ramp over the logarithm of the turns; the second result is then
              0.1 ln(factor) + 1, otherwise 1 (Peng et al., "YaRN", 2023, with the ramp
              over log turns).
    """
    if dim <= 0 or dim % 2:
        raise ValueError(f"dim must be positive and even, got {dim}")
    if not (base > 0 and factor > 0):
        raise ValueError(f"base and factor must be positive, got {base} and {factor}")
    i = torch.arange(0, dim, 2, dtype=torch.float64) / dim
    scale = 1.0
    if scaling == "ntk":
        if dim == 2:
            raise ValueError("scaling 'ntk' needs more than one pair (dim > 2)")
        base = base * factor ** (dim / (dim - 2))
    f = base ** -i
    if scaling == "linear":
        f = f / factor
    elif scaling == "parts":
        if context is None or context <= 0 or not 0 < slow < fast:
            raise ValueError("scaling 'parts' needs context > 0 and 0 < slow < fast")
        turns = context * f / (2 * math.pi)
        keep = ((turns / slow).log() / math.log(fast / slow)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1 - keep)
        scale = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "ntk"):
        raise ValueError(f"scaling must be None, 'linear', 'ntk' or 'parts', got {scaling!r}")
    return f.to(device), scale


# mattn_rotary as one record: sizes and types, eps and scale, strides, pointers
_RECORD = struct.Struct("=12i2f20q10Q")
assert _RECORD.size == ctypes.sizeof(_lib.MattnRotary)


class _Call:
    """One call's tensors and options, as mattn_rotary takes them."""

    def __init__(self, xs, positions, inv_freq, layout, scale, norm, weights, eps):
        self.positions, self.inv_freq, self.layout, self.scale = positions, inv_freq, layout, scale
        self.norm, self.weights, self.eps = norm, weights, eps
        self.device = xs[0].device

    def record(self, xs, ys, gs=None, inverse=False):
        B, L, H, D = xs[0].shape
        two = len(xs) == 2
        dense = (0, 0, 0)

        def strides(ts):
            return (*ts[0].stride()[:3], *(ts[1].stride()[:3] if two else dense)) if ts else (*dense, *dense)

        def pointers(ts):
            return (ts[0].data_ptr(), ts[1].data_ptr() if two else 0) if ts else (0, 0)

        pos, f = self.positions, self.inv_freq
        w = [0 if x is None else x.data_ptr() for x in self.weights] if self.norm else [0, 0]
        return _lib.MattnRotary.from_buffer_copy(_RECORD.pack(
            B, L, D, 0 if f is None else 2 * f.numel(), len(xs), H, xs[1].shape[2] if two else 0, DTYPES[xs[0].dtype],
            self.layout, inverse, self.norm, 0 if pos is None else pos.element_size(), self.eps, self.scale,
            *((0, 0) if pos is None else pos.stride() if pos.dim() == 2 else (0, pos.stride(0))),
            *strides(xs), *strides(ys), *strides(gs), *pointers(xs), *pointers(ys), *pointers(gs),
            w[0], w[1] if two else 0, 0 if pos is None else pos.data_ptr(), 0 if f is None else f.data_ptr()))

    def forward(self, xs, inverse=False):
        ys = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs]
        live = [t for t, x in enumerate(xs) if x.numel()]
        if live:
            p = self.only(live).record([xs[t] for t in live], [ys[t] for t in live], inverse=inverse)
            with launch_on(self.device):
                _lib.check(_lib.load().mattn_rotary_fwd(ctypes.byref(p), stream(self.device)), "mattn_rotary_fwd")
        return ys

    def backward(self, xs, gs, weights_too):
        """Gradients of the inputs and, where weights_too, of the weights (float32)."""
        if not self.norm:  # (of a linear map that keeps lengths: the turn back)
            return self.forward(gs, inverse=True), None
        ys = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in xs]
        live = [t for t, x in enumerate(xs) if x.numel()]
        # (a tensor of no rows is left out of the launch, and its weight's gradient zero)
        dw = [(torch.empty if x.numel() else torch.zeros)(x.shape[3], dtype=torch.float32, device=x.device) if weights_too else None
              for x in xs]
        if live:
            lib = _lib.load()
            p = self.only(live).record([xs[t] for t in live], [ys[t] for t in live], [gs[t] for t in live])
            nws = lib.mattn_norm_rotary_bwd_workspace_bytes(ctypes.byref(p))
            ws = torch.empty(nws, dtype=torch.uint8, device=self.device)
            d = [dw[t].data_ptr() if weights_too else None for t in live]
            with launch_on(self.device):
                _lib.check(lib.mattn_norm_rotary_bwd(ctypes.byref(p), d[0], d[1] if len(d) > 1 else None, ws.data_ptr(),
                                                     nws, stream(self.device)), "mattn_norm_rotary_bwd")
        return ys, dw

    def only(self, live):
        """The call with the tensors ``live`` alone."""
        if len(live) == 2 or not self.norm:
            return self
        c = object.__new__(_Call)
        c.__dict__.update(self.__dict__, weights=[self.weights[t] for t in live])
        return c


class _Rotary(torch.autograd.Function):
    """Residuals: nothing but the angles' inputs, and with the norm x and the weights
    (the statistics are formed again from x, which the backward reads in any case)."""

    @staticmethod
    def forward(ctx, call, n, *tensors):
        xs = tensors[:n]
        ctx.call, ctx.n = call, n
        # (angles and weights too: a change in place before the backward is an error)
        ctx.save_for_backward(call.positions, call.inv_freq, *tensors[n:], *(xs if call.norm else ()))
        ctx.given = [w if w is None else w.dtype for w in tensors[n:]]
        return tuple(call.forward(xs))

    @staticmethod
    @once_differentiable
    def backward(ctx, *gs):
        gs = [rows(g) for g in gs]
        saved = ctx.saved_tensors  # (read in any case: that is where a changed one is noticed)
        xs = saved[-ctx.n:] if ctx.call.norm else gs
        weights_too = any(ctx.needs_input_grad[2 + ctx.n:])
        dx, dw = ctx.call.backward(xs, gs, weights_too)
        dws = [None if dt is None or not weights_too else w.to(dt) for dt, w in zip(ctx.given, dw or [None] * len(ctx.given))]
        return (None, None, *dx, *dws)


def _rotate(name, q, k, weights, positions, inv_freq, layout, scale, norm, eps):
    xs = [q] if k is None else [q, k]
    given = [w for w in (weights if norm else ()) if w is not None]
    three = q.dim() == 3
    for x in xs:
        if x.dim() not in (3, 4) or (x.dim() == 3) != three:
            raise ValueError(f"{name}: q and k must both be [B, L, H, d] or [L, H, d], got {[tuple(x.shape) for x in xs]}")
    if three:
        xs = [x[None] for x in xs]
    B, L, _, D = xs[0].shape
    if any(x.shape[:2] != (B, L) or x.shape[3] != D for x in xs):
        raise ValueError(f"{name}: q and k must agree in batch, length and head dimension, got {[tuple(x.shape) for x in xs]}")
    if xs[0].dtype not in DTYPES or xs[-1].dtype != xs[0].dtype:
        raise TypeError(f"{name}: q and k must have one dtype of {[str(t) for t in DTYPES]}, got {[x.dtype for x in xs]}")
    if D > MAX_D or D == 0:
        raise NotImplementedError(f"{name}: head dimension {D} is not supported (1 to {MAX_D})")
    if layout not in LAYOUTS:
        raise ValueError(f"{name}: layout must be 'half' or 'interleaved', got {layout!r}")
    if not abs(scale) < 3.4028235677973366e38:
        raise ValueError(f"{name}: scale must be a finite float32, got {scale}")
    if inv_freq is None:
        if not norm:
            raise ValueError(f"{name} needs inv_freq")
    else:
        if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1:
            raise TypeError(f"{name}: inv_freq must be a float64 vector (rotary_frequencies), got {inv_freq.dtype} {tuple(inv_freq.shape)}")
        if 2 * inv_freq.numel() > D:
            raise ValueError(f"{name}: {inv_freq.numel()} pairs do not fit a head dimension of {D}")
        inv_freq = inv_freq.detach().contiguous()
    if positions is not None:
        if positions.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"{name}: positions must be int32 or int64, got {positions.dtype}")
        if tuple(positions.shape) not in ((L,), (B, L)):
            raise ValueError(f"{name}: positions must be [{L}] or [{B}, {L}], got {tuple(positions.shape)}")
    for w in given:
        if w.shape != (D,) or w.dtype not in DTYPES:
            raise ValueError(f"{name}: weights must be [{D}] of a floating dtype, got {w.dtype} {tuple(w.shape)}")
    if norm and not 0 <= eps < 3.4028235677973366e38:
        raise ValueError(f"{name}: eps must be a finite float32 and not negative, got {eps}")
    on_gpu(name, *xs, positions, inv_freq, *given)
    xs = [rows(x) for x in xs]
    w32 = [None if w is None else w.detach().float().contiguous() for w in weights[: len(xs)]] if norm else None
    call = _Call(xs, positions, inv_freq, LAYOUTS[layout], float(scale), norm, w32, float(eps))
    if torch.is_grad_enabled() and any(x.requires_grad for x in (*xs, *given)):
        out = _Rotary.apply(call, len(xs), *xs, *(weights[: len(xs)] if norm else ()))
    else:
        out = call.forward(xs)
    if three:
        out = [y[0] for y in out]
    return out[0] if k is None else tuple(out)


def rotary(q: torch.Tensor, k: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *,
           inv_freq: torch.Tensor, layout: str = "half", scale: float = 1.0):
    """q (and k) with the pairs of their first 2 * len(inv_freq) columns turned by
    position * inv_freq and scaled by ``scale``; the columns behind them as they are.

    q, k: [B, L, Hq, d] and [B, L, Hk, d] (or [L, H, d]), one dtype (bfloat16, float16
        or float32), d <= 512, any strides; the results are dense, of the same dtype.
    positions: int32 or int64, [L] or [B, L]; None: 0 .. L - 1.  Any value: of packed
        documents, of tokens far into a cache, negative ones.
    inv_freq, scale: rotary_frequencies' results (inv_freq on q's device).
    layout: "half" pairs the columns (i, i + dim / 2), "interleaved" (2 i, 2 i + 1).

    Returns q' (k None) or (q', k'), differentiable once w.r.t. q and k.  Angles are
    formed in float64 (far positions keep theirs), products in float32.
    """
    return _rotate("rotary", q, k, None, positions, inv_freq, layout, scale, False, 0.0)


def norm_rotary(q: torch.Tensor, k: Optional[torch.Tensor] = None, q_weight: Optional[torch.Tensor] = None,
                k_weight: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, *,
                inv_freq: Optional[torch.Tensor] = None, layout: str = "half", scale: float = 1.0, eps: float = 1e-6):
    """``rotary`` of the RMS norm of each head's row: x (mean x^2 + eps)^-1/2 times the
    weight, statistics in float32, rounded once at the end.

    q_weight, k_weight: [d], float32 or a 16-bit dtype (None: ones); their gradients are
        summed in float32 in a fixed order and returned in their dtype.
    inv_freq None: the norm alone.  Other arguments as for ``rotary``.  Differentiable
    once w.r.t. q, k and the weights.
    """
    return _rotate("norm_rotary", q, k, (q_weight, k_weight), positions, inv_freq, layout, scale, True, eps)
