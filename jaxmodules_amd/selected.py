"""Sparse attention over key blocks that a cheap score selects for each query.

Where ``flex_attention`` takes a ``BlockMask`` that the program knows beforehand, here
the data decide: ``block_means`` forms the mean key of each block, ``select_blocks``
scores every block by the dot product of its mean with the query (summed over the query
heads that share a key head) and keeps the best few, ``selected_attention`` attends to
the keys of those blocks, forward and backward:

    means = block_means(k, 64)
    blocks = select_blocks(q, means, 64, 16)               # int32 [B, N, Hkv, 16]
    o = selected_attention(q, k, v, blocks, 64)

The choice itself carries no gradient.  For tokens served from a cache give ``starts``
(position of the first query of each sequence) and ``lengths`` (keys held), and keep the
means with ``block_means(k, 64, lengths=lengths, out=means, new=tokens)``.

Tensors are [B, L, H, d] as for ``masked_attention_via_map``; query head h reads key
head h // (Hq / Hkv).  There is no CPU code path.
"""
from __future__ import annotations

import ctypes
import itertools
import math
import struct
from typing import Optional

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._operands import DTYPES, launch_on, on_gpu, rows, stream
from .attention import _aligned, _copy_rows, _ready, _rows_like, _workspace

__all__ = ["block_means", "select_blocks", "selected_attention"]

MAX_D = 128
MAX_COUNT = 1024


def _check_block_size(name, block_size):
    if isinstance(block_size, bool) or not isinstance(block_size, int) or block_size <= 0 or block_size % 16:
        raise ValueError(f"{name}: block_size must be a positive multiple of 16, got {block_size!r}")


def _check_heads(name, x, what, dtype=None):
    if x.dim() != 4:
        raise ValueError(f"{name}: {what} must be [B, L, H, d], got {tuple(x.shape)}")
    if x.dtype not in DTYPES or (dtype is not None and x.dtype != dtype):
        raise TypeError(f"{name}: {what} has dtype {x.dtype}" + (f", expected {dtype}" if dtype else ""))
    if not 0 < x.shape[3] <= MAX_D:
        raise NotImplementedError(f"{name}: head dimension {x.shape[3]} is not supported (1 to {MAX_D})")


def _check_sequences(name, B, **tensors):
    for what, t in tensors.items():
        if t is not None and (t.dtype != torch.int32 or tuple(t.shape) != (B,)):
            raise TypeError(f"{name}: {what} must be int32 [{B}], got {t.dtype} {tuple(t.shape)}")


def _dense(t):
    return t if t is None else t.contiguous()


def _ptr(t):
    return None if t is None else t.data_ptr()


def _operand(x):
    """Rows at 16-byte addresses, the columns zero-padded to a multiple of 8."""
    d = x.shape[3]
    if d % 8 == 0:
        return _ready(x)
    y = _rows_like(x, (d + 7) // 8 * 8, False)
    if x.numel():
        with launch_on(x.device):
            _copy_rows([(x, y)])
    return y


def block_means(k: torch.Tensor, block_size: int, lengths: Optional[torch.Tensor] = None, *,
                out: Optional[torch.Tensor] = None, new: Optional[int] = None) -> torch.Tensor:
    """Mean key of each block of ``block_size`` keys: float32 [B, ceil(L / block_size),
    H, d] of k [B, L, H, d] (float64 sums, rounded once).

    lengths: int32 [B], keys held by each sequence (None: L; clamped to [0, L]); a block
        holding fewer keys is averaged over those, one holding none is 0.
    out, new: write into ``out`` (dense) only the blocks that hold one of the last
        ``new`` keys of each sequence, as after appending to a cache; returns out.

    Not differentiable (k's gradient flows through the attention alone).
    """
    name = "block_means"
    _check_block_size(name, block_size)
    _check_heads(name, k, "k")
    B, L, H, d = k.shape
    nblk = -(-L // block_size)
    _check_sequences(name, B, lengths=lengths)
    if (out is None) != (new is None):
        raise ValueError(f"{name}: out and new go together")
    if out is not None:
        if out.dtype != torch.float32 or tuple(out.shape) != (B, nblk, H, d) or not out.is_contiguous():
            raise ValueError(f"{name}: out must be dense float32 {(B, nblk, H, d)}, got {out.dtype} {tuple(out.shape)}")
        if isinstance(new, bool) or not isinstance(new, int) or not 0 <= new <= L:
            raise ValueError(f"{name}: new must be an integer of 0 to {L}, got {new!r}")
    on_gpu(name, k, lengths, out)
    k, lengths = rows(k.detach()), _dense(lengths)
    if out is None:
        out = torch.empty((B, nblk, H, d), dtype=torch.float32, device=k.device)
    if out.numel() == 0 or new == 0:
        return out
    p = _lib.MattnMeans(B=B, L=L, H=H, D=d, dtype=DTYPES[k.dtype], block_size=block_size, new_keys=new or 0,
                        k=k.data_ptr(), means=out.data_ptr(), lengths=_ptr(lengths))
    p.k_stride[:] = k.stride()[:3]
    with launch_on(k.device):
        _lib.check(_lib.load().mattn_block_means(ctypes.byref(p), stream(k.device)), "mattn_block_means")
    return out


def select_blocks(q: torch.Tensor, means: torch.Tensor, block_size: int, count: int, *, is_causal: bool = True,
                  first: int = 1, last: int = 1, starts: Optional[torch.Tensor] = None,
                  lengths: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The blocks each query attends to: int32 [B, N, Hkv, count], ascending, -1 behind.

    q: [B, N, Hq, d]; means: float32 [B, blocks, Hkv, d] (block_means).  Query i of
    sequence b is at position starts[b] + i (None: i) and sees the blocks below
    ceil(lengths[b] / block_size) (None: all) and, with is_causal, those up to its own
    position's.  The ``first`` first and ``last`` last blocks it sees are always among
    its ``count``; the others are the best by (sum of the group's queries) . mean, in
    float64, equal scores by the lower index, NaN lowest.  A query that sees at most
    ``count`` blocks gets them all.
    """
    name = "select_blocks"
    _check_block_size(name, block_size)
    _check_heads(name, q, "q")
    _check_heads(name, means, "means", torch.float32)
    B, N, Hq, d = q.shape
    nblk, Hkv = means.shape[1:3]
    if means.shape[0] != B or means.shape[3] != d or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{name}: q {tuple(q.shape)} and means {tuple(means.shape)} do not belong together")
    for what, x in (("count", count), ("first", first), ("last", last)):
        if isinstance(x, bool) or not isinstance(x, int) or x < 0:
            raise ValueError(f"{name}: {what} must be a non-negative integer, got {x!r}")
    if not 0 < count <= MAX_COUNT or first + last > count:
        raise ValueError(f"{name}: count must be 1 to {MAX_COUNT} and at least first + last, got {count}, {first}, {last}")
    _check_sequences(name, B, starts=starts, lengths=lengths)
    on_gpu(name, q, means, starts, lengths)
    out = torch.empty((B, N, Hkv, count), dtype=torch.int32, device=q.device)
    if out.numel() == 0 or nblk == 0:
        return out.fill_(-1)
    q, means, starts, lengths = _operand(q.detach()), _operand(means.detach()), _dense(starts), _dense(lengths)
    p = _lib.MattnSelect(B=B, L=N, nblk=nblk, Hq=Hq, Hkv=Hkv, D=q.shape[3], dtype=DTYPES[q.dtype], block_size=block_size,
                         count=count, first=first, last=last, causal=bool(is_causal), q=q.data_ptr(),
                         means=means.data_ptr(), starts=_ptr(starts), lengths=_ptr(lengths), blocks=out.data_ptr())
    p.q_stride[:] = q.stride()[:3]
    p.m_stride[:] = means.stride()[:3]
    lib = _lib.load()
    ws, wptr, nws = _scratch(lib.mattn_select_workspace_bytes(ctypes.byref(p)), q.device)
    with launch_on(q.device):
        _lib.check(lib.mattn_select_blocks(ctypes.byref(p), wptr, nws, stream(q.device)), "mattn_select_blocks")
    return out


def _scratch(nbytes, device):
    """(tensor, 256-byte aligned pointer, bytes); at least 256 bytes, so that a call the
    library refuses gets as far as its own error."""
    nbytes = max(nbytes, 256)
    ws, ptr = _workspace(nbytes, device)
    return ws, ptr, nbytes


# mattn_selected as one record: sizes and types, scale, 8 x 3 strides, pointers
_RECORD = struct.Struct("=10if4x24q3Q")
assert _RECORD.size == ctypes.sizeof(_lib.MattnSelected)


class _Call:
    """What a call of the attention is besides its tensors of values."""

    def __init__(self, blocks, starts, lengths, block_size, causal, scale):
        self.blocks, self.starts, self.lengths = blocks, starts, lengths
        self.block_size, self.causal, self.scale = block_size, causal, scale

    def record(self, q, k, v, o, do=None, dq=None, dk=None, dv=None):
        B, N, Hq, d = q.shape
        strides = [(0, 0, 0) if t is None else t.stride()[:3] for t in (q, k, v, o, do, dq, dk, dv)]
        return _lib.MattnSelected.from_buffer_copy(_RECORD.pack(
            B, N, k.shape[1], Hq, k.shape[2], d, DTYPES[q.dtype], self.block_size, self.blocks.shape[3], self.causal,
            self.scale, *itertools.chain(*strides), self.blocks.data_ptr(), _ptr(self.starts) or 0, _ptr(self.lengths) or 0))

    def forward(self, q, k, v, grads):
        """(O, what the backward keeps: float32 O, lse and the blocks' lists)."""
        lib = _lib.load()
        B, N, Hq, d = q.shape
        Hkv = k.shape[2]
        o = torch.empty((B, N, Hq, d), dtype=q.dtype, device=q.device)
        p = self.record(q, k, v, o)
        pr = ctypes.byref(p)
        _lib.check(lib.mattn_selected_validate(pr), "mattn_selected_fwd")
        o32 = lse = lists = None
        if grads:
            o32 = torch.empty((B, Hkv, N, Hq // Hkv, d), dtype=torch.float32, device=q.device)
            lse = torch.empty((B, Hkv, N, Hq // Hkv), dtype=torch.float32, device=q.device)
            lists, _, _ = _scratch(lib.mattn_selected_lists_bytes(pr), q.device)
        ws, wptr, nws = _scratch(lib.mattn_selected_fwd_workspace_bytes(pr), q.device)
        with launch_on(q.device):
            _lib.check(lib.mattn_selected_fwd(pr, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), _ptr(o32),
                                              _ptr(lse), _aligned(lists), wptr, nws, stream(q.device)),
                       "mattn_selected_fwd")
        return o, o32, lse, lists

    def backward(self, q, k, v, o32, lse, lists, do):
        lib = _lib.load()
        dq, dk, dv = (torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k, v))
        p = self.record(q, k, v, dq, do, dq, dk, dv)
        pr = ctypes.byref(p)
        ws, wptr, nws = _scratch(lib.mattn_selected_bwd_workspace_bytes(pr), q.device)
        with launch_on(q.device):
            _lib.check(lib.mattn_selected_bwd(pr, q.data_ptr(), k.data_ptr(), v.data_ptr(), o32.data_ptr(), do.data_ptr(),
                                              lse.data_ptr(), _aligned(lists), wptr, nws, dq.data_ptr(), dk.data_ptr(),
                                              dv.data_ptr(), stream(q.device)), "mattn_selected_bwd")
        return dq, dk, dv


class _Selected(torch.autograd.Function):
    """Residuals: q, k, v, O in float32 (delta = dO . O is a small difference where one
    key dominates), the rows' log-sum-exp and the queries of each block, listed."""

    @staticmethod
    def forward(ctx, q, k, v, call):
        ctx.d, ctx.call = q.shape[3], call
        q, k, v = (_operand(x) for x in (q, k, v))
        o, o32, lse, lists = call.forward(q, k, v, True)
        ctx.save_for_backward(q, k, v, o32, lse, lists, call.blocks, call.starts, call.lengths)
        return o if ctx.d == q.shape[3] else o[..., : ctx.d].contiguous()

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        q, k, v, o32, lse, lists, *_ = ctx.saved_tensors
        grads = ctx.call.backward(q, k, v, o32, lse, lists, _operand(do))
        if ctx.d != q.shape[3]:
            grads = tuple(g[..., : ctx.d].contiguous() for g in grads)
        return (*grads, None)


def selected_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, blocks: torch.Tensor, block_size: int, *,
                       is_causal: bool = True, starts: Optional[torch.Tensor] = None,
                       lengths: Optional[torch.Tensor] = None, scale: Optional[float] = None) -> torch.Tensor:
    """Softmax attention of each query over the keys of its blocks.

    q: [B, N, Hq, d]; k, v: [B, L, Hkv, d], one dtype (bfloat16, float16, float32),
        d <= 128 (a multiple of 8 runs without a copy), any strides.
    blocks: int32 [B, N, Hkv, count], count <= 1024: block indices of each query and key
        head, in any order; -1, indices past the blocks a query sees, and repeated ones
        are skipped.
    starts, lengths: int32 [B]: query i of sequence b is at position starts[b] + i
        (None: i) and sees keys below lengths[b] (None: L; clamped to [0, L]) and, with
        is_causal, up to its own position.  Keys it does not see are not read into its
        result, whatever they hold.
    scale: of the scores (default 1 / sqrt(d)); finite, below 2e38.

    Returns [B, N, Hq, d] in q's dtype; differentiable once w.r.t. q, k and v (blocks,
    starts and lengths must not change before the backward).  A query without a key gives
    zeros and zero gradients.  Products are of the inputs' type (weights and dS rounded
    to it), sums float32; repeated calls give the same bits.
    """
    name = "selected_attention"
    _check_block_size(name, block_size)
    _check_heads(name, q, "q")
    _check_heads(name, k, "k", q.dtype)
    _check_heads(name, v, "v", q.dtype)
    B, N, Hq, d = q.shape
    L, Hkv = k.shape[1:3]
    if k.shape != v.shape or k.shape[0] != B or k.shape[3] != d or Hkv == 0 or Hq % Hkv:
        raise ValueError(f"{name}: q {tuple(q.shape)}, k {tuple(k.shape)} and v {tuple(v.shape)} do not belong together")
    if blocks.dtype != torch.int32 or blocks.dim() != 4 or tuple(blocks.shape[:3]) != (B, N, Hkv):
        raise TypeError(f"{name}: blocks must be int32 [{B}, {N}, {Hkv}, count], got {blocks.dtype} {tuple(blocks.shape)}")
    if blocks.shape[3] > MAX_COUNT:
        raise NotImplementedError(f"{name}: {blocks.shape[3]} blocks of a query are more than {MAX_COUNT}")
    _check_sequences(name, B, starts=starts, lengths=lengths)
    s = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not abs(s) < 2e38:  # (times log2 e it has to be a float32)
        raise ValueError(f"{name}: scale must be finite and below 2e38, got {scale}")
    on_gpu(name, q, k, v, blocks, starts, lengths)
    grads = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad)
    if q.numel() == 0 or k.numel() == 0 or blocks.numel() == 0:  # no query, or none with a key
        zero = torch.zeros(q.shape, dtype=q.dtype, device=q.device)
        return _Nothing.apply(q, k, v, zero) if grads else zero
    call = _Call(blocks.contiguous(), _dense(starts), _dense(lengths), block_size, bool(is_causal), s)
    if grads:
        return _Selected.apply(q, k, v, call)
    o = call.forward(*(_operand(x) for x in (q, k, v)), False)[0]
    return o if o.shape[3] == d else o[..., :d].contiguous()


class _Nothing(torch.autograd.Function):
    """Zeros that depend on q, k and v in name only."""

    @staticmethod
    def forward(ctx, q, k, v, zero):
        ctx.like = [(x.shape, x.dtype, x.device) for x in (q, k, v)]
        return zero.clone()

    @staticmethod
    @once_differentiable
    def backward(ctx, do):
        return (*(torch.zeros(s, dtype=t, device=d) for s, t, d in ctx.like), None)
