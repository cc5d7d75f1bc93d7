"""Checks of arguments and launches that the operators around the attention share."""
from __future__ import annotations

import contextlib

import torch

from . import _lib

DTYPES = {torch.bfloat16: _lib.MATTN_BF16, torch.float16: _lib.MATTN_F16, torch.float32: _lib.MATTN_F32}
_NO_GUARD = contextlib.nullcontext()


def on_gpu(name, *tensors):
    """All tensors (None: left out) are on one GPU (RuntimeError, ValueError otherwise)."""
    dev = tensors[0].device
    for t in tensors:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} runs on the GPU only (no CPU code path)")
        if t.device != dev:
            raise ValueError(f"{name}: tensors on {dev} and {t.device}")


def launch_on(device):
    """Context in which kernels are launched on ``device`` (whatever the current one)."""
    return _NO_GUARD if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream(device) -> int:
    return torch._C._cuda_getCurrentRawStream(device.index)


def rows(t):
    """t with contiguous columns and without negative strides (torch has none)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()
