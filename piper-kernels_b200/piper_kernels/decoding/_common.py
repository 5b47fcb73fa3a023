"""Checks and launch helpers that the decoding operators share.

Everything here runs on the host before any device work.  These operators are
called once per layer and token, so the checks read tensor attributes only.
"""

from __future__ import annotations

from functools import lru_cache

import torch

from .. import _native
from .._targets import AcceleratorTarget

DTYPE_CODES = {torch.float16: _native.FLOAT16, torch.bfloat16: _native.BFLOAT16}
SUPPORTED_HEAD_DIMS = (64, 128)
MAX_NODES = 64


@lru_cache(maxsize=None)
def _is_sm100(index: int) -> bool:
    return AcceleratorTarget.from_device(torch.device("cuda", index)).supports_tcgen05_int8


def require_device(operator: str, device: torch.device) -> None:
    """Raise unless ``device`` is an sm_100 GPU."""
    if device.type == "cuda" and _is_sm100(device.index if device.index is not None else torch.cuda.current_device()):
        return
    target = AcceleratorTarget.from_device(device)
    raise RuntimeError(
        f"{operator}'s B200 backend requires CUDA tensors on an sm_100 GPU, "
        f"got device {device} ({target.architecture or target.backend}); "
        "this package has no CPU or generic-GPU fallback"
    )


def check_tensor(
    operator: str,
    name: str,
    tensor: torch.Tensor,
    shape: tuple[int | None, ...],
    dtype: torch.dtype,
    device: torch.device,
) -> None:
    """Check one argument's shape (None: any size), type, device and contiguous last dimension."""
    if tensor.ndim != len(shape) or any(want is not None and got != want for got, want in zip(tensor.shape, shape)):
        wanted = ", ".join("any" if n is None else str(n) for n in shape)
        raise ValueError(f"{operator} {name} must have shape [{wanted}], got {tuple(tensor.shape)}")
    if tensor.dtype is not dtype:
        raise ValueError(f"{operator} {name} must use {str(dtype).removeprefix('torch.')}, got {tensor.dtype}")
    if tensor.device != device:
        raise ValueError(f"{operator} {name} must be on {device}, got {tensor.device}")
    if tensor.layout is not torch.strided:
        raise ValueError(f"{operator} {name} must use strided layout")
    if tensor.ndim and tensor.shape[-1] > 1 and tensor.stride(-1) != 1:
        raise ValueError(f"{operator} {name}'s last dimension must be contiguous")


def check_half(operator: str, name: str, dtype: torch.dtype) -> None:
    if dtype not in DTYPE_CODES:
        raise ValueError(f"{operator} {name} must use float16 or bfloat16, got {dtype}")


def check_no_grad(operator: str, *tensors: torch.Tensor) -> None:
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise RuntimeError(f"{operator} is an inference-only operator and does not support autograd")


def launch(what: str, device: torch.device, call, *args) -> None:
    """Call a C entry point on ``device``'s current stream (its last argument)."""
    if device.index == torch.cuda.current_device():
        status = call(*args, torch.cuda.current_stream(device).cuda_stream)
    else:
        with torch.cuda.device(device):
            status = call(*args, torch.cuda.current_stream(device).cuda_stream)
    if status:
        _native.check(status, what)
