"""Checks and launch helpers that the decoding operators share.

Everything here runs on the host before any device work.  These operators are
called once per layer and token, often with a few microseconds of GPU work, so
an eager call goes to the native binding first (:func:`direct`), which checks
its arguments without messages; only what it does not take comes to the checks
here, which say what is wrong.
"""

from __future__ import annotations

import torch

from .. import _native
from .._targets import AcceleratorTarget

DTYPE_CODES = {torch.float16: _native.FLOAT16, torch.bfloat16: _native.BFLOAT16}
SUPPORTED_HEAD_DIMS = (64, 128)
MAX_NODES = 64

_binding = None


def direct(name: str, what: str, *args):
    """Outputs of the native binding's function, or None: the call goes on through the checks.

    That is so under ``torch.compile`` and other modes that trace or transform
    operators, for tensor subclasses (both then reach the registered operator),
    and for arguments that the operator does not take.
    """
    global _binding
    if torch.compiler.is_compiling():
        return None
    if _binding is None:
        _binding = _native.binding()
    out = getattr(_binding, name)(*args)
    if type(out) is int:
        _native.check(out, what)
    return out


_sm100_devices: dict[int, bool] = {}


def require_device(operator: str, device: torch.device) -> None:
    """Raise unless ``device`` is an sm_100 GPU."""
    if device.type == "cuda":
        if device.index in _sm100_devices:
            return
        if AcceleratorTarget.from_device(device).supports_tcgen05_int8:
            _sm100_devices[device.index] = True
            return
    target = AcceleratorTarget.from_device(device)
    raise RuntimeError(
        f"{operator}'s B200 backend requires CUDA tensors on an sm_100 GPU, "
        f"got device {device} ({target.architecture or target.backend}); "
        "this package has no CPU or generic-GPU fallback"
    )


def fits(tensor: torch.Tensor, shape: tuple[int, ...], dtype: torch.dtype, device: torch.device) -> bool:
    """Whether :func:`check_tensor` would accept the argument (``shape`` in whole numbers, not empty)."""
    return (
        tensor.shape == shape
        and tensor.dtype is dtype
        and tensor.device == device
        and tensor.layout is torch.strided
        and (tensor.stride(-1) == 1 or shape[-1] <= 1)
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


def refuse_grad(operator: str) -> None:
    raise RuntimeError(f"{operator} is an inference-only operator and does not support autograd")


def _stream(index: int) -> int:
    return torch.cuda.current_stream(index).cuda_stream


# The same handle without a Stream object around it (0.1 against 2.2 us), where torch has it.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", _stream)


def launch(what: str, device: torch.device, call, *args) -> None:
    """Call a C entry point on ``device``'s current stream (its last argument)."""
    index = device.index
    if index == torch.cuda.current_device():
        status = call(*args, _raw_stream(index))
    else:
        with torch.cuda.device(device):
            status = call(*args, _raw_stream(index))
    if status:
        _native.check(status, what)
