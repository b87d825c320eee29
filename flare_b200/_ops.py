"""What the operators outside the render path (embedding, recurrence, microscale) share on the host: the type
codes of the C ABI, argument checks in the renderer's manner (ValueError), the stream and device of a call."""
from __future__ import annotations

from contextlib import nullcontext

import torch

TYPE_CODE = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # FLARE_F32, FLARE_F16, FLARE_BF16
MICRO = 3                                                            # FLARE_MICRO
INDEX_CODE = {torch.int32: 0, torch.int64: 1}                        # FLARE_I32, FLARE_I64


_raw_stream = torch._C._cuda_getCurrentRawStream
_same_device = nullcontext()


def ptr(t):
    return 0 if t is None else t.data_ptr()


def need(t, name, dtypes, device=None):
    """A CUDA tensor of one of `dtypes`, on `device` if given."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: expected a torch.Tensor, got {type(t).__name__}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name}: dtype {t.dtype}, expected {' or '.join(str(d) for d in dtypes)}")
    if not t.is_cuda:
        raise ValueError(f"{name}: tensor must be on a CUDA device")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: tensor on {t.device}, expected {device}")
    return t


def need_shape(t, name, shape):
    if t.shape != shape:
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple(shape)}")
    return t


def on(device):
    """Makes `device` current for the launches inside."""
    return _same_device if torch.cuda.current_device() == device.index else torch.cuda.device(device)


def stream(device):
    """The handle of the device's current stream."""
    return _raw_stream(device.index)


def workspace(nbytes, device):
    """Scratch of one call, from the caching allocator, so that it belongs to the call's stream or graph."""
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def rows(t):
    """(rows, width) view of a tensor whose leading dimensions step evenly and whose last one is dense, or a copy
    that is one."""
    width = t.shape[-1]
    if t.dim() == 2 and (t.stride(1) == 1 or width <= 1) and t.stride(0) >= width:
        return t
    return t.reshape(-1, width).contiguous() if width else t.reshape(t.numel() // max(width, 1), width)
