"""What the linear-layer wrappers share: argument checks, and running a call on
its tensors' device and stream. The checks are written for speed: the smallest
calls take a few microseconds on the device."""
from __future__ import annotations

import torch

DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # TOCR_DTYPE_*

_raw_stream = torch._C._cuda_getCurrentRawStream  # without building a Stream object
_current_device = torch.cuda.current_device


def dense(t: torch.Tensor, name: str, device: int, dtypes: tuple) -> int:
    """The address of a contiguous tensor of one of `dtypes` on CUDA device
    number `device`."""
    if t.get_device() != device or device < 0:
        where = f"cuda:{device}" if device >= 0 else "a CUDA device"
        raise ValueError(f"{name} must live on {where}, not on {t.device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(map(str, dtypes))}, not {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def shaped(t: torch.Tensor, name: str, shape: tuple) -> None:
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")


def on(device: int, stream, launch):
    """launch(raw stream) with CUDA device `device` current: on `stream`, or on
    the device's current stream. What launch() allocates belongs to that stream."""
    if stream is None and _current_device() == device:
        return launch(_raw_stream(device))
    with torch.cuda.device(device):
        if stream is None:
            return launch(_raw_stream(device))
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(int(stream), device=device)
        if stream.device.index != device:
            raise ValueError(f"the stream belongs to {stream.device}, the tensors to cuda:{device}")
        with torch.cuda.stream(stream):
            return launch(stream.cuda_stream)
