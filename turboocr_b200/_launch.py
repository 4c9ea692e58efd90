"""What the linear-layer wrappers share: argument checks, and running a call on
its tensors' device and stream."""
from __future__ import annotations

import torch

DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}  # TOCR_DTYPE_*


def dense(t: torch.Tensor, name: str, device: torch.device, *dtypes: torch.dtype) -> int:
    """The address of a contiguous CUDA tensor of one of `dtypes` on `device`."""
    if t.device != device or not t.is_cuda:
        raise ValueError(f"{name} must live on {device} (a CUDA device), not on {t.device}")
    if t.dtype not in dtypes:
        raise ValueError(f"{name} must be {' or '.join(map(str, dtypes))}, not {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")
    return t.data_ptr()


def shaped(t: torch.Tensor, name: str, *shape: int) -> None:
    if tuple(t.shape) != shape:
        raise ValueError(f"{name} must have shape {shape}, not {tuple(t.shape)}")


def on(device: torch.device, stream, launch):
    """launch(raw stream) with `device` current: on `stream`, or on the
    device's current stream. What launch() allocates belongs to that stream."""
    if stream is None and torch.cuda.current_device() == device.index:
        return launch(torch.cuda.current_stream().cuda_stream)
    with torch.cuda.device(device):
        if stream is None:
            return launch(torch.cuda.current_stream().cuda_stream)
        if not hasattr(stream, "cuda_stream"):
            stream = torch.cuda.ExternalStream(int(stream), device=device)
        if stream.device != device:
            raise ValueError(f"the stream belongs to {stream.device}, the tensors to {device}")
        with torch.cuda.stream(stream):
            return launch(stream.cuda_stream)
