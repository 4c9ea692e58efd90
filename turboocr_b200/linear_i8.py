"""INT8 linear layers with a scale per token and per output channel over the
C-ABI, for the recognizer's linear layers.

    wq, ws = linear_i8.quantize_rows(weight)          # [N, K], once
    y = linear_i8.linear(x, wq, ws, bias, act="hardswish", err=err)

Work is enqueued on the current stream of the tensors' device (or on
``stream=``) and returns immediately. ``err`` is a device int32 that the caller
zeroed once: it becomes non-zero if a bounded device-side wait gave up. The
scratch memory of a call comes from torch's allocator, on the call's stream.
"""
from __future__ import annotations

import torch

from ._launch import DTYPES, dense, on, shaped
from ._lib import call, lib

ACTS = {"none": 0, "relu": 1, "hardswish": 2}  # TOCR_ACT_*
_FLOATS = tuple(DTYPES)
_F32 = (torch.float32,)
_I32 = (torch.int32,)
_I8 = (torch.int8,)


def pitch(K: int) -> int:
    """Bytes from row to row of codes: K rounded up to a multiple of 16."""
    return (K + 15) // 16 * 16


def quantize_rows(x: torch.Tensor, *, stream=None) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes int8 [rows, pitch(K)], scales fp32 [rows]) of x [rows, K] (fp16,
    bf16 or fp32): scale = max(max|x| * (1 / 127), 2^-126) in fp32, code = x /
    scale to the nearest integer, ties to even; zeros behind K. A row with an infinity or a
    NaN gets the scale NaN and codes 0."""
    if x.dim() != 2:
        raise ValueError("x is [rows, K]")
    dev = x.get_device()
    px = dense(x, "x", dev, _FLOATS)
    rows, K = x.shape

    def launch(s):
        codes = torch.empty(rows, pitch(K), dtype=torch.int8, device=x.device)
        scales = torch.empty(rows, dtype=torch.float32, device=x.device)
        call("tocr_quant_rows_i8", px, DTYPES[x.dtype], rows, K, codes.data_ptr(),
             scales.data_ptr(), s)
        return codes, scales

    return on(dev, stream, launch)


def _weights(wq, ws, bias, K, dev, act, out_dtype, err):
    N = wq.shape[0]
    shaped(wq, "wq", (N, pitch(K)))
    shaped(ws, "ws", (N,))
    pb = None
    if bias is not None:
        shaped(bias, "bias", (N,))
        pb = dense(bias, "bias", dev, _F32)
    if act not in ACTS:
        raise ValueError(f"act must be one of {', '.join(ACTS)}, not {act!r}")
    if out_dtype not in DTYPES:
        raise ValueError(f"out_dtype must be one of {', '.join(map(str, DTYPES))}")
    pe = dense(err, "err", dev, _I32)
    if not err.numel():
        raise ValueError("err must hold one int32")
    return N, pe, (dense(wq, "wq", dev, _I8), dense(ws, "ws", dev, _F32), pb, N, ACTS[act],
                   DTYPES[out_dtype])


def linear(x: torch.Tensor, wq: torch.Tensor, ws: torch.Tensor, bias: torch.Tensor | None = None,
           *, err: torch.Tensor, act: str = "none", out_dtype: torch.dtype | None = None,
           stream=None) -> torch.Tensor:
    """act(x W^T + bias) [rows, N] for x [rows, K] (fp16, bf16 or fp32),
    quantised per row in the call, and weights as quantize_rows gives them.
    out_dtype: x's by default. The sum is exact, the rest fp32, rounded once."""
    if x.dim() != 2 or wq.dim() != 2:
        raise ValueError("x is [rows, K], wq is [N, pitch(K)]")
    dev = x.get_device()
    rows, K = x.shape
    px = dense(x, "x", dev, _FLOATS)
    out_dtype = x.dtype if out_dtype is None else out_dtype
    N, pe, w = _weights(wq, ws, bias, K, dev, act, out_dtype, err)

    def launch(s):
        y = torch.empty(rows, N, dtype=out_dtype, device=x.device)
        n = lib().tocr_linear_i8_workspace_bytes(rows, K)
        buf = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        call("tocr_linear_i8", px, DTYPES[x.dtype], rows, K, *w, y.data_ptr(),
             buf.data_ptr() if n else None, n, pe, s)
        return y

    return on(dev, stream, launch)


def linear_codes(xq: torch.Tensor, sx: torch.Tensor, K: int, wq: torch.Tensor, ws: torch.Tensor,
                 bias: torch.Tensor | None = None, *, err: torch.Tensor, act: str = "none",
                 out_dtype: torch.dtype = torch.float16, stream=None) -> torch.Tensor:
    """linear() on rows that quantize_rows has quantised already (several layers
    on the same activations quantise them once), or on any int8 codes. K below
    2^17 (products of -128 fill the 32 bits of the sum there)."""
    if xq.dim() != 2 or wq.dim() != 2:
        raise ValueError("xq is [rows, pitch(K)], wq is [N, pitch(K)]")
    dev = xq.get_device()
    rows = xq.shape[0]
    shaped(xq, "xq", (rows, pitch(K)))
    shaped(sx, "sx", (rows,))
    px, psx = dense(xq, "xq", dev, _I8), dense(sx, "sx", dev, _F32)
    N, pe, w = _weights(wq, ws, bias, K, dev, act, out_dtype, err)

    def launch(s):
        y = torch.empty(rows, N, dtype=out_dtype, device=xq.device)
        call("tocr_linear_i8_codes", px, psx, rows, K, *w, y.data_ptr(), pe, s)
        return y

    return on(dev, stream, launch)
