"""Training and scoring of the recognizer's linear head over the C-ABI:
cross entropy of the head's logits (features [rows, K] times weights
[classes, K] plus bias) for a target class per time step, and its gradient,
without storing the logits. tocr_rec_head_ctc_f16 serves the same layer; the
step indices that it writes are targets as they are.

Work is enqueued on the current stream of the tensors' device (or on
``stream=``) and returns immediately. ``err`` is a device int32 that the caller
zeroed once: it becomes non-zero if a bounded device-side wait gave up. The
scratch memory of a call comes from torch's allocator, on the call's stream.
"""
from __future__ import annotations

import torch

from ._launch import DTYPES, dense, on, shaped
from ._lib import call, lib

_F32 = (torch.float32,)
_I32 = (torch.int32,)
_INTS = (torch.int32, torch.int64)
_HALVES = (torch.float16, torch.bfloat16)


def _common(feat, weight, bias, targets, err):
    if feat.dim() != 2 or weight.dim() != 2:
        raise ValueError("features are [rows, K], weights [classes, K]")
    dev = feat.get_device()
    rows, K = feat.shape
    V = weight.shape[0]
    shaped(weight, "weight", (V, K))
    shaped(targets, "targets", (rows,))
    dt = feat.dtype
    pf = dense(feat, "feat", dev, _HALVES)
    pw = dense(weight, "weight", dev, (dt,))
    pb = None
    if bias is not None:
        shaped(bias, "bias", (V,))
        pb = dense(bias, "bias", dev, _F32)
    pt = dense(targets, "targets", dev, _INTS)
    pe = dense(err, "err", dev, _I32)
    if not err.numel():
        raise ValueError("err must hold one int32")
    return (dev, rows, K, V, pe,
            (pf, pw, pb, pt, targets.dtype is torch.int64, rows, K, V, DTYPES[dt]))


def cross_entropy(feat: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
                  targets: torch.Tensor, *, err: torch.Tensor, stream=None):
    """(loss, lse), both fp32 [rows]: loss = lse - logit[target]. feat [rows, K]
    and weight [classes, K] fp16 or bf16, K a multiple of 8 up to 256, bias
    fp32 [classes] or None, targets int32 or int64 [rows]. A target outside
    [0, classes) marks padding: loss and lse 0, and the row's features are not
    looked at. Not an autograd function: the gradient is cross_entropy_backward's,
    and tensors that require grad are refused where grad mode is on."""
    if torch.is_grad_enabled() and (feat.requires_grad or weight.requires_grad
                                    or (bias is not None and bias.requires_grad)):
        raise ValueError("the loss would carry no graph: call cross_entropy under torch.no_grad() "
                         "or on detached tensors, and cross_entropy_backward for the gradient")
    dev, rows, K, V, pe, args = _common(feat, weight, bias, targets, err)

    def launch(s):
        loss = torch.empty(rows, dtype=torch.float32, device=feat.device)
        lse = torch.empty_like(loss)
        n = lib().tocr_rec_head_ce_workspace_bytes(rows, K, V, 0)
        ws = torch.empty(n, dtype=torch.uint8, device=feat.device)
        call("tocr_rec_head_ce", *args, loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), n, pe, s)
        return loss, lse

    return on(dev, stream, launch)


def cross_entropy_backward(feat: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None,
                           targets: torch.Tensor, lse: torch.Tensor, grad_loss: torch.Tensor, *,
                           err: torch.Tensor, need_feat: bool = True, need_weight: bool = True,
                           need_bias: bool = True, stream=None):
    """(dfeat, dweight, dbias) for the weight grad_loss[i] (fp32 [rows]) of every
    row's loss, with lse as cross_entropy returned it for the same inputs.
    dfeat and dweight have the inputs' type, dbias is fp32 (None without a
    bias); a gradient that is not needed is None. Padding rows get zeros."""
    dev, rows, K, V, pe, args = _common(feat, weight, bias, targets, err)
    shaped(lse, "lse", (rows,))
    shaped(grad_loss, "grad_loss", (rows,))
    pl, pg = dense(lse, "lse", dev, _F32), dense(grad_loss, "grad_loss", dev, _F32)

    def launch(s):
        dfeat = torch.empty_like(feat) if need_feat else None
        dweight = torch.empty_like(weight) if need_weight else None
        dbias = torch.empty_like(bias) if need_bias and bias is not None else None
        n = lib().tocr_rec_head_ce_workspace_bytes(rows, K, V, 1)
        ws = torch.empty(n, dtype=torch.uint8, device=feat.device)
        call("tocr_rec_head_ce_backward", *args, pl, pg,
             dfeat.data_ptr() if need_feat else None,
             dweight.data_ptr() if need_weight else None,
             dbias.data_ptr() if dbias is not None else None, ws.data_ptr(), n, pe, s)
        return dfeat, dweight, dbias

    return on(dev, stream, launch)
