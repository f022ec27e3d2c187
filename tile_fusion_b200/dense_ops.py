"""Dense operators of a training step beside the fused layers, registered under ``torch.ops.sw_gcn`` (:mod:`.sw_gcn`)::

    torch.ops.sw_gcn.linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean")

``linear_cross_entropy`` is the softmax cross entropy of ``x @ weight.T`` (weight stored ``[out, in]``, as in the layers)
against class indices, without the logits in memory, with the gradients of both operands.  Rows whose target is
``ignore_index`` do not count: they add nothing to the loss or to the weight's gradient and receive a gradient of zero,
whatever they hold.  ``reduction``: "mean" over the rows that count (zero if none does), "sum", or "none" (a loss to each
row).  The loss is fp32.

The operators take fp32, bf16 and fp16 CUDA tensors whose last dimension is contiguous or is made so, run on the current
stream of the tensors' device, take their workspaces from torch's allocator, and can be captured into CUDA graphs.  They
are differentiable once.
"""
from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


def _on(t):
    return torch.cuda.device(t.device), lambda: torch.cuda.current_stream(t.device).cuda_stream


def _check_values(name, what, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"sw_gcn.{name}: {what} must be a CUDA tensor")
    if t.dtype not in _DTYPES:
        raise ValueError(f"sw_gcn.{name}: {what} must be float32, bfloat16 or float16, not {t.dtype}")


def _rows(t):
    """t as [rows, columns] whose rows do not overlap and have their values side by side."""
    t = t.reshape(-1, t.shape[-1])
    return t if (t.shape[1] == 1 or t.stride(1) == 1) and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _ld(t):
    """Values from one row to the next (of a single row any number: its own length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        L = _lib.lib()
        xr, w, t = _rows(x), _rows(weight), target.reshape(-1).to(torch.int64).contiguous()
        n, d, v = xr.shape[0], xr.shape[1], w.shape[0]
        code = _DTYPES[x.dtype]
        guard, stream = _on(x)
        with guard:
            loss = torch.empty(n if reduction == 0 else (), device=x.device, dtype=torch.float32)
            lse = torch.empty(n, device=x.device, dtype=torch.float32)
            work = torch.empty(L.tf_linear_ce_work_bytes(n, d, v, code, 0), device=x.device, dtype=torch.uint8)
            _lib.check(L.tf_linear_ce_fwd(xr.data_ptr(), _ld(xr), w.data_ptr(), _ld(w), code, t.data_ptr(), n, d, v, ignore_index,
                                          reduction, loss.data_ptr(), lse.data_ptr(), work.data_ptr(), work.numel(), stream()))
        ctx.save_for_backward(xr, w, t, lse)
        ctx.args = (ignore_index, reduction, x.shape, weight.shape)
        return loss.reshape(target.shape) if reduction == 0 else loss

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        L = _lib.lib()
        xr, w, t, lse = ctx.saved_tensors
        ignore_index, reduction, x_shape, w_shape = ctx.args
        n, d, v = xr.shape[0], xr.shape[1], w.shape[0]
        code = _DTYPES[xr.dtype]
        guard, stream = _on(xr)
        with guard:
            g = grad.reshape(-1).to(torch.float32).contiguous()
            dx = torch.empty((n, d), device=xr.device, dtype=xr.dtype) if ctx.needs_input_grad[0] else None
            dw = torch.empty((v, d), device=xr.device, dtype=xr.dtype) if ctx.needs_input_grad[1] else None
            work = torch.empty(L.tf_linear_ce_work_bytes(n, d, v, code, 1), device=xr.device, dtype=torch.uint8)
            _lib.check(L.tf_linear_ce_bwd(xr.data_ptr(), _ld(xr), w.data_ptr(), _ld(w), code, t.data_ptr(), n, d, v, ignore_index,
                                          reduction, lse.data_ptr(), g.data_ptr(), dx.data_ptr() if dx is not None else None,
                                          dw.data_ptr() if dw is not None else None, work.data_ptr(), work.numel(), stream()))
        return (dx.reshape(x_shape) if dx is not None else None, dw.reshape(w_shape) if dw is not None else None, None, None, None)


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    name = "linear_cross_entropy"
    _check_values(name, "x", x)
    _check_values(name, "weight", weight)
    if reduction not in _REDUCTIONS:
        raise ValueError(f"sw_gcn.{name}: reduction must be none, mean or sum, not {reduction!r}")
    if weight.dim() != 2 or x.dim() < 1 or x.shape[-1] != weight.shape[1]:
        raise ValueError(f"sw_gcn.{name}: x {tuple(x.shape)} and weight {tuple(weight.shape)} do not chain")
    if weight.shape[0] == 0 or weight.shape[1] == 0:
        raise ValueError(f"sw_gcn.{name}: the weight is empty")
    if x.dtype != weight.dtype:
        raise ValueError(f"sw_gcn.{name}: x is {x.dtype}, weight {weight.dtype}")
    if target.dtype not in (torch.int64, torch.int32) or target.shape != x.shape[:-1]:
        raise ValueError(f"sw_gcn.{name}: target must hold one int64 or int32 class for each row of x")
    if x.device != weight.device or x.device != target.device:
        raise ValueError(f"sw_gcn.{name}: x, weight and target must be on one device")
    return _LinearCrossEntropy.apply(x, weight, target, int(ignore_index), _REDUCTIONS[reduction])
