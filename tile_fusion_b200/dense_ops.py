"""Dense operators of a training step beside the fused layers, registered under ``torch.ops.sw_gcn`` (:mod:`.sw_gcn`)::

    torch.ops.sw_gcn.layer_norm(x, weight=None, bias=None, eps=1e-5, checkpoint=False)
    torch.ops.sw_gcn.pack8(x, relu=False)                      -> codes, exponents
    torch.ops.sw_gcn.unpack8(codes, exponents, dtype=None)     -> the values they stand for
    torch.ops.sw_gcn.weight_grad8(grad, codes, exponents)      -> grad.T @ values
    torch.ops.sw_gcn.fusedGeMMSpMM_ck8(adj, feature, weight, schedule, num_threads, relu=False)
    torch.ops.sw_gcn.linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean")

``layer_norm`` is over the last dimension, with the gradients of x, weight and bias; weight and bias have x's type or
another of the three.  With ``checkpoint`` it keeps x in 8 bits for the backward pass (x itself can be freed): y is still
that of x, the gradients are those of the formula at the kept values.

``pack8`` puts activations [rows, columns] into 8 bits: 32 neighbouring columns share a power of two, a value is a whole
number of steps of its 64th part, the nearest one, at most 127 of them.  ``codes`` is int8 [rows, columns] with rows that
start on multiples of 32, ``exponents`` uint8 [rows, columns / 32 rounded up]; a group that holds an infinity or a NaN reads
back as NaN.  With ``relu`` negative values become zero first, and a code of -128 is a positive value that rounds to zero, so
that ``codes != 0`` says where the value was positive.  ``weight_grad8`` is the weight gradient of a layer whose input was
packed, in grad's type, of at most 2^26 entries.  These three carry no graph; ``fusedGeMMSpMM_ck8`` is the layer that uses them:
``adj @ (h @ weight.T)`` with ``h = feature``, or with ``relu`` ``h = max(feature, 0)``, of which it keeps the 8 bits instead of
the 32; the forward result and the gradient of feature are those of ``fusedGeMMSpMM``, the weight's gradient is taken at the
kept values.

``linear_cross_entropy`` is the softmax cross entropy of ``x @ weight.T`` (weight stored ``[out, in]``, as in the layers)
against class indices, without the logits in memory, with the gradients of both operands, which have the same type.  Rows whose target is
``ignore_index`` do not count: they add nothing to the loss or to the weight's gradient and receive a gradient of zero,
whatever they hold.  ``reduction``: "mean" over the rows that count (zero if none does), "sum", or "none" (a loss to each
row).  The loss is fp32.  fp32 operands are multiplied as two fp16 planes: 22 bits of values down to 2^-17 of their tensor's largest.

The operators take fp32, bf16 and fp16 CUDA tensors whose last dimension is contiguous or is made so, run on the current
stream of the tensors' device, take their workspaces from torch's allocator, and can be captured into CUDA graphs.  They
are differentiable once, backwards; a forward-mode tangent is refused.  (A captured backward pass belongs in ``torch.autograd.grad``, or to leaves of which no eager graph is
alive: autograd accumulates into a leaf on the stream of the graph that made its accumulator, which a capture cannot wait for.)
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

_DTYPES = {torch.float32: _lib.F32, torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
_MOST = 0x7f000000
_REDUCTIONS = {"none": 0, "mean": 1, "sum": 2}


_current_device = getattr(torch._C, "_cuda_getDevice", None) or torch.cuda.current_device
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda d: torch.cuda.current_stream(d).cuda_stream)


def _tangents():
    """Whether forward-mode tangents may go with the tensors: autograd's functions refuse those, where plain calls would drop them."""
    return forward_ad._current_level >= 0


def _refuse_tangent(name, t):
    if forward_ad.unpack_dual(t).tangent is not None:
        raise RuntimeError(f"sw_gcn.{name} carries no graph: a forward-mode tangent would be lost")


def _on_device_of_first(f):
    """f with the device of its first tensor as the current one, on that device's current stream (given as the last argument)."""
    def run(t, *args):
        d = t.get_device()
        if d == _current_device():
            return f(t, *args, _raw_stream(d))
        with torch.cuda.device(d):
            return f(t, *args, _raw_stream(d))
    return run


def _check_values(name, what, t):
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"sw_gcn.{name}: {what} must be a CUDA tensor")
    if t.dtype not in _DTYPES:
        raise ValueError(f"sw_gcn.{name}: {what} must be float32, bfloat16 or float16, not {t.dtype}")


def _rows(t):
    """t as [rows, columns] whose rows do not overlap and have their values side by side."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    if t.shape[0] > _MOST or t.shape[1] > _MOST:
        raise ValueError(f"sw_gcn: matrices of at most {_MOST} rows and columns, not {tuple(t.shape)}")
    if t.is_contiguous():
        return t
    return t if t.stride(1) == 1 and t.stride(0) >= t.shape[1] else t.contiguous()


def _ld(t):
    """Values from one row to the next (of a single row any number: its own length)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _fine(t, d):
    """Whether t holds values that the library takes, on device d."""
    return t.is_cuda and t.dtype in _DTYPES and t.get_device() == d


def _same_device(name, *tensors):
    first = tensors[0].device
    if any(t is not None and t.device != first for t in tensors):
        raise ValueError(f"sw_gcn.{name}: the tensors must be on one device")


def _ptr(t):
    return t.data_ptr() if t is not None else None


@_on_device_of_first
def _pack(x, relu, stream):
    """Codes [rows, columns rounded up to 32] and exponents of a matrix."""
    n, d = x.shape
    ld = -(-d // 32) * 32
    codes = torch.empty((n, ld), device=x.device, dtype=torch.int8)
    exponents = torch.empty((n, ld // 32), device=x.device, dtype=torch.uint8)
    _lib.check(_lib.lib().tf_pack8(x.data_ptr(), _ld(x), _DTYPES[x.dtype], n, d, int(relu), codes.data_ptr(), ld, exponents.data_ptr(), stream))
    return codes, exponents


@_on_device_of_first
def _unpack(codes, ld, exponents, dtype, n, d, stream):
    out = torch.empty((n, d), device=codes.device, dtype=dtype)
    _lib.check(_lib.lib().tf_unpack8(codes.data_ptr(), ld, exponents.data_ptr(), _DTYPES[dtype], n, d, out.data_ptr(), d, stream))
    return out


@_on_device_of_first
def _weight_grad(g, codes, ld, exponents, nb, stream):
    L = _lib.lib()
    m, na, code = g.shape[0], g.shape[1], _DTYPES[g.dtype]
    out = torch.empty((na, nb), device=g.device, dtype=g.dtype)
    work = torch.empty(L.tf_weight_grad8_work_floats(m, na, nb, code), device=g.device, dtype=torch.float32)
    _lib.check(L.tf_weight_grad8(g.data_ptr(), _ld(g), code, na, codes.data_ptr(), ld, exponents.data_ptr(), nb, m, out.data_ptr(),
                                 work.data_ptr(), work.numel(), stream))
    return out


@_on_device_of_first
def _relu_grad(grad, codes, stream):
    n, d = grad.shape
    _lib.check(_lib.lib().tf_relu_grad8(codes.data_ptr(), codes.shape[1], _DTYPES[grad.dtype], n, d, grad.data_ptr(), d, stream))
    return grad


def relu_grad8_(grad, codes):
    """grad (a contiguous matrix, in place) where the packed value was positive, zero elsewhere; codes: whole groups of 32, as they are packed."""
    _check_values("relu_grad8_", "grad", grad)
    if grad.dim() != 2 or not grad.is_contiguous():
        raise ValueError(f"sw_gcn.relu_grad8_: grad must be a contiguous matrix, not {tuple(grad.shape)} with strides {grad.stride()}")
    if codes.dtype != torch.int8 or codes.device != grad.device or not codes.is_contiguous() or codes.shape != (grad.shape[0], -(-grad.shape[1] // 32) * 32):
        raise ValueError(f"sw_gcn.relu_grad8_: codes must be contiguous int8 on grad's device, [{grad.shape[0]}, {-(-grad.shape[1] // 32) * 32}], not {tuple(codes.shape)}")
    return _relu_grad(grad, codes)


def _packed(name, codes, exponents):
    """Codes as the library reads them: rows of whole groups of 32 that start on multiples of 32 bytes, and their length."""
    if not codes.is_cuda or codes.dtype != torch.int8 or codes.dim() != 2 or exponents.dtype != torch.uint8:
        raise ValueError(f"sw_gcn.{name}: codes must be a CUDA int8 matrix and exponents a uint8 one, as pack8 gives them")
    n, d = codes.shape
    ld = -(-d // 32) * 32
    if d == 0 or exponents.shape != (n, ld // 32):
        raise ValueError(f"sw_gcn.{name}: codes {tuple(codes.shape)} need exponents [{n}, {ld // 32}], not {list(exponents.shape)}")
    if exponents.get_device() != codes.get_device():
        _same_device(name, codes, exponents)
    at = codes.storage_offset()
    if codes.stride(1) != 1 or (n > 1 and codes.stride(0) != ld) or codes.data_ptr() % 32 or codes.untyped_storage().nbytes() - at < n * ld:
        codes = torch.nn.functional.pad(codes, (0, ld - d)).contiguous()
    return codes, exponents.contiguous(), ld


def pack8(x, relu=False):
    if not _fine(x, x.get_device()):
        _check_values("pack8", "x", x)
    if x.dim() != 2 or x.shape[1] == 0:
        raise ValueError(f"sw_gcn.pack8: x must be a matrix of at least one column, not {tuple(x.shape)}")
    if _tangents():
        _refuse_tangent("pack8", x)
    codes, exponents = _pack(_rows(x), relu)
    d = x.shape[1]
    return (codes if codes.shape[1] == d else codes[:, :d]), exponents


def unpack8(codes, exponents, dtype=None):
    dtype = torch.float32 if dtype is None else dtype
    if dtype not in _DTYPES:
        raise ValueError(f"sw_gcn.unpack8: dtype must be float32, bfloat16 or float16, not {dtype}")
    d = codes.shape[-1] if codes.dim() else 0
    codes, exponents, ld = _packed("unpack8", codes, exponents)
    return _unpack(codes, ld, exponents, dtype, codes.shape[0], d)


def refuse_weight_grad8(name, na, nb):
    """A weight gradient [na, nb] that the library does not take, before anything is allocated for it."""
    if na * nb > 1 << 26 or max(na, nb) > 1 << 20:
        raise ValueError(f"sw_gcn.{name}: a weight gradient from 8 bits has at most 2^26 entries, 2^20 to a side, not [{na}, {nb}]")


def weight_grad8(grad, codes, exponents):
    name = "weight_grad8"
    _check_values(name, "grad", grad)
    if grad.dim() != 2 or codes.dim() != 2 or grad.shape[0] != codes.shape[0] or grad.shape[1] == 0:
        raise ValueError(f"sw_gcn.{name}: grad {tuple(grad.shape)} and codes {tuple(codes.shape)} do not chain")
    if _tangents():
        _refuse_tangent(name, grad)
    nb = codes.shape[1]
    refuse_weight_grad8(name, grad.shape[1], nb)
    codes, exponents, ld = _packed(name, codes, exponents)
    _same_device(name, grad, codes)
    return _weight_grad(_rows(grad), codes, ld, exponents, nb)


@_on_device_of_first
def _layer_norm_forward(xr, w, b, eps, stats, keep, stream):
    """y, mean and rstd, codes and exponents (None where not asked for)."""
    n, d = xr.shape
    first = w if w is not None else b if b is not None else xr
    y = torch.empty((n, d), device=xr.device, dtype=xr.dtype)
    s = torch.empty((2, n), device=xr.device, dtype=torch.float32) if stats else None
    at = s.data_ptr() if stats else None
    ld = -(-d // 32) * 32
    codes = torch.empty((n, ld), device=xr.device, dtype=torch.int8) if keep else None
    exponents = torch.empty((n, ld // 32), device=xr.device, dtype=torch.uint8) if keep else None
    _lib.check(_lib.lib().tf_layer_norm_fwd(xr.data_ptr(), _ld(xr), _DTYPES[xr.dtype], _ptr(w), _ptr(b), _DTYPES[first.dtype], n, d, eps,
                                            y.data_ptr(), d, at, at + 4 * n if stats else None, _ptr(codes), ld, _ptr(exponents), stream))
    return y, s, codes, exponents


@_on_device_of_first
def _layer_norm_backward(g, x, codes, exponents, w, s, dtype, w_dtype, want, stream):
    L = _lib.lib()
    n, d = g.shape
    dx = torch.empty((n, d), device=g.device, dtype=dtype) if want[0] else None
    dw = torch.empty(d, device=g.device, dtype=w_dtype) if want[1] else None
    db = torch.empty(d, device=g.device, dtype=w_dtype) if want[2] else None
    sums = want[1] or want[2]
    work = torch.empty(L.tf_layer_norm_work_floats(n, d), device=g.device, dtype=torch.float32) if sums else None
    at = s.data_ptr()
    _lib.check(L.tf_layer_norm_bwd(_ptr(x), _ld(x) if x is not None else d, _ptr(codes), codes.shape[1] if codes is not None else 0,
                                   _ptr(exponents), _DTYPES[dtype], _ptr(w), _DTYPES[w_dtype], n, d, at, at + 4 * n, g.data_ptr(), _ld(g),
                                   _ptr(dx), d, _ptr(dw), _ptr(db), _ptr(work), work.numel() if sums else 0, stream))
    return dx, dw, db


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps, checkpoint):
        need, shape = ctx.needs_input_grad, x.shape
        xr = _rows(x)
        w = weight.contiguous() if weight is not None else None
        b = bias.contiguous() if bias is not None else None
        y, s, codes, exponents = _layer_norm_forward(xr, w, b, eps, True, checkpoint and (need[0] or need[1]))
        ctx.save_for_backward(xr if codes is None else None, codes, exponents, w, s)
        ctx.args = (shape, x.dtype, (w if w is not None else b if b is not None else x).dtype)
        return y if len(shape) == 2 else y.view(shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        x, codes, exponents, w, s = ctx.saved_tensors
        shape, dtype, w_dtype = ctx.args
        dx, dw, db = _layer_norm_backward(_rows(grad), x, codes, exponents, w, s, dtype, w_dtype, ctx.needs_input_grad)
        return dx if dx is None or len(shape) == 2 else dx.view(shape), dw, db, None, None


def _refuse_layer_norm(x, weight, bias):
    """Says what is wrong with the arguments of layer_norm, if anything is."""
    name = "layer_norm"
    _check_values(name, "x", x)
    if x.dim() < 1 or x.shape[-1] == 0:
        raise ValueError(f"sw_gcn.{name}: x must have a last dimension of at least one value, not {tuple(x.shape)}")
    for what, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_values(name, what, t)
            if t.shape != x.shape[-1:]:
                raise ValueError(f"sw_gcn.{name}: {what} must have {x.shape[-1]} values, not {tuple(t.shape)}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise ValueError(f"sw_gcn.{name}: weight is {weight.dtype}, bias {bias.dtype}")
    _same_device(name, x, weight, bias)


def layer_norm(x, weight=None, bias=None, eps=1e-5, checkpoint=False):
    shape = x.shape
    d, last = x.get_device(), shape[-1:]
    # (one expression where all is well: the checks one by one cost a small call a tenth of its time)
    if not (_fine(x, d) and last and last[0] > 0 and (weight is None or (_fine(weight, d) and weight.shape == last))
            and (bias is None or (_fine(bias, d) and bias.shape == last and (weight is None or weight.dtype == bias.dtype)))):
        _refuse_layer_norm(x, weight, bias)
    if _tangents() or torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps, checkpoint)
    w = weight.contiguous() if weight is not None else None
    b = bias.contiguous() if bias is not None else None
    y = _layer_norm_forward(_rows(x), w, b, eps, False, False)[0]
    return y if len(shape) == 2 else y.view(shape)


@_on_device_of_first
def _loss_forward(xr, w, t, ignore_index, reduction, stream):
    L = _lib.lib()
    n, d, v, code = xr.shape[0], xr.shape[1], w.shape[0], _DTYPES[xr.dtype]
    loss = torch.empty(n if reduction == 0 else (), device=xr.device, dtype=torch.float32)
    lse = torch.empty(n, device=xr.device, dtype=torch.float32)
    work = torch.empty(L.tf_linear_ce_work_bytes_for(xr.data_ptr(), _ld(xr), w.data_ptr(), _ld(w), n, d, v, code, 0), device=xr.device, dtype=torch.uint8)
    _lib.check(L.tf_linear_ce_fwd(xr.data_ptr(), _ld(xr), w.data_ptr(), _ld(w), code, t.data_ptr(), n, d, v, ignore_index, reduction,
                                  loss.data_ptr(), lse.data_ptr(), work.data_ptr(), work.numel(), stream))
    return loss, lse


@_on_device_of_first
def _loss_backward(xr, w, t, lse, grad, ignore_index, reduction, want, stream):
    L = _lib.lib()
    n, d, v, code = xr.shape[0], xr.shape[1], w.shape[0], _DTYPES[xr.dtype]
    dx = torch.empty((n, d), device=xr.device, dtype=xr.dtype) if want[0] else None
    dw = torch.empty((v, d), device=xr.device, dtype=xr.dtype) if want[1] else None
    work = torch.empty(L.tf_linear_ce_work_bytes_for(xr.data_ptr(), _ld(xr), w.data_ptr(), _ld(w), n, d, v, code, 1), device=xr.device, dtype=torch.uint8)
    _lib.check(L.tf_linear_ce_bwd(xr.data_ptr(), _ld(xr), w.data_ptr(), _ld(w), code, t.data_ptr(), n, d, v, ignore_index, reduction,
                                  lse.data_ptr(), grad.data_ptr(), _ptr(dx), _ptr(dw), work.data_ptr(), work.numel(), stream))
    return dx, dw


def _classes(target):
    return target if target.dim() == 1 and target.dtype == torch.int64 and target.is_contiguous() else target.reshape(-1).to(torch.int64).contiguous()


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, target, ignore_index, reduction):
        xr, w, t = _rows(x), _rows(weight), _classes(target)
        loss, lse = _loss_forward(xr, w, t, ignore_index, reduction)
        ctx.save_for_backward(xr, w, t, lse)
        ctx.args = (ignore_index, reduction, x.shape)
        return loss if reduction or target.dim() == 1 else loss.view(target.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        xr, w, t, lse = ctx.saved_tensors
        ignore_index, reduction, shape = ctx.args
        g = grad if grad.dtype == torch.float32 and grad.is_contiguous() else grad.to(torch.float32).contiguous()
        dx, dw = _loss_backward(xr, w, t, lse, g, ignore_index, reduction, ctx.needs_input_grad)
        return dx if dx is None or len(shape) == 2 else dx.view(shape), dw, None, None, None


def _refuse_linear_cross_entropy(x, weight, target, reduction):
    """Says what is wrong with the arguments of linear_cross_entropy, if anything is."""
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
    _same_device(name, x, weight, target)


def linear_cross_entropy(x, weight, target, ignore_index=-100, reduction="mean"):
    d, code = x.get_device(), _REDUCTIONS.get(reduction)
    if not (_fine(x, d) and _fine(weight, d) and target.is_cuda and target.get_device() == d and x.dtype == weight.dtype and code is not None
            and weight.dim() == 2 and x.dim() > 0 and x.shape[-1] == weight.shape[1] and weight.numel() > 0
            and target.dtype in (torch.int64, torch.int32) and target.shape == x.shape[:-1]):
        _refuse_linear_cross_entropy(x, weight, target, reduction)
    if _tangents() or torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        return _LinearCrossEntropy.apply(x, weight, target, ignore_index, code)
    loss, _ = _loss_forward(_rows(x), _rows(weight), _classes(target), ignore_index, code)
    return loss if code or target.dim() == 1 else loss.view(target.shape)
