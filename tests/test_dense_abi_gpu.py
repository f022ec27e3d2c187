"""The C entry points of the dense operators on a GPU, where they allow more than tensors of torch show: results that start anywhere."""
import ctypes as C

import pytest

from tile_fusion_b200 import _lib
from tests.test_linear_ce import TYPES, make

pytestmark = pytest.mark.gpu

CODE = {"float32": _lib.F32, "bfloat16": _lib.BF16, "float16": _lib.F16}


def stream():
    import torch
    return torch.cuda.current_stream().cuda_stream


def space(n, d, v, dtype, backward):
    import torch
    return torch.empty(_lib.lib().tf_linear_ce_work_bytes(n, d, v, CODE[dtype], backward), device="cuda", dtype=torch.uint8)


def forward(x, w, t, reduction, work=None):
    """loss and lse2 of tf_linear_ce_fwd, which were NaN-free garbage before."""
    import torch
    n, d, v, dtype = x.shape[0], x.shape[1], w.shape[0], str(x.dtype)[6:]
    loss, lse = torch.full((n if reduction == 0 else 1,), 7.0, device="cuda"), torch.full((n,), 7.0, device="cuda")
    work = space(n, d, v, dtype, 0) if work is None else work
    _lib.check(_lib.lib().tf_linear_ce_fwd(x.data_ptr(), d, w.data_ptr(), d, CODE[dtype], t.data_ptr(), n, d, v, -100, reduction, loss.data_ptr(),
                                           lse.data_ptr(), work.data_ptr(), work.numel(), stream()))
    return loss, lse


def backward(x, w, t, reduction, lse, grad, dx, dw, work=None):
    n, d, v, dtype = x.shape[0], x.shape[1], w.shape[0], str(x.dtype)[6:]
    work = space(n, d, v, dtype, 1) if work is None else work
    _lib.check(_lib.lib().tf_linear_ce_bwd(x.data_ptr(), d, w.data_ptr(), d, CODE[dtype], t.data_ptr(), n, d, v, -100, reduction, lse.data_ptr(),
                                           grad.data_ptr(), dx.data_ptr(), dw.data_ptr(), work.data_ptr(), work.numel(), stream()))


# gradients in a flat buffer, some values behind its start: aligned to a value only, to 8 and to 16 bytes
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(300, 64, 40), (130, 256, 64), (65, 40, 10), (300, 64, 300), (20_000, 72, 300)])
@pytest.mark.parametrize("off", [1, 2, 4, 8])
def test_gradients_that_start_anywhere(built_lib, dtype, n, d, v, off):
    import torch
    x, w, t = make(n, d, v, dtype)
    grad = torch.ones(1, device="cuda")
    _, lse = forward(x, w, t, 2)
    results = []
    for o in (0, off):
        flat = torch.full((n * d + v * d + 64,), 5.0, device="cuda", dtype=x.dtype)
        dx, dw = flat[o:o + n * d], flat[o + n * d + o:o + n * d + o + v * d]
        backward(x, w, t, 2, lse, grad, dx, dw)
        assert (flat[:o] == 5).all() and (flat[o + n * d + o + v * d:] == 5).all() and (flat[o + n * d:o + n * d + o] == 5).all()
        results.append((dx.clone(), dw.clone()))
    assert all(torch.equal(a, b) for a, b in zip(*results))
