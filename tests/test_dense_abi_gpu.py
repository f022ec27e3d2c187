"""The C entry points of the dense operators on a GPU, where they allow more than tensors of torch show: results that start anywhere; and what a
bounded wait that ran out leaves."""
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


@pytest.fixture
def no_waits(built_lib):
    """Inside, every bounded wait gives up at once: nothing is waited for that does not come, no product is issued, and a kernel leaves as soon
    as the copies that it has started have landed."""
    from contextlib import contextmanager

    @contextmanager
    def inside():
        L = _lib.lib()
        assert L.tf_dense_set_wait_limit(0) == _lib.TF_OK
        try:
            yield
        finally:
            assert L.tf_dense_set_wait_limit(1 << 22) == _lib.TF_OK
    return inside


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(300, 64, 40), (20_000, 256, 64), (300, 64, 300), (1000, 640, 3000)])
def test_losses_whose_waits_run_out(no_waits, dtype, n, d, v):
    """NaN in the losses, in what the backward pass takes from the forward one, and in the gradients; and a status."""
    import torch
    L = _lib.lib()
    x, w, t = make(n, d, v, dtype)
    grad = torch.ones(n, device="cuda")
    counts = t >= 0
    good, lse = forward(x, w, t, 0)
    dx, dw, lost_dx, lost_dw = (torch.zeros_like(a) for a in (x, w, x, w))
    backward(x, w, t, 0, lse, grad, dx, dw)
    work = space(n, d, v, dtype, 0)
    with no_waits():
        loss, lost = forward(x, w, t, 0, work)
        assert L.tf_linear_ce_status(work.data_ptr(), stream()) == _lib.TF_ERR_TIMEOUT
        assert loss[counts].isnan().all() and (loss[~counts] == 0).all() and lost.isnan().all()
        for reduction in (1, 2):
            assert forward(x, w, t, reduction)[0].isnan().all()
        more = space(n, d, v, dtype, 1)
        backward(x, w, t, 0, lse, grad, lost_dx, lost_dw, more)
        assert L.tf_linear_ce_status(more.data_ptr(), stream()) == _lib.TF_ERR_TIMEOUT
        assert lost_dx.isnan().all() and lost_dw.isnan().all()
    backward(x, w, t, 0, lost, grad, lost_dx, lost_dw, more)  # gradients of a loss that was lost
    assert L.tf_linear_ce_status(more.data_ptr(), stream()) == _lib.TF_OK
    assert lost_dx[counts].isnan().all() and (lost_dx[~counts] == 0).all() and lost_dw.isnan().all()
    loss, again = forward(x, w, t, 0, work)
    assert L.tf_linear_ce_status(work.data_ptr(), stream()) == _lib.TF_OK
    backward(x, w, t, 0, again, grad, lost_dx, lost_dw)
    assert torch.equal(loss, good) and torch.equal(again, lse) and torch.equal(lost_dx, dx) and torch.equal(lost_dw, dw)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,na,nb", [(5, 20, 64), (5003, 47, 256), (20_003, 256, 100)])
@pytest.mark.parametrize("strided", [False, True])
def test_weight_gradients_whose_waits_run_out(no_waits, dtype, m, na, nb, strided):
    import torch
    from tests.test_pack8 import data
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    g = data(m, na + 3, dtype)[:, :na] if strided else data(m, na, dtype)
    codes, exps = ops.pack8(data(m, nb, "float32", 1))
    want = ops.weight_grad8(g, codes, exps)
    with no_waits():
        assert ops.weight_grad8(g, codes, exps).isnan().all()
    assert torch.equal(ops.weight_grad8(g, codes, exps), want)


@pytest.mark.parametrize("v", [40, 300])
def test_status_of_a_call_of_no_rows(built_lib, v):
    """The work space may hold anything before a call."""
    import torch
    L = _lib.lib()
    x, w, t = make(4, 64, v, "float32")
    for backward_ in (0, 1):
        work = torch.full((L.tf_linear_ce_work_bytes(0, 64, v, _lib.F32, backward_),), 255, device="cuda", dtype=torch.uint8)
        for reduction in (0, 1):
            work.fill_(255)
            if backward_:
                dw = torch.ones_like(w)
                backward(x[:0], w, t[:0], reduction, torch.empty(0, device="cuda"), torch.ones(1, device="cuda"), x[:0], dw, work)
                assert (dw == 0).all()
            else:
                forward(x[:0], w, t[:0], reduction, work)
            assert L.tf_linear_ce_status(work.data_ptr(), stream()) == _lib.TF_OK
