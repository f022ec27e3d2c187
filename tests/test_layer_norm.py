"""Layer norm and its gradients (csrc/layer_norm.cu) against the formulas in fp64.

Tolerances, relative to the 2-norm, u = half a step of the values' type: results are rounded once (u).  Sums over n <= 16 384
columns of fp32 terms keep 2^-24 sqrt(n) of their terms' norm (a thread adds 16 in turn, the rest pairwise), below 1e-6; the
mean is subtracted from values of at most 8 standard deviations' distance, 4 bits at most: 1e-6.  Sums over rows: chains of m / 4096
terms and more for fewer CTAs, below 2^-24 times their number, at most 3e-6 here, of sums that random signs make as small as
their terms' norm.  Asserted u + 3e-6 for y and dx, u + 5e-6 for dw and db.
"""
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def reference(x, w, b, g, eps=1e-5, kept=None):
    import torch
    x = x.detach().double()
    mean, var = x.mean(-1, keepdim=True), x.var(-1, unbiased=False, keepdim=True)
    r = (var + eps).rsqrt()
    wd = w.detach().double() if w is not None else torch.ones(x.shape[-1], device=x.device, dtype=torch.float64)
    y = (x - mean) * r * wd + (b.detach().double() if b is not None else 0)
    xh = ((x if kept is None else kept.double()) - mean) * r
    g = g.double()
    h = g * wd
    dx = r * (h - h.mean(-1, keepdim=True) - xh * (h * xh).mean(-1, keepdim=True))
    rows = tuple(range(x.dim() - 1))
    return y, dx, (g * xh).sum(rows), g.sum(rows)


def near(got, want, tol):
    assert got.shape == want.shape
    off = (got.double() - want).norm().item()
    assert off <= tol * want.norm().item() + 1e-30, off / max(want.norm().item(), 1e-30)


def data(shape, dtype, w_dtype=None, seed=0):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    t, wt, d = getattr(torch, dtype), getattr(torch, w_dtype or dtype), shape[-1]
    x = (r(*shape) * (0.5 + torch.rand(d, generator=gen, device="cuda")) + r(*shape[:-1], 1)).to(t)
    return x, (1 + 0.1 * r(d)).to(wt), (0.1 * r(d)).to(wt), r(*shape).to(t)


def run(x, w, b, g, checkpoint=False, eps=1e-5):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, w, b = (t.detach().requires_grad_() if t is not None else None for t in (x, w, b))
    y = torch.ops.sw_gcn.layer_norm(x, w, b, eps, checkpoint)
    grads = iter(torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], g))
    return (y.detach(), *(next(grads) if t is not None else None for t in (x, w, b)))


def check(x, w, b, g, checkpoint=False):
    import torch
    u, uw = U[str(x.dtype)[6:]], U[str((w if w is not None else x).dtype)[6:]]
    kept = torch.ops.sw_gcn.unpack8(*torch.ops.sw_gcn.pack8(x.reshape(-1, x.shape[-1])), torch.float32).reshape(x.shape) if checkpoint else None
    got, want = run(x, w, b, g, checkpoint), reference(x, w, b, g, kept=kept)
    near(got[0], want[0], u + 3e-6)
    near(got[1], want[1], u + 3e-6)
    if w is not None:
        near(got[2], want[2], uw + 5e-6)
    if b is not None:
        near(got[3], want[3], uw + 5e-6)
    for p, q in zip(got, run(x, w, b, g, checkpoint)):
        assert p is None or torch.equal(p, q)


# columns around what eight lanes, a warp and a CTA hold with 16, 8, 4 and 2 bytes an access; rows around those of a CTA
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 7), (1, 512), (33, 64), (257, 100), (70, 128), (65, 129), (1000, 256), (31, 514), (300, 602),
                                       (129, 1024), (17, 1433), (40, 4096), (9, 8192), (5, 8200), (3, 12_001), (2, 16_384), (20_000, 47)])
@pytest.mark.parametrize("checkpoint", [False, True])
def test_values_and_gradients(built_lib, dtype, rows, cols, checkpoint):
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    if cols == 1:  # one column: xh is zero, and dx a difference of equal numbers
        x, w, b, g = data((rows, cols), dtype)
        got, want = run(x, w, b, g), reference(x, w, b, g)
        near(got[0], want[0], U[dtype] + 3e-6)
        near(got[3], want[3], U[dtype] + 5e-6)
        assert got[1].abs().max().item() <= 1e-6 * g.abs().max().item() / 1e-5 ** 0.5
        return
    check(*data((rows, cols), dtype, seed=rows + cols), checkpoint=checkpoint)
