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
    # (dw and db are rounded to the type of weight and bias, which is one)
    u, uw = U[str(x.dtype)[6:]], U[str(next(t for t in (w, b, x) if t is not None).dtype)[6:]]
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


@pytest.mark.parametrize("dtype,w_dtype", [("float32", "float32"), ("bfloat16", "float32"), ("float16", "float32"), ("float32", "bfloat16"), ("bfloat16", "float16")])
@pytest.mark.parametrize("cols", [96, 1000])
def test_weights_of_other_types_and_none(built_lib, dtype, w_dtype, cols):
    x, w, b, g = data((37, cols), dtype, w_dtype)
    check(x, w, b, g)
    check(x, w, None, g)
    check(x, None, b, g)
    check(x, None, None, g)
    check(x, w, None, g, checkpoint=True)


@pytest.mark.parametrize("dtype", list(U))
def test_strides_dimensions_and_empty(built_lib, dtype):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, w, b, g = data((4, 6, 50), dtype)
    check(x, w, b, g)
    want = run(x.reshape(24, 50), w, b, g.reshape(24, 50))
    wide = torch.zeros(24, 61, device="cuda", dtype=x.dtype)
    wide[:, 5:55] = x.reshape(24, 50)
    for xs, gs in ((wide[:, 5:55], g.reshape(24, 50)), (x.reshape(24, 50).t().contiguous().t(), g.reshape(24, 50).t().contiguous().t()), (x.reshape(24, 50), g.reshape(24, 50)[:, :])):
        for p, q in zip(run(xs, w, b, gs), want):
            assert torch.equal(p, q)
    row = run(x[0, 0], w, b, g[0, 0])
    assert row[0].shape == (50,) and torch.equal(row[0], want[0][0])
    shared = run(x.reshape(24, 50), w, b, g[0, :1].expand(24, 50))  # one gradient for all rows
    near(shared[3], 24 * g[0, 0].double(), U[dtype] + 5e-6)
    y, dx, dw, db = run(x.reshape(24, 50)[:0], w, b, g.reshape(24, 50)[:0])
    assert y.shape == (0, 50) and dx.shape == (0, 50) and (dw == 0).all() and (db == 0).all()


def test_far_from_zero_and_bad_rows(built_lib):
    """Rows whose mean is 2 000 times their spread keep their variance (centred values), constant rows give the bias, and a row that
    is not finite leaves the others alone."""
    import torch
    x, w, b, g = data((64, 256), "float32")
    far = x + 2000
    # x is off by 2^-13 in units of 1 (its own rounding, which the reference has too); the mean by 2^-13 more at most
    near(run(far, w, b, g)[0], reference(far, w, b, g)[0], 2.0 ** -13)
    flat = torch.full_like(x, 3.25)
    y, dx, _, _ = run(flat, w, b, g)
    assert torch.equal(y, b.expand_as(y)) and dx.isfinite().all()
    bad = x.clone()
    bad[5] = float("nan")
    bad[9, 3] = float("inf")
    keep = [i for i in range(64) if i not in (5, 9)]
    got, want = run(bad, w, b, g), run(x, w, b, g)
    assert torch.equal(got[0][keep], want[0][keep]) and torch.equal(got[1][keep], want[1][keep])
    assert got[0][[5, 9]].isnan().all()


def test_against_differences(built_lib):
    import torch
    x, w, b, g = data((10, 40), "float32")
    _, dx, dw, db = run(x, w, b, g)
    gen = torch.Generator(device="cuda").manual_seed(1)
    f = lambda x, w, b: (run(x, w, b, g)[0].double() * g.double()).sum().item()  # noqa: E731
    for i, grad in enumerate((dx, dw, db)):
        u = torch.randn(grad.shape, generator=gen, device="cuda")
        u /= u.norm()
        h, at = 2.0 ** -6, [x, w, b]
        up, down = list(at), list(at)
        up[i], down[i] = at[i] + h * u, at[i] - h * u
        # y carries 2^-22 in 400 terms of about one: 1e-5 over 2 h; the third-order term is h^2 of a derivative of order one
        assert abs((f(*up) - f(*down)) / (2 * h) - (grad.double() * u).sum().item()) <= 2e-3 * grad.norm().item() + 1e-3


def test_streams_and_graphs(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, w, b, g = data((200, 640), "bfloat16")
    want = run(x, w, b, g, True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, b, g, True)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(got, want))
    xs, ws, bs = (t.clone().requires_grad_() for t in (x, w, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = torch.ops.sw_gcn.layer_norm(xs, ws, bs, 1e-5, True)
        grads = torch.autograd.grad(y, (xs, ws, bs), g)
    x2 = data((200, 640), "bfloat16", seed=7)[0]
    for a, want_ in ((x2, run(x2, w, b, g, True)), (x, want)):
        with torch.no_grad():
            xs.copy_(a)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip((y.detach(), *grads), want_))


def test_refusals(built_lib):
    import torch
    from tile_fusion_b200 import _lib, sw_gcn  # noqa: F401
    call = torch.ops.sw_gcn.layer_norm
    x, w, b, g = data((4, 16), "float32")
    for args in ((x.cpu(),), (x.double(),), (x, w[:8]), (x, w, b[:8]), (x, w.cpu()), (x, w, b.bfloat16()), (x[:, :0],), (x, w.long())):
        with pytest.raises(ValueError):
            call(*args)
    with pytest.raises(_lib.TileFusionError, match="columns"):
        call(torch.zeros(2, 16_385, device="cuda"))


def test_tangents_and_traces(built_lib):
    """A forward-mode tangent is refused, not dropped, whether or not anything requires a gradient; a trace records the operator."""
    import torch
    from torch.autograd import forward_ad
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    gen = torch.Generator(device="cuda").manual_seed(0)
    x, z = torch.randn(2, 30, 40, generator=gen, device="cuda")
    w, b = torch.randn(2, 40, generator=gen, device="cuda")
    y, yz = ops.layer_norm(x, w, b), ops.layer_norm(z, w, b)
    with forward_ad.dual_level():
        dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), w, b), (x, dual(w), b), (x, w, dual(b))):
            with pytest.raises(RuntimeError):
                ops.layer_norm(*args)
            with pytest.raises(RuntimeError), torch.no_grad():
                ops.layer_norm(*args)
        assert torch.equal(ops.layer_norm(x, w, b), y)
    traced = torch.jit.trace(lambda t: ops.layer_norm(t, w, b), (x,))
    assert torch.equal(traced(x), y) and torch.equal(traced(z), yz)
