"""Softmax cross entropy of a linear layer without its logits (csrc/linear_ce.cu) against the formula in fp64.

Tolerances.  u = 2^-24 (fp32), 2^-8 (bf16), 2^-11 (fp16) is half a step of the operands' type.
  loss   logits of |l| <= ~12 summed in chains of at most 24 additions that cut off (2^-23 of the sum each) and added up by at
         most 2^6 roundings in fp32; 16-bit operands multiply exactly, split fp32 operands leave out 3 * 2^-22 of a product.
         Together below 40 * 2^-23 of |x| |w| <= 60: 3e-4 in the worst case, and its root mean square over the terms of random
         signs is 10 to 50 times smaller.  Asserted: 2e-5 absolute on a loss of 1 to 12.
  dx, dw relative to the 2-norm.  Slopes are rounded once (u; fp32: two planes, 2^-22), sums are rounded once (u), a logit error of
         1e-5 shows as 1e-5 of a slope: asserted 2 u + 2e-5 (fp32: 2e-5).
"""
import math

import pytest

pytestmark = pytest.mark.gpu

TYPES = ("float32", "bfloat16", "float16")


def make(n, d, v, dtype, seed=0, ignored=0.2):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = getattr(torch, dtype)
    w = (torch.randn(v, d, generator=g, device="cuda") / math.sqrt(d)).to(t)
    target = torch.randint(0, v, (n,), generator=g, device="cuda")
    x = (torch.randn(n, d, generator=g, device="cuda") + 3 * w[target].float()).to(t)
    target[torch.rand(n, generator=g, device="cuda") < ignored] = -100
    return x, w, target


def reference(x, w, target, reduction="mean", grad=1.0):
    import torch
    x, w = x.detach().double(), w.detach().double()
    ok = target != -100
    x = torch.where(ok[:, None], x, 0)
    logp = torch.log_softmax(x @ w.t(), 1)
    at = torch.where(ok, target, 0)
    rows = torch.where(ok, -logp.gather(1, at[:, None])[:, 0], 0)
    number = max(1, int(ok.sum())) if reduction == "mean" else 1
    p = logp.exp()
    p[torch.arange(len(at), device=at.device), at] -= 1
    g = torch.as_tensor(grad, device=x.device, dtype=torch.float64) / number
    p = p * (ok * g)[:, None]
    loss = rows if reduction == "none" else rows.sum() / number
    return loss, p @ w, p.t() @ x


def near(got, want, u):
    off = (got.double() - want).norm().item()
    assert off <= (2 * u + 2e-5 if u > 2 ** -20 else 2e-5) * want.norm().item() + 1e-30, off / max(want.norm().item(), 1e-30)


U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def run(x, w, target, reduction="mean", grad=None):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, w = x.detach().requires_grad_(), w.detach().requires_grad_()
    loss = torch.ops.sw_gcn.linear_cross_entropy(x, w, target, -100, reduction)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), grad))


# rows around a tile of 256 and a CTA's 128, columns around a slice of 64 terms and off the 16-byte grid, vocabularies around the
# widths 64, 128 and 256 of a tile
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(1, 8, 2), (1, 64, 1000), (5, 33, 7), (128, 64, 64), (129, 65, 65), (255, 128, 128), (257, 96, 257),
                                   (300, 200, 513), (64, 1024, 5000), (1000, 50, 47), (513, 130, 129)])
def test_loss_and_gradients(built_lib, dtype, n, d, v):
    x, w, t = make(n, d, v, dtype, seed=n + d)
    scale = float(n) if dtype == "float16" else 1.0
    import torch
    loss, dx, dw = run(x, w, t, grad=torch.tensor(scale, device="cuda"))
    want, wx, ww = reference(x, w, t, grad=scale)
    assert loss.dtype == torch.float32 and dx.dtype == x.dtype and dw.dtype == w.dtype
    assert abs(loss.double() - want).item() <= 2e-5
    near(dx, wx, U[dtype])
    near(dw, ww, U[dtype])
    again = run(x, w, t, grad=torch.tensor(scale, device="cuda"))
    assert torch.equal(again[0], loss) and torch.equal(again[1], dx) and torch.equal(again[2], dw)


# several pieces of the vocabulary, sums cut in parts, and the reductions
@pytest.mark.parametrize("n,d,v,dtype", [(4096, 64, 70_001, "bfloat16"), (3000, 40, 50_000, "float32"), (9000, 72, 33, "float16")])
@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_pieces_and_reductions(built_lib, n, d, v, dtype, reduction):
    import torch
    x, w, t = make(n, d, v, dtype)
    g = torch.linspace(-1, 2, n, device="cuda") if reduction == "none" else torch.tensor(64.0 if reduction == "mean" else 0.25, device="cuda")
    loss, dx, dw = run(x, w, t, reduction, g)
    want, wx, ww = reference(x, w, t, reduction, g)
    assert loss.shape == want.shape
    assert (loss.double() - want).abs().max().item() <= 2e-5 * (n if reduction == "sum" else 1)
    near(dx, wx, U[dtype])
    near(dw, ww, U[dtype])


@pytest.mark.parametrize("n,d,v,dtype", [(20_000, 41, 7_000, "float32"), (20_000, 63, 15_000, "bfloat16"), (20_000, 300, 100, "float32"), (19_001, 129, 301, "float16")])
def test_rows_of_gradients_that_start_anywhere(built_lib, n, d, v, dtype):
    """Enough tiles that no sum is cut, so that the products store the gradients themselves; the first two in pieces of classes.

    A mean over 19 001 rows makes gradients of 1e-6, below fp16's smallest normal number 2^-14, where its steps are 2^-24 whatever the
    value: a result is off by half of that, 2^-25, besides its relative part; over all of them by 2^-25 sqrt(their number) at most."""
    import torch
    x, w, target = make(n, d, v, dtype)
    got = run(x, w, target)
    want = reference(x, w, target)
    assert abs(got[0].item() - want[0].item()) <= 2e-5
    for g, r in zip(got[1:], want[1:]):
        off, steps = (g.double() - r).norm().item(), 2.0 ** -25 * math.sqrt(r.numel()) if dtype == "float16" else 0.0
        assert off <= (2 * U[dtype] + 2e-5) * r.norm().item() + steps, off / r.norm().item()
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_that_do_not_count_reach_nothing(built_lib, dtype):
    import torch
    x, w, t = make(300, 64, 130, dtype)
    clean = run(x, w, t)
    bad = t == -100
    assert bad.any()
    x2 = x.clone()
    x2[bad] = float("nan")
    x2[bad.nonzero()[0]] = float("inf")
    for a, b in zip(run(x2, w, t), clean):
        assert torch.equal(a, b)
    assert (clean[1][bad] == 0).all()
    none = torch.full_like(t, -100)
    loss, dx, dw = run(x2, w, none)
    assert loss.item() == 0 and (dx == 0).all() and (dw == 0).all()
    loss, dx, dw = run(x2, w, none, "none", torch.ones(300, device="cuda"))
    assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all()


def test_classes_outside_are_seen(built_lib):
    import torch
    x, w, t = make(50, 32, 10, "float32", ignored=0)
    t[7], t[9] = 10, -3
    loss, dx, _ = run(x, w, t, "none", torch.ones(50, device="cuda"))
    assert loss.isnan().nonzero().flatten().tolist() == [7, 9]
    assert dx.isnan().any(1).nonzero().flatten().tolist() == [7, 9]


@pytest.mark.parametrize("big", [1e-25, 1e-6, 1e12])
def test_magnitudes(built_lib, big):
    """fp32 operands of any magnitude: the planes' powers of two follow the largest value."""
    x, w, t = make(200, 96, 300, "float32")
    loss, dx, dw = run(x * big, w / big, t)
    want, wx, ww = reference(x * big, w / big, t)
    assert abs(loss.double() - want).item() <= 2e-5
    near(dx, wx, U["float32"])
    near(dw, ww, U["float32"])


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_dimensions_and_index_types(built_lib, dtype):
    import torch
    x, w, t = make(60, 48, 70, dtype)
    want = run(x, w, t)
    wide = torch.zeros(60, 57, device="cuda", dtype=x.dtype)
    wide[:, 3:51] = x
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    call = torch.ops.sw_gcn.linear_cross_entropy
    for xs, ws, ts in ((wide[:, 3:51], w, t), (x, w.t().contiguous().t(), t.int()), (x.reshape(3, 20, 48), w, t.reshape(3, 20)), (x.flip(0).flip(0), w, t)):
        xs, ws = xs.detach().requires_grad_(), ws.detach().requires_grad_()
        loss = call(xs, ws, ts)
        gx, gw = torch.autograd.grad(loss, (xs, ws))
        assert torch.equal(loss, want[0]) and torch.equal(gx.reshape(60, 48), want[1]) and torch.equal(gw, want[2])
    one = x[:1].expand(60, 48).detach().requires_grad_()  # rows that are one row in memory
    loss = call(one, w, t)
    assert abs(loss.double() - reference(x[:1].expand(60, 48), w, t)[0]).item() <= 2e-5
    with torch.no_grad():
        assert torch.equal(call(x, w, t), want[0])
    only = w.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(call(x, only, t), only)[0], want[2])
    only = x.detach().requires_grad_()
    assert torch.equal(torch.autograd.grad(call(only, w, t), only)[0], want[1])
    empty = call(x[:0], w, t[:0])
    assert empty.item() == 0
    none = torch.full((60,), 7, device="cuda")
    assert call(x, w, none, 7).item() == 0 and call(x, w, none, 7, "none").shape == (60,)


def test_against_differences(built_lib):
    """The gradient along a direction, and the loss to both sides of it: in fp32 losses carry 1e-6, a step of 1/32 leaves 4e-4 of a
    third-order term."""
    import torch
    x, w, t = make(100, 32, 50, "float32")
    _, dx, dw = run(x, w, t)
    g = torch.Generator(device="cuda").manual_seed(5)
    for a, grad in (("x", dx), ("w", dw)):
        u = torch.randn(grad.shape, generator=g, device="cuda")
        u /= u.norm()
        h = 1 / 32
        f = lambda s: run(x + s * u if a == "x" else x, w + s * u if a == "w" else w, t, "sum")[0].double()  # noqa: E731
        number = int((t != -100).sum())
        assert abs(((f(h) - f(-h)) / (2 * h) / number).item() - (grad * u).sum().item()) <= 2e-3 * grad.norm().item() + 1e-4 / number


def test_streams_and_graphs(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, w, t = make(300, 64, 500, "float32")
    want = run(x, w, t)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run(x, w, t)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    xs, ws = x.clone().requires_grad_(), w.clone().requires_grad_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = torch.ops.sw_gcn.linear_cross_entropy(xs, ws, t)
        grads = torch.autograd.grad(loss, (xs, ws))
    x2, w2, _ = make(300, 64, 500, "float32", seed=3)
    want2 = run(x2, w2, t)
    for a, b, want_ in ((x2, w2, want2), (x, w, want)):
        with torch.no_grad():
            xs.copy_(a)
            ws.copy_(b)
        graph.replay()
        assert torch.equal(loss.detach(), want_[0]) and torch.equal(grads[0], want_[1]) and torch.equal(grads[1], want_[2])


def test_refusals(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    call = torch.ops.sw_gcn.linear_cross_entropy
    x, w, t = make(8, 16, 5, "float32")
    for args in ((x.cpu(), w, t), (x, w.cpu(), t), (x, w, t.cpu()), (x.double(), w.double(), t), (x, w.bfloat16(), t), (x[:, :8], w, t), (x, w, t[:4]),
                 (x, w, t.float()), (x, w[0], t), (x, w[:0], t), (x, w, t, -100, "average")):
        with pytest.raises(ValueError):
            call(*args)
    loss = call(x.requires_grad_(), w, t)
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# the one class of a part, a part among others, all classes; few classes and many
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v,first,last", [(300, 64, 40, 39, 40), (300, 64, 65, 64, 65), (300, 64, 129, 128, 129), (300, 64, 257, 256, 257), (200, 40, 1000, 64, 192),
                                              (9000, 24, 20_001, 19_968, 20_001), (50, 48, 200, 0, 200)])
def test_classes_that_are_nan_are_seen(built_lib, dtype, n, d, v, first, last):
    """A NaN among a row's logits makes its loss NaN, wherever the row's target is; rows that do not count have none."""
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, w, t = make(n, d, v, dtype)
    t[t >= first] = 0
    w[first:last] = float("nan")
    loss = torch.ops.sw_gcn.linear_cross_entropy(x, w, t, -100, "none")
    assert loss[t >= 0].isnan().all() and (loss[t < 0] == 0).all()
    assert torch.ops.sw_gcn.linear_cross_entropy(x, w, t).isnan()
    _, dx, _ = run(x, w, t)
    assert dx[t >= 0].isnan().all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,v", [(100, 40), (100, 300), (9000, 40), (9000, 300)])
@pytest.mark.parametrize("size", [1e-36, 1e-30])
def test_tiny_gradients_of_rows(built_lib, dtype, n, v, size):
    """A gradient to each row, all of them tiny and some zero: the power of two that brings the largest to one is held in the range.

    fp32 and bf16: as elsewhere, in the types' normal range.  fp16: results are below half of its smallest number."""
    import torch
    x, w, t = make(n, 64, v, dtype)
    g = size * torch.linspace(1, 4, n, device="cuda")
    g[::7] = 0
    _, dx, dw = run(x, w, t, "none", g)
    _, wx, ww = reference(x, w, t, "none", g)
    assert (dx[::7] == 0).all()
    if dtype == "float16":
        assert (dx == 0).all() and (dw == 0).all()
    else:
        scale = 1 / size  # (squares of 1e-36 are no numbers of fp32; the norms are fp64's)
        near(dx.double() * scale, wx * scale, U[dtype])
        near(dw.double() * scale, ww * scale, U[dtype])


@pytest.mark.parametrize("v", [40, 300])
def test_rows_of_zeros_beside_huge_ones(built_lib, v):
    """fp32 operands of 2^100 and rows of zeros, whose logits are zero: their loss is log(classes), their gradient (1 / classes - onehot) @ w."""
    import torch
    x, w, t = make(64, 32, v, "float32", ignored=0)
    x, w = x * 2.0 ** 100, w * 2.0 ** 100
    x[::2] = 0
    g = torch.zeros(64, device="cuda")
    g[::2] = 1
    loss, dx, _ = run(x, w, t, "none", g)
    want, wx, _ = reference(x[::2], w, t[::2], "none", 1.0)
    assert (loss[::2].double() - want).abs().max().item() <= 2e-5
    near(dx[::2], wx, U["float32"])


def test_tangents_and_traces(built_lib):
    """A forward-mode tangent is refused, not dropped; a trace records the operator."""
    import torch
    from torch.autograd import forward_ad
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    call = torch.ops.sw_gcn.linear_cross_entropy
    x, w, t = make(30, 40, 50, "float32")
    z = make(30, 40, 50, "float32", seed=1)[0]
    loss, other = call(x, w, t), call(z, w, t)
    with forward_ad.dual_level():
        for a, b in ((forward_ad.make_dual(x, torch.ones_like(x)), w), (x, forward_ad.make_dual(w, torch.ones_like(w)))):
            with pytest.raises(RuntimeError):
                call(a, b, t)
        assert torch.equal(call(x, w, t), loss)
    traced = torch.jit.trace(lambda a: call(a, w, t), (x,))
    assert torch.equal(traced(x), loss) and torch.equal(traced(z), other)


@pytest.mark.parametrize("dtype", TYPES[1:])
def test_memory_of_a_large_vocabulary(built_lib, dtype):
    """Beside the gradients: the piece of the slope, the copy of x and less; no copy of the weight."""
    import torch
    n, d, v = 64, 1024, 100_000
    x, w, t = make(n, d, v, dtype)
    run(x, w, t)
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with torch.no_grad():
        from tile_fusion_b200 import sw_gcn  # noqa: F401
        torch.ops.sw_gcn.linear_cross_entropy(x, w, t)
    assert torch.cuda.max_memory_allocated() - before < 2 * v * d // 8
    torch.cuda.reset_peak_memory_stats()
    run(x, w, t)
    assert torch.cuda.max_memory_allocated() - before < 2 * v * d + (100 << 20)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,d,v", [(1, 1, 2), (3, 1, 100), (2, 257, 2), (1, 300, 65), (5, 2, 20_000)])
def test_smallest_sizes(built_lib, dtype, n, d, v):
    """One row, one column: slopes are rounded to the type before products of one or two terms, so tolerances are taken of the summands, not of
    their sum: 2 u of sum |P| |w|."""
    import torch
    x, w, t = make(n, d, v, dtype, ignored=0)
    loss, dx, dw = run(x, w, t, "sum")
    want, wx, ww = reference(x, w, t, "sum")
    assert abs(loss.double() - want).item() <= 2e-5 * n
    logp = torch.log_softmax(x.double() @ w.double().t(), 1)
    p = logp.exp()
    p[torch.arange(n, device="cuda"), t] -= 1
    bound = 2 * U[dtype] + 2e-5
    small = 2.0 ** -24 if dtype == "float16" else 0.0  # (its steps below 2^-14)
    assert ((dx.double() - wx).abs() <= bound * (p.abs() @ w.double().abs()) + small).all()
    assert ((dw.double() - ww).abs() <= bound * (p.abs().t() @ x.double().abs()) + small + 1e-6 * x.double().abs().sum(0)).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [8, 257])
def test_one_class(built_lib, dtype, d):
    """The loss over one class is zero whatever the logits, up to their rounding: 2^-23 of |logit| < 32."""
    import torch
    x, w, t = make(40, d, 1, dtype)
    loss, dx, dw = run(x, w, t, "sum")
    assert abs(loss.item()) <= 40 * 2.0 ** -18
    assert dx.abs().max().item() <= 2.0 ** -18 * w.abs().max().item() and dw.abs().max().item() <= 40 * 2.0 ** -18 * x.abs().max().item()
