"""The dense operators together, as a deep GCN trains with them: a layer that keeps its input in 8 bits, a norm that keeps its input in 8
bits, the next layer behind its ReLU, and the loss; values and gradients against the same formulas in fp64, at the kept values.

The adjacency is symmetric, as the layers assume.  Hidden values next to zero fall on one side of the ReLU or on the other by
rounding; the reference takes the side from the fp32 values.  Tolerance: products of at most 64 terms by split TF32 (2e-6),
norms and sums of fp32 terms (5e-6, see their tests), through two layers and their gradients: 1e-4 of the 2-norm.
"""
import math

import pytest

pytestmark = pytest.mark.gpu


def near(got, want, tol=1e-4):
    off = (got.double() - want).norm().item()
    assert off <= tol * want.norm().item(), off / want.norm().item()


def graph(n, seed=0):
    import numpy as np
    import torch
    from tile_fusion_b200 import synth
    ap, ai, ax = synth.rmat_gcn(seed, n, 8)
    a = torch.sparse_csr_tensor(torch.from_numpy(np.asarray(ap)), torch.from_numpy(np.asarray(ai)), torch.from_numpy(np.asarray(ax)), size=(len(ap) - 1,) * 2).cuda()
    return a, a.to_dense().double()


@pytest.mark.parametrize("relu", [False, True])
def test_layer_that_keeps_8_bits(built_lib, relu):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    adj, dense = graph(1000)
    n = dense.shape[0]
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, 40, generator=gen, device="cuda").requires_grad_()
    w = (torch.randn(24, 40, generator=gen, device="cuda") / 6).requires_grad_()
    g = torch.randn(n, 24, generator=gen, device="cuda")
    sched = ops.inspect(adj, 64)
    y = ops.fusedGeMMSpMM_ck8(adj, x, w, sched, 4, relu)
    assert torch.equal(y, ops.fusedGeMMSpMM(adj, torch.relu(x) if relu else x, w, sched, 4))
    dx, dw = torch.autograd.grad(y, (x, w), g)
    kept = ops.unpack8(*ops.pack8(x.detach(), relu)).double()
    ag = dense @ g.double()
    near(dw, ag.t() @ kept)
    near(dx, (ag @ w.double()) * (x > 0 if relu else 1))
    # the plain layer's gradients, whose weight gradient the 8 bits are 1 % off at most: half a step is 2^-7 of a group's largest value
    px, pw = x.detach().requires_grad_(), w.detach().requires_grad_()
    want = torch.autograd.grad(ops.fusedGeMMSpMM(adj, torch.relu(px) if relu else px, pw, sched, 4), (px, pw), g)
    assert torch.equal(dx, want[0])
    near(dw, want[1].double(), 1e-2)
    with torch.no_grad():
        assert torch.equal(ops.fusedGeMMSpMM_ck8(adj, x, w, sched, 4, relu), y)
    with pytest.raises(ValueError):
        ops.fusedGeMMSpMM_ck8(adj, x[:, :8], w, sched, 4, relu)


def test_training_step(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    adj, dense = graph(1500, seed=2)
    n, f, h, classes = dense.shape[0], 48, 64, 37
    gen = torch.Generator(device="cuda").manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    x = r(n, f)
    w1, w2, head = (r(h, f) / math.sqrt(f)).requires_grad_(), (r(h, h) / math.sqrt(h)).requires_grad_(), (r(classes, h) / math.sqrt(h)).requires_grad_()
    gain, shift = (1 + 0.1 * r(h)).requires_grad_(), (0.1 * r(h)).requires_grad_()
    target = torch.randint(0, classes, (n,), generator=gen, device="cuda")
    target[::3] = -100
    params = (w1, gain, shift, w2, head)

    def step():
        a = ops.fusedGeMMSpMM_ck8(adj, x, w1, [], 4, False)
        b = ops.layer_norm(a, gain, shift, 1e-5, True)
        c = ops.fusedGeMMSpMM_ck8(adj, b, w2, [], 4, True)
        loss = ops.linear_cross_entropy(c, head, target)
        return loss, a, b, c, torch.autograd.grad(loss, params)

    loss, a, b, c, grads = step()
    kept = lambda t, relu: ops.unpack8(*ops.pack8(t.detach(), relu)).double()  # noqa: E731
    d1, d2, dh, dg, ds = (p.detach().double() for p in (w1, w2, head, gain, shift))
    ra = dense @ (x.double() @ d1.t())
    mean, var = ra.mean(1, keepdim=True), ra.var(1, unbiased=False, keepdim=True)
    rstd = (var + 1e-5).rsqrt()
    rb = (ra - mean) * rstd * dg + ds
    on = b.detach() > 0
    rc = dense @ (torch.where(on, rb, 0) @ d2.t())
    logp = torch.log_softmax(rc @ dh.t(), 1)
    ok = target >= 0
    rows = ok.nonzero()[:, 0]
    near(a.detach(), ra, 2e-5)
    near(b.detach(), rb, 5e-5)
    near(c.detach(), rc, 5e-5)
    want = -logp[rows, target[rows]].mean()
    assert abs(loss.item() - want.item()) <= 1e-4
    p = logp.exp()
    p[rows, target[rows]] -= 1
    p = p * (ok / len(rows))[:, None]
    gc = p @ dh
    ag = dense @ gc
    gb = (ag @ d2) * on
    xh = (kept(a, False) - mean) * rstd
    hh = gb * dg
    ga = rstd * (hh - hh.mean(1, keepdim=True) - xh * (hh * xh).mean(1, keepdim=True))
    ag1 = dense @ ga
    for got, ref in zip(grads, (ag1.t() @ kept(x, False), (gb * xh).sum(0), gb.sum(0), ag.t() @ kept(b, True), p.t() @ rc)):
        near(got, ref)
    again = step()
    assert torch.equal(again[0], loss) and all(torch.equal(s, t) for s, t in zip(again[4], grads))


def test_weights_whose_gradient_is_refused(built_lib):
    """2^27 entries: refused before anything is allocated, by the layer in its forward pass, not in the backward one."""
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    i = torch.arange(5, dtype=torch.int32)
    adj = torch.sparse_csr_tensor(i, i[:4], torch.ones(4), size=(4, 4)).cuda()
    w = torch.zeros(1 << 14, 1 << 13, device="cuda").requires_grad_()
    with pytest.raises(ValueError, match="entries"):
        ops.fusedGeMMSpMM_ck8(adj, torch.ones(4, 1 << 13, device="cuda"), w, [], 1)
    codes, exponents = ops.pack8(torch.ones(2, 1 << 20, device="cuda"))
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    with pytest.raises(ValueError, match="entries"):
        ops.weight_grad8(torch.ones(2, 1 << 20, device="cuda"), codes, exponents)
    assert torch.cuda.max_memory_allocated() < before + (1 << 31)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float16", "columns first"])
def test_layer_of_other_features(built_lib, dtype, relu):
    """Features in 16 bits, or whose columns lie apart, are the same as their copy in fp32, stay as they are, and are copied once."""
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    adj, _ = graph(20_000)
    n, k = adj.shape[0], 512
    gen = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(n, k, generator=gen, device="cuda")
    x = (x.t().contiguous().t() if dtype == "columns first" else x.to(getattr(torch, dtype))).requires_grad_()
    w = (torch.randn(24, k, generator=gen, device="cuda") / 6).requires_grad_()
    g = torch.randn(n, 24, generator=gen, device="cuda")
    before = x.detach().clone()
    plain = x.detach().float().contiguous().requires_grad_()
    y = ops.fusedGeMMSpMM_ck8(adj, plain, w, [], 4, relu)
    want = (y.detach(),) + torch.autograd.grad(y, (plain, w), g)
    del y, plain
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    y = ops.fusedGeMMSpMM_ck8(adj, x, w, [], 4, relu)
    assert torch.cuda.max_memory_allocated() - held < 1.5 * 4 * n * k  # the copy in fp32, its 8 bits
    got = (y.detach(),) + torch.autograd.grad(y, (x, w), g)
    assert torch.equal(x.detach(), before) and got[1].dtype == x.dtype
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1].to(x.dtype)) and torch.equal(got[2], want[2])
