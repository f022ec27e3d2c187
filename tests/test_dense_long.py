"""The dense operators where offsets pass 32 bits: operands of more than 2^31 values.  Rows do not touch each other, so the last rows
are compared with the same operator on a copy of them alone (which the other tests compare with the formulas), in their places; sums
over rows have values in the first and the last rows only.

Tolerances: rows on their own are the same operations in the same order (bit by bit); the loss of many rows and of few may cut its
products differently, and sums over rows are added in another order: 2e-5 of the 2-norm, as for the sums of the other tests, and half a
step of the type where a result was rounded to it once on either side.
"""
import math

import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def ends(t, k):
    import torch
    return torch.cat((t[:k], t[-k:]))


def near(got, want, u):
    off = (got.double() - want.double()).norm().item()
    assert off <= (2 * u + 2e-5) * want.double().norm().item(), off / want.double().norm().item()


@pytest.mark.parametrize("cols,checkpoint", [(2048, False), (250, True)])
def test_layer_norm(built_lib, cols, checkpoint):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    n, k = 2 ** 31 // cols + 1000, 300
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(n, cols, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    g = torch.zeros_like(x)
    g[:k].normal_(generator=gen)
    g[-k:].normal_(generator=gen)
    w, b = torch.randn(cols, generator=gen, device="cuda"), torch.randn(cols, generator=gen, device="cuda")

    def run(x, g):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        y = ops.layer_norm(*leaves, 1e-5, checkpoint)
        return (y.detach(),) + torch.autograd.grad(y, leaves, g)

    y, dx, dw, db = run(x, g)
    want = run(ends(x, k), ends(g, k))
    assert torch.equal(ends(y, k), want[0])
    assert torch.equal(ends(dx, k), want[1])
    assert not dx[k:-k:1000].any()
    near(dw, want[2], U["float32"])
    near(db, want[3], U["float32"])


def test_8_bits(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    d, k = 100, 500
    n = 2 ** 31 // d + 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(n, d, device="cuda", dtype=torch.float16).normal_(generator=gen)
    codes, exponents = ops.pack8(x, True)
    some = ops.pack8(ends(x, k), True)
    assert torch.equal(ends(codes, k), some[0]) and torch.equal(ends(exponents, k), some[1])
    back = ops.unpack8(codes, exponents, torch.bfloat16)
    assert torch.equal(ends(back, k), ops.unpack8(*some, torch.bfloat16))
    del back, x
    g = torch.zeros(n, 104, device="cuda", dtype=torch.bfloat16)
    g[:k].normal_(generator=gen)
    g[-k:].normal_(generator=gen)
    near(ops.weight_grad8(g, codes, exponents), ops.weight_grad8(ends(g, k), *some), U["bfloat16"])


@pytest.mark.parametrize("d,v,dtype", [(256, 40, "bfloat16"), (2048, 300, "float16")])
def test_loss_of_many_rows(built_lib, d, v, dtype):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    n, k = 2 ** 31 // d + 1000, 500
    gen = torch.Generator(device="cuda").manual_seed(0)
    x = torch.empty(n, d, device="cuda", dtype=getattr(torch, dtype)).normal_(generator=gen)
    w = (torch.randn(v, d, generator=gen, device="cuda") / math.sqrt(d)).to(x.dtype)
    target = torch.full((n,), -100, device="cuda")
    target[:k] = torch.randint(0, v, (k,), generator=gen, device="cuda")
    target[-k:] = torch.randint(0, v, (k,), generator=gen, device="cuda")

    def run(x, target):
        x, p = x.detach().requires_grad_(), w.detach().requires_grad_()
        loss = torch.ops.sw_gcn.linear_cross_entropy(x, p, target, -100, "none")
        return (loss.detach(),) + torch.autograd.grad(loss.sum(), (x, p))

    loss, dx, dw = run(x, target)
    want = run(ends(x, k), ends(target, k))
    near(ends(loss, k), want[0], U["float32"])
    near(ends(dx, k), want[1], U[dtype])
    near(dw, want[2], U[dtype])
    assert not loss[k:-k].any() and not dx[k:-k:1000].any()


def test_loss_of_many_classes(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    n, d = 70, 4096
    v = 2 ** 31 // d + 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    w = (torch.empty(v, d, device="cuda", dtype=torch.bfloat16).normal_(generator=gen).mul_(1 / math.sqrt(d))).requires_grad_()
    x = torch.randn(n, d, generator=gen, device="cuda").to(torch.bfloat16).requires_grad_()
    target = torch.randint(v - 900, v, (n,), generator=gen, device="cuda")
    loss = torch.ops.sw_gcn.linear_cross_entropy(x, w, target, -100, "mean")
    dx, dw = torch.autograd.grad(loss, (x, w))
    with torch.no_grad():
        logits = torch.cat([x.double() @ p.double().t() for p in w.split(65536)], 1)
        p = torch.softmax(logits, 1)
        want = (torch.logsumexp(logits, 1) - logits.gather(1, target[:, None])[:, 0]).mean()
        p[torch.arange(n, device="cuda"), target] -= 1
        p /= n
        assert abs(loss.item() - want.item()) <= 2e-5
        near(dw[-1000:], p[:, -1000:].t() @ x.double(), U["bfloat16"])
        near(dw[:1000], p[:, :1000].t() @ x.double(), U["bfloat16"])
        near(dx, sum(q.double() @ c.double() for q, c in zip(p.split(65536, 1), w.split(65536))), U["bfloat16"])


def test_weight_gradient_of_many_rows_of_one_sign(built_lib):
    """The tensor core cuts off what it adds (2e-8 of the sum at a time), so an accumulator may not add up all rows: 10^8 equal products.
    Tolerance: at most 4 096 additions to a sum, 1e-4, and the result's rounding."""
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    n = 100_000_000
    codes, exponents = torch.ops.sw_gcn.pack8(torch.ones(1, 1, device="cuda"))
    g = torch.full((n, 8), 1 / 3000.5, device="cuda", dtype=torch.float16)
    one = codes.new_full((n, 32), int(codes[0, 0]))
    got = torch.ops.sw_gcn.weight_grad8(g, one, exponents[0, 0].expand(n, 1).contiguous())
    want = n * g[0, 0].double().item()
    off = (got.double() / want - 1).abs().max().item()
    assert off <= U["float16"] + 1e-4, off


@pytest.mark.parametrize("cols", [256, 250])
def test_mask_of_8_bits(built_lib, cols):
    """More than 2^31 codes: the gradient behind a ReLU, and the layer's codes, at the first rows and the last."""
    import torch
    from tile_fusion_b200 import dense_ops, sw_gcn  # noqa: F401
    n = 2 ** 31 // 256 + 1000
    gen = torch.Generator(device="cuda").manual_seed(0)
    codes = torch.randint(-1, 2, (n, 256), generator=gen, device="cuda", dtype=torch.int8)
    grad = torch.empty(n, cols, device="cuda", dtype=torch.bfloat16).normal_(generator=gen)
    want = [torch.where(c[:, :cols] != 0, g, torch.zeros_like(g)) for c, g in zip(codes.split(1 << 20), grad.split(1 << 20))]
    dense_ops.relu_grad8_(grad, codes)
    for got, w in zip(grad.split(1 << 20), want):
        assert torch.equal(got, w)
    del want
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,na,nb", [("bfloat16", 2048, 2048), ("float16", 1900, 2100)])
def test_weight_gradient_in_several_launches(built_lib, dtype, na, nb):
    """More ranges of 32 768 rows than are summed in one launch: values in the first and last rows and on both sides of the launches' border."""
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    n, k = 700_003, 200
    border = 16 * 31_824  # 22 ranges, of 31 824 rows (whole sixteens) each, 2^26 sums or 16 of them a launch
    gen = torch.Generator(device="cuda").manual_seed(0)
    some = torch.cat([torch.arange(a, b, device="cuda") for a, b in ((0, k), (border - k, border + k), (n - k, n))])
    x = torch.empty(n, nb, device="cuda", dtype=getattr(torch, dtype)).normal_(generator=gen)
    g = torch.zeros(n, na, device="cuda", dtype=x.dtype)
    g[some] = torch.empty(len(some), na, device="cuda", dtype=x.dtype).normal_(generator=gen)
    codes, exponents = ops.pack8(x)
    got = ops.weight_grad8(g, codes, exponents)
    kept = ops.unpack8(codes[some], exponents[some]).double()
    near(got, g[some].double().t() @ kept, U[dtype])
    assert torch.equal(got, ops.weight_grad8(g, codes, exponents))
    for part in (slice(0, k), slice(k, 3 * k), slice(3 * k, 4 * k)):  # each of the three has its say
        alone = torch.zeros_like(g)
        alone[some[part]] = g[some[part]]
        near(ops.weight_grad8(alone, codes, exponents), g[some[part]].double().t() @ kept[part], U[dtype])
