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
