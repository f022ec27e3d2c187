"""Activations in 8 bits (csrc/pack8.cu, pack8.cuh): every step but one rounding is exact, so codes and exponents are compared
bit by bit with the definition in fp64; and the weight gradient from them (csrc/weight_grad8.cu): exact products, chains of at
most 24 additions that cut off (2^-23 each) and fp32 sums of at most 2^13 of those: below 24 * 2^-23 + 2^-24 sqrt(2^13) of random
terms < 5e-6, and half a step u of the result's type.
"""
import pytest

pytestmark = pytest.mark.gpu

U = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}


def reference(x, relu):
    """Codes, exponent bytes and values by the definition."""
    import torch
    n, d = x.shape
    x = x.double()
    v = torch.where(x > 0, x, torch.where(x.isnan(), x, 0.0)) if relu else x
    p = torch.nn.functional.pad(v, (0, -d % 32)).reshape(n, -1, 32)
    bad = ~p.isfinite().all(2, keepdim=True)
    top = torch.where(bad, 1.0, p).abs().amax(2, keepdim=True)
    e = torch.floor(torch.log2(top.clamp(min=2.0 ** -120)))
    e = torch.where(torch.round(top / torch.exp2(e - 6)) > 127, e + 1, e).clamp(max=127)
    code = torch.round(torch.where(bad, 0.0, p) / torch.exp2(e - 6)).clamp(-127, 127)
    value = torch.where(bad, float("nan"), code * torch.exp2(e - 6)).reshape(n, -1)[:, :d]
    code = torch.where(bad, 0, code).reshape(n, -1)[:, :d]
    if relu:
        code = torch.where((x > 0) & (code == 0), -128, code)
    return code.to(torch.int8), torch.where(bad, 255, e + 127).reshape(n, -1).to(torch.uint8), value


def data(n, d, dtype, seed=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(n, d, generator=g, device="cuda") * torch.exp(2 * torch.randn(n, 1, generator=g, device="cuda"))).to(getattr(torch, dtype))


def check(x, relu):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    codes, exps = torch.ops.sw_gcn.pack8(x, relu)
    code, exp, value = reference(x, relu)
    finite = torch.nn.functional.pad(value, (0, -x.shape[1] % 32)).reshape(x.shape[0], -1, 32).isfinite().all(2) if x.numel() else exp == exp
    assert torch.equal(exps, exp)
    assert torch.equal(codes[value.isfinite()], code[value.isfinite()])
    if relu:
        assert torch.equal(codes != 0, x > 0)
    for t in (torch.float32, torch.bfloat16, torch.float16):
        got = torch.ops.sw_gcn.unpack8(codes, exps, t)
        assert got.dtype == t
        want = value.to(t)
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got[~got.isnan()], want[~want.isnan()])
    assert finite is not None


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("n,d", [(1, 1), (1, 32), (3, 33), (17, 100), (1000, 128), (333, 602), (5, 31), (70_001, 16), (2, 5000)])
def test_codes(built_lib, relu, dtype, n, d):
    check(data(n, d, dtype, n + d), relu)


@pytest.mark.parametrize("relu", [False, True])
def test_borders(built_lib, relu):
    """Ties, the largest value next to 128 steps, subnormals, the ends of the range, infinities and NaN, groups of zeros."""
    import torch
    x = torch.zeros(12, 64, device="cuda")
    x[0, :8] = torch.tensor([1.0, 0.5 / 64, 1.5 / 64, 2.5 / 64, -0.5 / 64, -1.5 / 64, 127.5 / 64 - 2 ** -20, 1e-9], device="cuda")
    x[1, 0], x[1, 1] = 127.5 / 64, 1.5 / 64                        # rounds to 128 steps: one more
    x[2, 0] = float(torch.tensor(127.5 / 64).nextafter(torch.tensor(0.0)))
    x[3, 0], x[3, 1] = 2.0 ** -149, -(2.0 ** -149)
    x[4, 0], x[4, 1] = 2.0 ** -120, 2.0 ** -126
    x[5, 0], x[5, 1] = torch.finfo(torch.float32).max, -1e38
    x[6, 0], x[6, 40] = float("inf"), 3.0
    x[7, 0], x[7, 40] = float("nan"), -3.0
    x[8, 63] = -float("inf")
    x[9] = -1.0
    x[10, 0], x[10, 1] = 2.0 ** -119, 2.0 ** -121
    check(x, relu)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("m", [1, 31, 33, 129, 5003])
@pytest.mark.parametrize("na,nb", [(47, 256), (256, 100), (7, 33), (128, 128), (130, 40), (300, 300), (64, 1), (1, 64), (512, 16)])
def test_weight_grad(built_lib, dtype, m, na, nb):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, g = data(m, nb, dtype, m + na), data(m, na, dtype, nb)
    codes, exps = torch.ops.sw_gcn.pack8(x, True)
    want = g.double().t() @ torch.ops.sw_gcn.unpack8(codes, exps).double()
    first = None
    for _ in range(2):
        got = torch.ops.sw_gcn.weight_grad8(g, codes, exps)
        assert got.dtype == g.dtype and got.shape == (na, nb)
        # sums beyond the type's range (fp16: some of 5 003 rows of these spreads) are infinities; next to its end either will do
        top, got64 = torch.finfo(g.dtype).max, got.double()
        assert torch.equal(got64[want.abs() > 1.001 * top], want[want.abs() > 1.001 * top].sign() * float("inf"))
        inside = want.abs() < 0.999 * top
        off = (got64 - want)[inside].norm().item()
        assert off <= (U[dtype] + 5e-6) * want[inside].norm().item(), off / want[inside].norm().item()
        assert first is None or torch.equal(got, first)
        first = got


def test_strides_and_foreign_codes(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    x = data(40, 75, "float32")
    codes, exps = ops.pack8(x)
    wide = torch.zeros(40, 90, device="cuda")
    wide[:, 7:82] = x
    for other in (wide[:, 7:82], x.t().contiguous().t(), x.requires_grad_()):
        c, e = ops.pack8(other)
        assert torch.equal(c, codes) and torch.equal(e, exps) and not c.requires_grad
    value = ops.unpack8(codes, exps)
    g = data(40, 9, "float32", 1)
    grad = ops.weight_grad8(g, codes, exps)
    for c in (codes.contiguous(), codes.clone(), codes.t().contiguous().t()):  # rows of 75 bytes, and columns in turn
        assert torch.equal(ops.unpack8(c, exps), value) and torch.equal(ops.weight_grad8(g, c, exps), grad)
    some = ops.unpack8(codes[8:24], exps[8:24])
    assert torch.equal(some, value[8:24])
    assert torch.equal(ops.weight_grad8(g[8:24], codes[8:24], exps[8:24]), ops.weight_grad8(g[8:24].clone(), codes[8:24].clone(), exps[8:24].clone()))
    gs = torch.zeros(40, 20, device="cuda")
    gs[:, 4:13] = g
    assert torch.equal(ops.weight_grad8(gs[:, 4:13], codes, exps), grad)
    none = ops.weight_grad8(g[:0], codes[:0], exps[:0])
    assert none.shape == (9, 75) and (none == 0).all()
    c, e = ops.pack8(x[:0])
    assert c.shape == (0, 75) and ops.unpack8(c, e).shape == (0, 75)


# ranges of 16 rows off the CTAs' ranges, operands that need several tiles, and G in all the ways that rows are read
@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("m,na,nb", [(100_003, 40, 60), (20_011, 256, 128), (20_011, 128, 256), (9_999, 257, 260), (30_001, 33, 300)])
def test_weight_grad_of_many_rows(built_lib, dtype, m, na, nb):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    gen = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, nb, generator=gen, device="cuda")
    g = (torch.randn(m, na, generator=gen, device="cuda") / m ** 0.5).to(getattr(torch, dtype))
    codes, exps = torch.ops.sw_gcn.pack8(x, False)
    want = g.double().t() @ torch.ops.sw_gcn.unpack8(codes, exps).double()
    got = torch.ops.sw_gcn.weight_grad8(g, codes, exps)
    off = (got.double() - want).norm().item()
    assert off <= (U[dtype] + 5e-6) * want.norm().item(), off / want.norm().item()


def test_rows_that_are_not_finite_and_large_steps(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, g = data(100, 64, "float32"), data(100, 20, "float32", 1)
    x[3, 40] = float("inf")
    codes, exps = torch.ops.sw_gcn.pack8(x)
    dw = torch.ops.sw_gcn.weight_grad8(g, codes, exps)
    assert dw[:, 32:].isnan().all() and dw[:, :32].isfinite().all()
    x = data(64, 32, "float32").sign() * 2.0 ** 120
    g = data(64, 20, "float32", 2) * 2.0 ** -100
    codes, exps = torch.ops.sw_gcn.pack8(x)
    want = g.double().t() @ x.double()
    assert (torch.ops.sw_gcn.weight_grad8(g, codes, exps).double() - want).norm().item() <= 5e-6 * want.norm().item()


def test_refusals(built_lib):
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    x = data(8, 40, "float32")
    codes, exps = ops.pack8(x)
    for f, args in ((ops.pack8, (x.cpu(),)), (ops.pack8, (x.double(),)), (ops.pack8, (x[0],)), (ops.pack8, (x[:, :0],)), (ops.unpack8, (codes.int(), exps)),
                    (ops.unpack8, (codes, exps[:, :1])), (ops.unpack8, (codes, exps, torch.float64)), (ops.unpack8, (codes.cpu(), exps.cpu())),
                    (ops.weight_grad8, (x[:4], codes, exps)), (ops.weight_grad8, (x.double(), codes, exps)), (ops.weight_grad8, (x, codes, exps.int()))):
        with pytest.raises(ValueError):
            f(*args)


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("n,d", [(1, 1), (37, 33), (500, 32), (333, 602), (64, 256), (70_001, 30), (3, 5000)])
def test_mask(built_lib, dtype, n, d):
    """relu_grad8_ alone: a gradient stays, bit by bit, where the packed value was positive, and is zero elsewhere, infinities and NaN among both."""
    import torch
    from tile_fusion_b200 import dense_ops, sw_gcn  # noqa: F401
    x, g = data(n, d, dtype, n), data(n, d, dtype, d)
    x[n // 2, d // 2] = 1e-7  # (rounds to zero)
    g[n // 2, d // 2], g[0, 0] = float("inf"), float("nan")
    codes = torch.ops.sw_gcn.pack8(x, True)[0]
    full = torch.as_strided(codes, (n, -(-d // 32) * 32), (-(-d // 32) * 32, 1))
    want = torch.where(x > 0, g, torch.zeros_like(g))
    got = dense_ops.relu_grad8_(g.clone(), full)
    assert torch.equal(got.view(torch.uint8), want.view(torch.uint8))


@pytest.mark.parametrize("dtype", list(U))
@pytest.mark.parametrize("na,nb", [(20, 64), (47, 256), (300, 40)])
def test_gradients_that_are_not_finite(built_lib, dtype, na, nb):
    """An infinity in G makes the sums that it takes part in infinite (NaN where it meets a zero, another sign or a NaN), as the formula has it."""
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x, g = data(150, nb, "float32"), data(150, na, dtype, 1)
    g[3, 2], g[7, 5], g[140, 5], g[60, 9], g[61, 10] = float("inf"), float("-inf"), float("inf"), float("nan"), float("inf")
    x[61, :3] = 0
    codes, exps = torch.ops.sw_gcn.pack8(x)
    got = torch.ops.sw_gcn.weight_grad8(g, codes, exps).double()
    want = g.double().t() @ torch.ops.sw_gcn.unpack8(codes, exps).double()
    bad = ~want.isfinite()
    assert bad.any(1).sum().item() == 4 and torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[want.isinf()], want[want.isinf()])
    off = (got - want)[~bad].norm().item()
    assert off <= (U[dtype] + 5e-6) * want[~bad].norm().item()


def test_gradients_next_to_the_end_of_fp32(built_lib):
    """Values beyond bf16's largest that are numbers."""
    import torch
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    x = data(40, 32, "float32").sign() * 2.0 ** -20
    g = data(40, 20, "float32", 2)
    g[:, 3] = torch.finfo(torch.float32).max
    g[5, 4] = -3.4e38
    codes, exps = torch.ops.sw_gcn.pack8(x)
    got = torch.ops.sw_gcn.weight_grad8(g, codes, exps).double()
    want = g.double().t() @ x.double()
    for c in range(20):  # (columns of their own size each)
        assert (got[c] - want[c]).norm().item() <= 5e-6 * 40 ** 0.5 * 2.0 ** -20 * g[:, c].double().norm().item()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_positive_values_far_below_their_groups(built_lib, dtype):
    """The smallest subnormals beside values of 2^8 and more: scaled, they are nothing, but they were positive."""
    import torch
    x = torch.zeros(6, 64, device="cuda", dtype=getattr(torch, dtype))
    tiny = 2.0 ** (-149 if dtype == "float32" else -133)
    for i, big in enumerate((1.0, 2.0 ** 7, 2.0 ** 8, 2.0 ** 30, 2.0 ** 126, 2.0 ** 127)):
        x[i, 0], x[i, 1], x[i, 2], x[i, 33] = big, tiny, -tiny, tiny
    check(x, True)
    check(x, False)


def test_tangents_and_traces(built_lib):
    """These operators carry no graph: a forward-mode tangent is refused, not dropped.  A trace records the operators themselves."""
    import torch
    from torch.autograd import forward_ad
    from tile_fusion_b200 import sw_gcn  # noqa: F401
    ops = torch.ops.sw_gcn
    x, g = data(20, 40, "float32"), data(20, 8, "float32", 1)
    codes, exps = ops.pack8(x)
    value, dw = ops.unpack8(codes, exps), ops.weight_grad8(g, codes, exps)
    with forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="pack8"):
            ops.pack8(forward_ad.make_dual(x, torch.ones_like(x)))
        with pytest.raises(RuntimeError, match="weight_grad8"):
            ops.weight_grad8(forward_ad.make_dual(g, torch.ones_like(g)), codes, exps)
        assert torch.equal(ops.unpack8(*ops.pack8(x)), value) and torch.equal(ops.weight_grad8(g, codes, exps), dw)
    z, h = data(20, 40, "float32", 2), data(20, 8, "float32", 3)
    traced = torch.jit.trace(lambda x, g: (ops.unpack8(*ops.pack8(x)), ops.weight_grad8(g, *ops.pack8(x))), (x, g))
    for a, b in ((x, g), (z, h)):
        codes, exps = ops.pack8(a)
        got = traced(a, b)
        assert torch.equal(got[0], ops.unpack8(codes, exps)) and torch.equal(got[1], ops.weight_grad8(b, codes, exps))


def test_mask_refuses(built_lib):
    import torch
    from tile_fusion_b200 import dense_ops
    g, c = torch.zeros(6, 40, device="cuda"), torch.zeros(6, 64, device="cuda", dtype=torch.int8)
    for grad, codes in ((g.cpu(), c), (g, c.cpu()), (g.double(), c), (g, c.int()), (g[:, :8], c), (g, c[:5]), (g, c[:, :40]), (g, c[:, :32]), (g[:, 0], c),
                        (torch.zeros(6, 70, device="cuda"), c)):
        with pytest.raises(ValueError):
            dense_ops.relu_grad8_(grad, codes)
    assert dense_ops.relu_grad8_(torch.ones(6, 40, device="cuda"), c).sum() == 0
    assert dense_ops.relu_grad8_(g[:0], c[:0]).shape == (0, 40)
