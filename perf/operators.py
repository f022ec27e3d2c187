"""Cases by which the speed of the training operators is measured: layer norm, activations kept in 8 bits, and the linear
cross entropy, as the layers of a deep graph network (and any other network of dense layers) call them.

``own`` false: the operators in elementary torch operations; true: the library's, through ``torch.ops.sw_gcn``.
"""
import math

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_GROUP = 32      # values that share a power of two
_EPS = 1e-5


def listed():
    return [
        # One row through a norm: inference for a single node or token, where the call itself is what counts.
        dict(name="norm_row", kind="norm", rows=1, cols=512, dtype="bf16", train=False, keep8=False),
        # The norm of a hidden layer of a full-batch GCN (the training benchmark's nodes), forward and backward.
        dict(name="norm_nodes", kind="norm", rows=120_001, cols=256, dtype="fp32", train=True, keep8=False),
        # The norm of a wide dense network in bf16.
        dict(name="norm_wide", kind="norm", rows=16_384, cols=4096, dtype="bf16", train=True, keep8=False),
        # A norm that keeps its input in 8 bits for its backward pass, on a width that is no multiple of anything in use.
        dict(name="norm_keep8", kind="norm", rows=50_021, cols=602, dtype="fp32", train=True, keep8=True),
        # A mini-batch's activations put into 8 bits and read back.
        dict(name="pack_batch", kind="pack", rows=300, cols=100, dtype="bf16", relu=False),
        # A large graph's hidden activations put into 8 bits behind their ReLU and read back: the attention benchmark's nodes.
        dict(name="pack_graph", kind="pack", rows=1_048_576, cols=128, dtype="fp32", relu=True),
        # The weight gradient of a narrow last layer from its input in 8 bits, in mixed precision.
        dict(name="grad8_last", kind="grad8", rows=500_009, cols=256, outs=47, dtype="bf16", relu=True),
        # The weight gradient of the first layer of the benchmark's two-layer GCN (100 -> 256, all nodes), in fp32.
        dict(name="grad8_first", kind="grad8", rows=2_449_029, cols=100, outs=256, dtype="fp32", relu=False),
        # The loss of a small evaluation batch over a small vocabulary.
        dict(name="loss_small", kind="loss", rows=64, cols=128, vocab=1000, dtype="fp32", train=False),
        # Node classification: many nodes, few classes, fp32, with its gradient.
        dict(name="loss_nodes", kind="loss", rows=120_001, cols=256, vocab=47, dtype="fp32", train=True),
        # A language model's head on a short batch, odd vocabulary.
        dict(name="loss_text", kind="loss", rows=4096, cols=2048, vocab=50_021, dtype="bf16", train=True),
        # The largest: a wide head, a large vocabulary, a full batch.
        dict(name="loss_large", kind="loss", rows=8192, cols=4096, vocab=128_000, dtype="fp16", train=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("norm", "pack", "grad8", "loss"))
    dtype = rng.choice(("fp32", "bf16", "fp16"))
    if kind == "norm":
        cols = _log(rng, 32, 8192)
        return dict(kind=kind, rows=_log(rng, 1, min(1 << 20, (1 << 27) // cols)), cols=cols, dtype=dtype, train=rng.random() < 0.7,
                    keep8=rng.random() < 0.3)
    if kind == "pack":
        cols = _log(rng, 16, 4096)
        return dict(kind=kind, rows=_log(rng, 1, min(2_500_000, (1 << 28) // cols)), cols=cols, dtype=dtype, relu=rng.random() < 0.5)
    if kind == "grad8":
        cols, outs = _log(rng, 16, 1024), _log(rng, 16, 512)
        return dict(kind=kind, rows=_log(rng, 1, min(2_500_000, (1 << 29) // (cols + outs))), cols=cols, outs=outs, dtype=dtype,
                    relu=rng.random() < 0.5)
    if rng.random() < 0.35:  # few classes, many rows
        return dict(kind=kind, rows=_log(rng, 1000, 500_000), cols=_log(rng, 16, 512), vocab=_log(rng, 10, 200), dtype=dtype,
                    train=rng.random() < 0.7)
    cols = _log(rng, 32, 4096)
    return dict(kind=kind, rows=_log(rng, 1, 8192), cols=cols, vocab=_log(rng, 500, 128_000), dtype=dtype, train=rng.random() < 0.7)


def _scale(case):
    """What the loss is multiplied by for its backward pass: in fp16 gradients of a mean over many rows would be too small."""
    return 2.0 ** int(math.log2(case["rows"])) if case["dtype"] == "fp16" else 1.0


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t, n, d = _TYPES[case["dtype"]], case["rows"], case["cols"]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    s = dict(case)
    if case["kind"] == "norm":
        # activations: columns of different spread, rows off zero
        s["x"] = (normal(n, d) * (0.5 + torch.rand(d, generator=g, device="cuda")) + normal(n, 1)).to(t).requires_grad_(case["train"])
        s["weight"] = (1 + 0.1 * normal(d)).to(t).requires_grad_(case["train"])
        s["bias"] = (0.1 * normal(d)).to(t).requires_grad_(case["train"])
        s["grad"] = normal(n, d).to(t)
    elif case["kind"] == "pack":
        s["x"] = (normal(n, d) * torch.exp(0.5 * normal(n, 1))).to(t)
    elif case["kind"] == "grad8":
        s["x"] = (normal(n, d) * torch.exp(0.5 * normal(n, 1))).to(t)
        s["grad"] = (normal(n, case["outs"]) / math.sqrt(n)).to(t)
    else:
        # a head in the middle of its training: a row's own class stands out of the others, one row in ten counts for nothing
        v = case["vocab"]
        s["weight"] = (normal(v, d) / math.sqrt(d)).to(t).requires_grad_(case["train"])
        s["target"] = torch.randint(0, v, (n,), generator=g, device="cuda")
        s["x"] = (normal(n, d) + 4 * s["weight"].detach()[s["target"]].float()).to(t).requires_grad_(case["train"])
        s["target"][torch.rand(n, generator=g, device="cuda") < 0.1] = -100
        s["scale"] = torch.tensor(_scale(case), device="cuda")
    return s


# ---- the plain forms ----

def _plain_pack(x, relu):
    """The values that 8 bits keep: groups of 32 columns of a row share a power of two, a value is a whole number of steps of
    its 64th part, at most 127 of them, the nearest one."""
    n, d = x.shape
    x = x.float()
    if relu:
        x = x.clamp(min=0)
    p = torch.nn.functional.pad(x, (0, -d % _GROUP)).view(n, -1, _GROUP)
    top = p.abs().amax(2, keepdim=True)
    e = (torch.frexp(top).exponent - 1).clamp(min=-120)

    def power(k):  # 2^k, bit by bit
        return ((k + 127) << 23).view(torch.float32)

    e = torch.where((top * power(6 - e)).round() > 127, e + 1, e).clamp(max=127)
    step = power(e - 6)
    return ((p * power(6 - e)).round().clamp(-127, 127) * step).view(n, -1)[:, :d]


def _plain_norm(s):
    x, w, b = s["x"].detach().float(), s["weight"].detach().float(), s["bias"].detach().float()
    mean = x.mean(1, keepdim=True)
    c = x - mean
    rstd = 1 / (c.square().mean(1, keepdim=True) + _EPS).sqrt()
    t = s["x"].dtype
    y = (c * rstd * w + b).to(t)
    if not s["train"]:
        return y
    xh = (_plain_pack(x, False) - mean) * rstd if s["keep8"] else c * rstd
    g = s["grad"].float()
    h = g * w
    dx = rstd * (h - h.mean(1, keepdim=True) - xh * (h * xh).mean(1, keepdim=True))
    return y, dx.to(t), (g * xh).sum(0).to(t), g.sum(0).to(t)


def _plain_loss(s):
    x, w, target = s["x"].detach().float(), s["weight"].detach().float(), s["target"]
    logits = x @ w.t()
    counts = target >= 0
    at = target.clamp(min=0)[:, None]
    lse = torch.logsumexp(logits, 1)
    number = counts.sum().clamp(min=1)
    loss = torch.where(counts, lse - logits.gather(1, at)[:, 0], 0).sum() / number
    if not s["train"]:
        return loss
    p = logits.sub_(lse[:, None]).exp_()
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    p.mul_((counts / number * s["scale"])[:, None])
    return loss, (p @ w).to(s["x"].dtype), (p.t() @ x).to(s["x"].dtype)


def _plain(s):
    if s["kind"] == "norm":
        return _plain_norm(s)
    if s["kind"] == "pack":
        return _plain_pack(s["x"], s["relu"]).to(s["x"].dtype)
    if s["kind"] == "grad8":
        return (s["grad"].float().t() @ _plain_pack(s["x"], s["relu"])).to(s["grad"].dtype)
    return _plain_loss(s)


# ---- the library's operators ----

def _own(s):
    from tile_fusion_b200 import sw_gcn  # noqa: F401  (registers torch.ops.sw_gcn)
    ops = torch.ops.sw_gcn
    if s["kind"] == "norm":
        y = ops.layer_norm(s["x"], s["weight"], s["bias"], _EPS, s["keep8"])
        return (y, *torch.autograd.grad(y, (s["x"], s["weight"], s["bias"]), s["grad"])) if s["train"] else y
    if s["kind"] == "pack":
        codes, exponents = ops.pack8(s["x"], s["relu"])
        return ops.unpack8(codes, exponents, s["x"].dtype)
    if s["kind"] == "grad8":
        codes, exponents = ops.pack8(s["x"], s["relu"])
        return ops.weight_grad8(s["grad"], codes, exponents)
    loss = ops.linear_cross_entropy(s["x"], s["weight"], s["target"])
    return (loss, *torch.autograd.grad(loss, (s["x"], s["weight"]), s["scale"])) if s["train"] else loss


def run(state):
    if own:
        return _own(state)
    with torch.no_grad():
        return _plain(state)


def work(case):
    n, d, b = case["rows"], case["cols"], _BYTES[case["dtype"]]
    if case["kind"] == "norm":
        return {"bytes": (4 if case["train"] else 2) * n * d * b + (4 if case["train"] else 2) * d * b, "flops": (20 if case["train"] else 8) * n * d}
    if case["kind"] == "pack":
        return {"bytes": 2 * n * d * b, "flops": 4 * n * d}
    if case["kind"] == "grad8":
        return {"bytes": (n * (d + case["outs"]) + d * case["outs"]) * b, "flops": 2 * n * d * case["outs"]}
    once = (n + case["vocab"]) * d * b
    return {"bytes": (2 if case["train"] else 1) * once + 8 * n, "flops": (6 if case["train"] else 2) * n * d * case["vocab"]}


# ---- the definitions in 64 bits ----

def _exact_pack(x, relu):
    n, d = x.shape
    a = torch.where(x > 0, x.double(), 0) if relu else x.double()
    out = torch.zeros(n, -(-d // _GROUP) * _GROUP, dtype=torch.float64, device=a.device)
    out[:, :d] = a
    groups = out.reshape(-1, _GROUP)
    top = groups.abs().max(1).values
    unit = torch.exp2(torch.floor(torch.log2(top.clamp(min=2.0 ** -120)))) / 64
    unit = torch.where(torch.round(top / unit) > 127, 2 * unit, unit).clamp(max=2.0 ** 121)[:, None]
    return (torch.round(groups / unit).clamp(-127, 127) * unit).reshape(n, -1)[:, :d]


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x = s["x"].detach()
        if case["kind"] == "pack":
            return _exact_pack(x, case["relu"])
        if case["kind"] == "grad8":
            return torch.einsum("io,ic->oc", s["grad"].double(), _exact_pack(x, case["relu"]))
        if case["kind"] == "norm":
            x64, w, b = x.double(), s["weight"].detach().double(), s["bias"].detach().double()
            var, mean = torch.var_mean(x64, 1, unbiased=False, keepdim=True)
            sd = torch.sqrt(var + _EPS)
            y = (x64 - mean) / sd * w + b
            if not case["train"]:
                return y
            kept = (_exact_pack(x, False) - mean) / sd if case["keep8"] else (x64 - mean) / sd
            g = s["grad"].double()
            gw = g * w
            along = torch.einsum("ij,ij->i", gw, kept)[:, None] / case["cols"]
            return y, (gw - gw.mean(1, keepdim=True) - kept * along) / sd, torch.einsum("ij,ij->j", g, kept), g.sum(0)
        w, target = s["weight"].detach().double(), s["target"]
        logp = torch.log_softmax(torch.einsum("id,vd->iv", x.double(), w), 1)
        rows = (target >= 0).nonzero()[:, 0]
        number = max(1, rows.numel())
        loss = -logp[rows, target[rows]].sum() / number
        if not case["train"]:
            return loss
        slope = logp.exp_()
        slope[rows, target[rows]] -= 1
        slope[target < 0] = 0
        slope *= s["scale"].double() / number
        return loss, slope @ w, torch.einsum("iv,id->vd", slope, x.double())
