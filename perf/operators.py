"""Cases, plain forms and 64-bit values of the group-norm and Muon operators.

Four operators: the forward of group norm with an activation on channels-last tensors, the same with its backward, the
orthogonalisation of a matrix by Newton-Schulz products, and the whole Muon update of a list of weight matrices.
`run` computes a case with the framework's kernels where `own` is true, and otherwise in elementary torch operations.
"""
import functools
import math
import os
import sys

import torch

own = False

EPS = 1e-5                              # of the group norm
COEF = (3.4445, -4.7750, 2.0315)        # a, b, c of X <- a X + (b A + c A^2) X, A = X X^T
STEPS = 5
NS_EPS = 1e-7
LR, MOMENTUM, DECAY = 2e-3, 0.95, 0.01


def _package():
    """The framework's package lies in a folder of its own below the repository's root."""
    path = os.path.join(os.getcwd(), "super-resolution_amd")
    if path not in sys.path:
        sys.path.insert(0, path)


# ------------------------------------------------------------------------------------------------ cases
def listed():
    def gn(name, train, batch, height, width, channels, groups, dtype, act):
        return dict(name=name, op="group_norm_train" if train else "group_norm", batch=batch, height=height, width=width,
                    channels=channels, groups=groups, dtype=dtype, act=act)

    def ns(name, batch, rows, cols, dtype):
        return dict(name=name, op="newton_schulz", batch=batch, rows=rows, cols=cols, dtype=dtype)

    def muon(name, layers, width, hidden, convs, outputs):
        return dict(name=name, op="muon", layers=layers, width=width, hidden=hidden, convs=convs, outputs=outputs)

    return [
        # the UNet encoder's bottleneck of one 256 x 256 frame: a call whose time is its latency
        gn("gn 1x16x16x64 f32", False, 1, 16, 16, 64, 8, "float32", "relu"),
        # a wide decoder stage with ten channels a group and sizes that no tile divides
        gn("gn 3x77x93x90 bf16", False, 3, 77, 93, 90, 9, "bfloat16", "gelu"),
        # full-resolution stage of a large image network, far beyond the caches
        gn("gn 4x512x512x128 bf16", False, 4, 512, 512, 128, 32, "bfloat16", "silu"),
        # the UNet encoder's first stage in its training step (8 patches of 256 x 256, 4 channels)
        gn("gn train 8x256x256x4 f32", True, 8, 256, 256, 4, 2, "float32", "silu"),
        # a middle stage with ten channels a group
        gn("gn train 2x128x128x320 bf16", True, 2, 128, 128, 320, 32, "bfloat16", "silu"),
        # a large training batch in fp32
        gn("gn train 16x64x64x512 f32", True, 16, 64, 64, 512, 32, "float32", "silu"),
        # one 1x1 convolution of the hyper-encoder
        ns("ns 64x64 f32", 1, 64, 64, "float32"),
        # odd sides, the longer one second
        ns("ns 777x2051 bf16", 1, 777, 2051, "bfloat16"),
        # a pair of square matrices in fp32
        ns("ns 2x2048x2048 f32", 2, 2048, 2048, "float32"),
        # the largest square matrix
        ns("ns 4096x4096 bf16", 1, 4096, 4096, "bfloat16"),
        # every matrix of the GazeTR hyper-encoder (two transformer layers of width 64, 1x1 convolutions, the x4 head)
        muon("muon hyper-encoder", 2, 64, 32, 6, 160),
        # a wider trunk of the same make
        muon("muon width 512", 2, 512, 2048, 2, 1000),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("group_norm", "group_norm_train", "newton_schulz", "muon"))
    if op.startswith("group_norm"):
        per_group, groups = rng.choice((1, 2, 3, 4, 5, 8, 10, 16, 20, 32)), _log(rng, 1, 40)
        channels = per_group * groups
        # pixels up to the largest listed forward (134 M elements) and training (33 M elements) case
        most = (128 << 20 if op == "group_norm" else 32 << 20) / channels
        batch = min(_log(rng, 1, 24), int(most))
        height, width = _log(rng, 1, 700), _log(rng, 1, 700)
        height = max(1, min(height, int(most / batch)))
        width = max(1, min(width, int(most / batch / height)))
        # at least 32 values a group: over two or three, what is left of x - mean is rounding
        width = max(width, -(-32 // (height * per_group)))
        # the derivative of ReLU jumps at 0: only its forward is drawn
        act = rng.choice(("none", "silu", "gelu") if op.endswith("train") else ("none", "relu", "silu", "gelu"))
        return dict(op=op, batch=batch, height=height, width=width, channels=channels, groups=groups,
                    dtype=rng.choice(("float32", "bfloat16")), act=act)
    if op == "newton_schulz":
        dtype = rng.choice(("float32", "bfloat16"))
        top = 2048 if dtype == "float32" else 4096
        rows, cols = _log(rng, 1, top), _log(rng, 1, top)
        m, n = min(rows, cols), max(rows, cols)
        batch = max(1, min(_log(rng, 1, 48), int(top ** 3 / (m * m * n))))
        return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=dtype)
    width = _log(rng, 16, 512)
    return dict(op=op, layers=rng.randint(1, 3), width=width, hidden=_log(rng, 16, 4 * width), convs=rng.randint(1, 6),
                outputs=_log(rng, 16, 1000))


def _matrices(case):
    """Shapes of a Muon case: per layer the in-projection, out-projection and two linears, then 1x1 convs, 3x3 convs as
    [out, in * 9] and the head."""
    w, h = case["width"], case["hidden"]
    per_layer = [(3 * w, w), (w, w), (h, w), (w, h)]
    return per_layer * case["layers"] + [(w, w)] * case["convs"] + [(max(1, w // 2), 9 * max(1, w // 4)), (case["outputs"], w)]


# ------------------------------------------------------------------------------------------------ inputs
def _gradients(gen, shape, dtype):
    """Matrices like a weight's gradient: a few directions of falling size over noise."""
    *lead, m, n = shape
    r = max(1, min(m, n) // 16)
    left = torch.randn(*lead, m, r, generator=gen, device="cuda")
    right = torch.randn(*lead, r, n, generator=gen, device="cuda")
    size = torch.logspace(0, -1, r, device="cuda") / math.sqrt(r)
    g = (left * size).matmul(right) + 0.1 * torch.randn(*shape, generator=gen, device="cuda")
    return (1e-3 * g).to(dtype)


def _inputs(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"].startswith("group_norm"):
        B, H, W, C = case["batch"], case["height"], case["width"], case["channels"]
        dtype = getattr(torch, case["dtype"])
        # a convolution's output: every channel with a mean and a spread of its own
        x = (randn(B, H, W, C) * (0.5 + randn(C).abs()) + randn(C)).to(dtype)
        s = dict(x=x, weight=1 + 0.2 * randn(C), bias=0.2 * randn(C))
        if case["op"].endswith("train"):
            s["dy"] = (0.01 * randn(B, H, W, C)).to(dtype)
        return s
    if case["op"] == "newton_schulz":
        return dict(g=_gradients(gen, (case["batch"], case["rows"], case["cols"]), getattr(torch, case["dtype"])))
    shapes = _matrices(case)
    return dict(grads=[_gradients(gen, sh, torch.float32) for sh in shapes],
                moms=[4 * _gradients(gen, sh, torch.float32) for sh in shapes],
                weights=[randn(*sh) / math.sqrt(sh[1]) for sh in shapes])


def prepare(case, seed):
    s = _inputs(case, seed)
    s["case"] = case
    if own:
        _package()
        if case["op"] == "muon":
            from kan_sr.muon import Muon
            params = [torch.nn.Parameter(w) for w in s["weights"]]
            for p, g in zip(params, s["grads"]):
                p.grad = g
            s["optimizer"] = Muon(params, lr=LR, momentum=MOMENTUM, weight_decay=DECAY)
            for p, m in zip(params, s["moms"]):
                s["optimizer"].state[p]["momentum_buffer"] = m
            s["params"] = params
        elif case["op"] == "group_norm_train":
            for k in ("x", "weight", "bias"):
                s[k].requires_grad_()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def _act(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "silu":
        return z / (1 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _group_norm(s, case):
    x = s["x"]
    B, H, W, C = x.shape
    G = case["groups"]
    xf = x.float().view(B, H * W, G, C // G)
    mean = xf.mean(dim=(1, 3), keepdim=True)
    d = xf - mean
    rstd = torch.rsqrt((d * d).mean(dim=(1, 3), keepdim=True) + EPS)
    xhat = (d * rstd).view(B, H * W, C)
    z = xhat * s["weight"] + s["bias"]
    y = _act(z, case["act"]).to(x.dtype).view(x.shape)
    if "dy" not in s:
        return y
    dz = s["dy"].float().view(z.shape) * _act_slope(z, case["act"])
    dweight, dbias = (dz * xhat).sum(dim=(0, 1)), dz.sum(dim=(0, 1))
    dxhat = (dz * s["weight"]).view(xf.shape)
    xhat = xhat.view(xf.shape)
    dx = rstd * (dxhat - dxhat.mean(dim=(1, 3), keepdim=True) - xhat * (dxhat * xhat).mean(dim=(1, 3), keepdim=True))
    return y, dx.to(x.dtype).view(x.shape), dweight, dbias


def _ns_step(x, _):
    a, b, c = COEF
    A = x.matmul(x.mT)
    return a * x + (b * A + c * A.matmul(A)).matmul(x)


def _newton_schulz(g):
    x = g.float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + NS_EPS)
    x = functools.reduce(_ns_step, range(STEPS), x)
    return (x.mT if tall else x).to(g.dtype).contiguous()


def _muon(weight, grad, mom):
    mom.mul_(MOMENTUM).add_(grad)
    o = _newton_schulz(grad + MOMENTUM * mom)
    weight.mul_(1 - LR * DECAY).sub_(o, alpha=LR * 0.2 * math.sqrt(max(weight.shape)))
    return weight, mom


def run(state):
    case = state["case"]
    op = case["op"]
    if not own:
        if op.startswith("group_norm"):
            return _group_norm(state, case)
        if op == "newton_schulz":
            return _newton_schulz(state["g"])
        return [_muon(w, g, m) for w, g, m in zip(state["weights"], state["grads"], state["moms"])]
    if op.startswith("group_norm"):
        from kan_sr.ops import group_norm_act
        y = group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], eps=EPS, activation=case["act"])
        if op == "group_norm":
            return y
        return (y,) + torch.autograd.grad(y, (state["x"], state["weight"], state["bias"]), state["dy"])
    if op == "newton_schulz":
        from kan_sr.muon import newton_schulz
        return newton_schulz(state["g"], steps=STEPS, coefficients=COEF, eps=NS_EPS)
    state["optimizer"].step()
    return list(zip(state["weights"], state["moms"]))


# ------------------------------------------------------------------------------------------------ the least a pass can cost
def _ns_flops(rows, cols):
    m, n = min(rows, cols), max(rows, cols)
    return STEPS * (3 * m * m * n + m * m * m)      # A and A^2 are symmetric: half of each


def work(case):
    if case["op"].startswith("group_norm"):
        e = case["batch"] * case["height"] * case["width"] * case["channels"]
        size = 4 if case["dtype"] == "float32" else 2
        train = case["op"].endswith("train")
        return {"bytes": e * size * (4 if train else 2) + case["channels"] * (16 if train else 8), "flops": e * (30 if train else 10)}
    if case["op"] == "newton_schulz":
        e, size = case["batch"] * case["rows"] * case["cols"], 4 if case["dtype"] == "float32" else 2
        return {"bytes": 2 * e * size, "flops": case["batch"] * _ns_flops(case["rows"], case["cols"])}
    shapes = _matrices(case)
    return {"bytes": sum(20 * r * c for r, c in shapes), "flops": sum(_ns_flops(r, c) for r, c in shapes)}


# ------------------------------------------------------------------------------------------------ 64 bits
def _exact_newton_schulz(g):
    """The iteration as one polynomial in the Gram matrix: with P = a I + b A + c A^2 and A' = P A P, X_5 = P_5 ... P_1 X_0."""
    x = g.double()
    if g.shape[-2] > g.shape[-1]:
        return _exact_newton_schulz(g.transpose(-2, -1)).transpose(-2, -1)
    x = x / (torch.linalg.matrix_norm(x, keepdim=True) + NS_EPS)
    a, b, c = COEF
    gram = torch.matmul(x, x.transpose(-2, -1).contiguous())
    eye = torch.eye(gram.shape[-1], dtype=torch.float64, device=x.device)
    product = eye
    for _ in range(STEPS):
        p = a * eye + torch.matmul(gram, b * eye + c * gram)
        product = torch.matmul(p, product)
        gram = torch.matmul(torch.matmul(p, gram), p)
    return torch.matmul(product, x)


def _exact_group_norm(case, s):
    G, B, C = case["groups"], case["batch"], case["channels"]

    def forward(x, w, b):
        v = x.reshape(B, -1, G, C // G)
        var, mean = torch.var_mean(v, dim=(1, 3), correction=0, keepdim=True)
        z = ((v - mean) / torch.sqrt(var + EPS)).reshape(x.shape) * w + b
        if case["act"] == "relu":
            return torch.maximum(z, torch.zeros_like(z))
        if case["act"] == "silu":
            return z * torch.sigmoid(z)
        if case["act"] == "gelu":
            return z * torch.special.ndtr(z)
        return z

    args = [s[k].double() for k in ("x", "weight", "bias")]
    if "dy" not in s:
        return forward(*args)
    args = [t.requires_grad_() for t in args]
    y = forward(*args)
    return (y.detach(),) + torch.autograd.grad(y, args, s["dy"].double())


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"].startswith("group_norm"):
        return _exact_group_norm(case, s)
    if case["op"] == "newton_schulz":
        return _exact_newton_schulz(s["g"])
    out = []
    for w, g, m in zip(s["weights"], s["grads"], s["moms"]):
        mom = MOMENTUM * m.double() + g.double()
        o = _exact_newton_schulz(g.double() + MOMENTUM * mom)
        out.append((w.double() - LR * (DECAY * w.double() + 0.2 * max(w.shape) ** 0.5 * o), mom))
    return out
