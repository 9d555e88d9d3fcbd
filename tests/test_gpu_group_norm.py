"""Group norm + activation on channels-last tensors (kan_sr.ops.group_norm_act): values and gradients against the formula in
64 bits, against differences, over layouts, types and sizes where it can go wrong."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24                                   # half a step of fp32, relative to the value


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def formula(x, w, b, G, eps, act):
    """64-bit y with autograd, and what the tolerances need: xhat, z, mean, rstd broadcast to x's shape."""
    B, C = x.shape[0], x.shape[-1]
    v = x.reshape(B, -1, G, C // G)
    mean = v.mean(dim=(1, 3), keepdim=True)
    rstd = 1 / torch.sqrt((v - mean).square().mean(dim=(1, 3), keepdim=True) + eps)
    xhat = ((v - mean) * rstd).reshape(x.shape)
    z = xhat * w + b
    y = {"none": lambda: z, "relu": lambda: z.clamp_min(0), "silu": lambda: z * torch.sigmoid(z),
         "gelu": lambda: z * 0.5 * (1 + torch.erf(z / math.sqrt(2)))}[act]()
    full = lambda t: t.expand(v.shape).reshape(x.shape)  # noqa: E731
    return y, xhat, z, full(mean), full(rstd)


def z_error(x, w, b, xhat, z, mean, rstd):
    """Bound of |z - z64| in fp32.  mean: a fixed-order sum of sums, at most 32 roundings of its terms on the way, each of size
    |x| <= sigma-free bound |mean| + |x|; x - mean and the products round once more.  rstd: the variance is a sum of squares
    with at most 64 roundings, halved by the square root.  Together at most 48 units of (|x| + |mean|) rstd |w| + |z| + |b|."""
    return 48 * U32 * ((x.abs() + mean.abs()) * rstd * w.abs() + xhat.abs() * w.abs() + z.abs() + b.abs())


def case(shape, G, dtype, act, seed=0, offset=1.0, affine=True):
    g = torch.Generator().manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(shape, generator=g) * (0.5 + torch.rand(C, generator=g)) + offset * torch.randn(C, generator=g)).to(dtype)
    w = 1 + 0.3 * torch.randn(C, generator=g) if affine else torch.ones(C)
    b = 0.3 * torch.randn(C, generator=g) if affine else torch.zeros(C)
    dy = torch.randn(shape, generator=g).to(dtype)
    return x, w, b, dy


def check(x, w, b, dy, G, act, eps=1e-5, affine=True, xd=None, dyd=None, backward=True):
    from kan_sr.ops import group_norm_act
    dtype = x.dtype
    x64 = x.double().requires_grad_()
    w64, b64 = w.double().requires_grad_(), b.double().requires_grad_()
    y64, xhat, z, mean, rstd = formula(x64, w64, b64, G, eps, act)
    with torch.no_grad():
        ez = z_error(x64, w64, b64, xhat, z, mean, rstd)
    if act == "relu":
        dy = torch.where(z.detach().abs() > 4 * ez, dy.double(), 0.0).to(dtype)   # the slope jumps at z = 0: no gradient there
        dyd = dy.cuda()
    xd = x.cuda() if xd is None else xd
    xd = xd.detach().requires_grad_(backward)
    wd, bd = (w.cuda().requires_grad_(backward), b.cuda().requires_grad_(backward)) if affine else (None, None)
    y = group_norm_act(xd, G, wd, bd, eps=eps, activation=act)
    assert y.dtype is dtype and y.shape == x.shape and y.is_contiguous()
    # |act'| <= 1.13; the activation itself: exp2 / rcp / erf of a few units each, on values of at most |z| + 1
    tol = 1.2 * ez + 16 * U32 * (z.abs() + 1) + (half_step(dtype) * (y64.abs() + 2 * ez) if dtype is torch.bfloat16 else 0)
    err = (y.double().cpu() - y64).abs()
    assert bool((err <= tol).all()), float((err / tol).max())
    if not backward:
        return
    y64.backward(dy.double())
    y.backward(dy.cuda() if dyd is None else dyd)
    with torch.no_grad():
        # dz = dy act'(z): |act''| <= 1, act' of a few units; dx = rstd (w dz - mean - xhat mean): every term with the error of
        # dz and of xhat (ez / |w|, bounded through (|x| + |mean|) rstd), and sums of at most 64 roundings
        exh = 48 * U32 * ((x64.abs() + mean.abs()) * rstd + xhat.abs())
        adz = dy.double().abs() * 1.13
        edz = dy.double().abs() * (ez + 16 * U32)
        B, C = x.shape[0], x.shape[-1]
        gmean = lambda t: t.reshape(B, -1, G, C // G).mean(dim=(1, 3), keepdim=True).expand(B, x[0].numel() // C, G, C // G).reshape(x.shape)  # noqa: E731
        aw = w64.abs()
        m1, m2 = gmean(adz * aw), gmean(adz * aw * xhat.abs())
        e = (edz + 64 * U32 * adz) * aw
        tol = rstd * (e + gmean(e) + xhat.abs() * gmean(e * xhat.abs() + adz * aw * exh) + exh * m2) + 64 * U32 * rstd * (m1 + xhat.abs() * m2)
        if dtype is torch.bfloat16:
            tol = tol + half_step(dtype) * (x64.grad.abs() + tol)
        err = (xd.grad.double().cpu() - x64.grad).abs()
        assert xd.grad.dtype is dtype and bool((err <= tol + 1e-300).all()), float((err / (tol + 1e-300)).max())
        if affine:
            csum = lambda t: t.reshape(-1, C).sum(0)  # noqa: E731
            tb = csum(edz + 64 * U32 * adz)
            tw = csum(edz * xhat.abs() + adz * exh + 64 * U32 * adz * xhat.abs())
            assert bool(((bd.grad.double().cpu() - b64.grad).abs() <= tb).all())
            assert bool(((wd.grad.double().cpu() - w64.grad).abs() <= tw).all())


SHAPES = [((1, 1), 1), ((1, 1, 1, 4), 2), ((2, 3, 5, 6), 3), ((1, 16, 16, 64), 8), ((3, 7, 9, 90), 9), ((2, 5, 2050), 1),
          ((2, 33, 1040), 65), ((300, 2, 8), 2), ((1, 9001, 3), 1), ((2, 64, 48, 4), 2), ((5, 1, 12), 4), ((2, 40, 41, 320), 32),
          ((1, 11, 13, 4099), 1), ((4, 257, 24), 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", SHAPES)
def test_values_and_gradients(shape, G, dtype):
    act = ["none", "relu", "silu", "gelu"][(shape[-1] + shape[0]) % 4]
    check(*case(shape, G, dtype, act), G, act)


# too large for one workgroup: groups of 12, 10, 6, 7 and 1 channels (vectors share 4, 2, 1 of them), of several channel blocks, of
# more chunks than are joined without a launch
CHUNKED = [((1, 48, 50, 24), 2), ((2, 47, 47, 40), 4), ((1, 3000, 24), 4), ((1, 2500, 56), 8), ((1, 16500, 136), 136),
           ((1, 400, 2080), 5), ((2, 130, 127, 320), 32)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", CHUNKED)
def test_groups_in_chunks(shape, G, dtype):
    check(*case(shape, G, dtype, "silu", seed=9), G, "silu")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
def test_every_activation(act, dtype):
    check(*case((2, 19, 17, 40), 4, dtype, act, seed=3), 4, act)


def test_without_affine_and_large_mean():
    check(*case((2, 21, 32), 4, torch.float32, "silu", affine=False), 4, "silu", affine=False)
    # mean 2000 spreads: E[x^2] - mean^2 in fp32 would leave nothing of the variance
    check(*case((2, 100, 60, 16), 2, torch.float32, "none", offset=2000.0), 2, "none")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lo,C,wide", [(0, 24, 40), (3, 24, 41), (8, 32, 64)])
def test_channel_slices_and_strided_gradients_in_place(lo, C, wide, dtype):
    x, w, b, dy = case((3, 6, 7, C), 4, dtype, "silu", seed=5)
    big = torch.full((3, 6, 7, wide), float("nan"), dtype=dtype).cuda()
    gbig = big.clone()
    big[..., lo:lo + C] = x.cuda()
    gbig[..., lo:lo + C] = dy.cuda()
    check(x, w, b, dy, 4, "silu", xd=big[..., lo:lo + C], dyd=gbig[..., lo:lo + C])


def test_other_strides_take_a_copy():
    x, w, b, dy = case((2, 6, 5, 12), 3, torch.float32, "gelu", seed=6)
    check(x, w, b, dy, 3, "gelu", xd=x.cuda().permute(0, 3, 1, 2).contiguous().permute(0, 2, 3, 1))      # NCHW memory
    crop = torch.zeros(2, 9, 8, 12).cuda()
    crop[:, 1:7, 2:7] = x.cuda()
    check(x, w, b, dy, 3, "gelu", xd=crop[:, 1:7, 2:7])
    ones = torch.ones_like(dy)
    check(x, w, b, ones, 3, "gelu", dyd=torch.ones(1, device="cuda").expand(2, 6, 5, 12))               # y.sum().backward()


def test_empty_tensors():
    from kan_sr.ops import group_norm_act
    for shape in ((0, 4, 8), (3, 0, 8)):
        x = torch.empty(shape, device="cuda", requires_grad=True)
        w, b = torch.ones(8, device="cuda", requires_grad=True), torch.zeros(8, device="cuda", requires_grad=True)
        y = group_norm_act(x, 2, w, b, activation="silu")
        assert y.shape == shape
        y.sum().backward()
        assert x.grad.shape == shape and float(w.grad.abs().sum()) == 0 and float(b.grad.abs().sum()) == 0


def test_constant_group_and_non_finite_values():
    from kan_sr.ops import group_norm_act
    x = torch.full((2, 50, 8), 3.0, device="cuda")
    assert float(group_norm_act(x, 2).abs().max()) == 0.0
    x = torch.randn(2, 50, 8, device="cuda")
    ref = group_norm_act(x, 2)
    x[1, 7, 5] = float("inf")
    y = group_norm_act(x, 2)
    assert torch.equal(y[0], ref[0]) and torch.equal(y[1, :, :4], ref[1, :, :4])       # other images and groups
    assert bool(torch.isnan(y[1, :, 4:]).all())


def test_gradient_against_differences():
    from kan_sr.ops import group_norm_act
    x, w, b, dy = case((2, 9, 8, 12), 3, torch.float32, "silu", seed=9)
    d = [torch.randn(t.shape, generator=torch.Generator().manual_seed(10 + i)) for i, t in enumerate((x, w, b))]
    args = [t.cuda().requires_grad_() for t in (x, w, b)]
    grads = torch.autograd.grad(group_norm_act(args[0], 3, args[1], args[2], activation="silu"), args, dy.cuda())
    slope = sum(float((g.double().cpu() * v.double()).sum()) for g, v in zip(grads, d))
    h = 2.0 ** -8

    def f(s):
        a = [(t.double() + s * h * v.double()).float().cuda() for t, v in zip((x, w, b), d)]
        return float((group_norm_act(a[0], 3, a[1], a[2], activation="silu").double().cpu() * dy.double()).sum())

    # central differences of step 2^-8: the cubic term is h^2 / 6 of a third derivative of the size of the values (a few units
    # per element, random signs), rounding 1e-7 sqrt(n) / h
    size = float(dy.double().norm())
    assert abs((f(1) - f(-1)) / (2 * h) - slope) <= 40 * h * h * size + 4e-6 / h * size, slope


def test_only_the_gradients_that_are_asked_for():
    from kan_sr.ops import group_norm_act
    x, w, b, dy = (t.cuda() for t in case((2, 30, 16), 4, torch.float32, "silu", seed=11))
    full = torch.autograd.grad(group_norm_act(x.requires_grad_(), 4, w.requires_grad_(), b.requires_grad_(), activation="silu"), (x, w, b), dy)
    x2 = x.detach()
    gw, = torch.autograd.grad(group_norm_act(x2, 4, w, b.detach(), activation="silu"), (w,), dy)
    gx, = torch.autograd.grad(group_norm_act(x, 4, w.detach(), b.detach(), activation="silu"), (x,), dy)
    assert torch.equal(gw, full[1]) and torch.equal(gx, full[0])
    assert not group_norm_act(x2, 4).requires_grad


def test_side_stream_and_repeated_runs_are_bit_equal():
    from kan_sr.ops import group_norm_act
    x, w, b, dy = (t.cuda() for t in case((4, 65, 33, 48), 6, torch.float32, "gelu", seed=12))

    def run():
        args = [t.detach().requires_grad_() for t in (x, w, b)]
        y = group_norm_act(args[0], 6, args[1], args[2], activation="gelu")
        return (y.detach(),) + torch.autograd.grad(y, args, dy)

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(first, second))


def test_calls_on_two_streams_at_once():
    from kan_sr.ops import group_norm_act
    cases = [case(s, G, t, "silu", seed=11) + (G,) for s, G, t in
             (((2, 130, 127, 320), 32, torch.bfloat16), ((4, 64, 64, 64), 8, torch.float32), ((1, 90, 90, 24), 2, torch.float32))]

    def run(x, w, b, dy, G):
        x, w, b = (t.cuda().requires_grad_() for t in (x, w, b))
        dy = dy.cuda()
        torch.cuda.current_stream().synchronize()
        y = group_norm_act(x, G, w, b, activation="silu")
        return (y,) + torch.autograd.grad(y, (x, w, b), dy)

    want = [run(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for k in range(3):
        for c, st in zip(cases, streams):
            with torch.cuda.stream(st):
                got.append(run(*c))
    torch.cuda.synchronize()
    for k, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[k % 3])), k


def test_captured_into_a_graph_and_replayed():
    from kan_sr.ops import group_norm_act
    x, w, b, dy = (t.cuda() for t in case((2, 31, 30, 40), 4, torch.float32, "silu", seed=13))

    def run(x):
        args = [t.detach().requires_grad_() for t in (x, w, b)]
        y = group_norm_act(args[0], 4, args[1], args[2], activation="silu")
        return (y.detach(),) + torch.autograd.grad(y, args, dy)

    run(x)
    static = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(static)
    for k in range(4):
        fresh = x * (k + 1) + k
        static.copy_(fresh)
        graph.replay()
        torch.cuda.synchronize()
        want = run(fresh)                              # eager work between the replays
        assert all(torch.equal(a, c) for a, c in zip(out, want)), k


def test_offsets_beyond_32_bits():
    from kan_sr.ops import group_norm_act
    C, S = 64, (1 << 25) + 77                          # 2.1e9 elements, 4.3 GB in bf16
    x = torch.empty(1, S, C, device="cuda", dtype=torch.bfloat16).normal_(2.0, 3.0)
    x[0, -5:] += 40
    y = group_norm_act(x, 2, activation="silu")
    v = x.view(S, 2, 32)
    n = S * 32
    mean = torch.stack([v[:, g].sum(dtype=torch.float64) for g in range(2)]) / n
    sq = torch.zeros(2, dtype=torch.float64, device="cuda")
    for part in v.split(1 << 22):
        sq += (part.double() - mean[:, None]).square().sum(dim=(0, 2))
    z = (v[-4096:].double() - mean[:, None]) / torch.sqrt(sq / n + 1e-5)[:, None]
    ref = (z * torch.sigmoid(z)).view(1, 4096, C)
    err = (y[:, -4096:].double() - ref).abs()
    assert bool((err <= half_step(torch.bfloat16) * ref.abs() + 200 * U32 * (1 + ref.abs())).all())
