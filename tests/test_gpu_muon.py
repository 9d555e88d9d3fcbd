"""Newton-Schulz orthogonalisation and the Muon update (kan_sr.muon) against the iteration in 64 bits.

Tolerances: the iteration multiplies a rounding of an early step by up to 3.4445 per later step, by how much depends on the
singular values.  `model` runs the same iteration in 64 bits with nothing but the operands' roundings put in (f16 hi + lo, or
one f16 with diagonals and linear term exact); the kernels also round every fp32 accumulation, hence the factor."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
COEF = (3.4445, -4.7750, 2.0315)


def exact(u, steps=5, coef=COEF, eps=1e-7):
    x = u.double()
    if x.shape[-2] > x.shape[-1]:
        return exact(u.mT, steps, coef, eps).mT
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + eps)
    for _ in range(steps):
        A = x @ x.mT
        x = coef[0] * x + (coef[1] * A + coef[2] * (A @ A)) @ x
    return x


def f16(x):
    return (x * 1024).half().double() / 1024


def pair(x):
    hi = f16(x)
    return hi + f16((x - hi) * 1024) / 1024


def model(u, split, steps=5, coef=COEF, eps=1e-7):
    x = u.double()
    if x.shape[-2] > x.shape[-1]:
        return model(u.mT, split, steps, coef, eps).mT
    r = pair if split else f16
    eye = torch.eye(x.shape[-2], dtype=torch.float64)
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + eps)
    for k in range(steps):
        xr = x if k == 0 else r(x)
        A = xr @ xr.mT
        d = A.diagonal(dim1=-2, dim2=-1)
        R = r(A - A * eye)
        sq = R @ R
        B = coef[1] * R + coef[2] * ((d[..., :, None] + d[..., None, :]) * R + sq)
        e = coef[1] * d + coef[2] * (d * d + sq.diagonal(dim1=-2, dim2=-1))
        x = (coef[0] + e)[..., None] * (x if k == 0 else pair(x)) + r(B - B * eye) @ xr
    return x


def compare(y, u, split, **kw):
    """y: the kernel's result.  8 x the model's error: an accumulator of K terms rounds as often again as its operands, and the
    sign pattern is another one.  Result types: half a step (bf16 2^-8, fp32 2^-24)."""
    ref = exact(u.cpu(), **kw)
    assert y.shape == u.shape and y.dtype is u.dtype and y.is_contiguous()
    norm = ref.norm(dim=(-2, -1))
    tol = 8 * (model(u.cpu(), split, **kw) - ref).norm(dim=(-2, -1)) + norm * 32 * 2.0 ** -24
    err = y.double().cpu() - ref
    rounding = torch.finfo(y.dtype).eps / 2 * ref.abs()
    over = (err.abs() - rounding).clamp_min(0)
    assert bool((over.norm(dim=(-2, -1)) <= tol).all()), float((over.norm(dim=(-2, -1)) / tol.clamp_min(1e-300)).max())
    # no single element further off than a few times what an even spread allows: a wrong tile would be
    rms = tol / math.sqrt(u.shape[-1] * u.shape[-2])
    few = max(8.0, math.sqrt(u.shape[-1] * u.shape[-2]) / 4) if u.shape[-1] * u.shape[-2] < 4096 else 24.0
    assert bool((over <= few * rms[..., None, None]).all())
    if split and u.dtype is torch.float32 and u[..., 0, 0].numel() and kw.get("steps", 5) == 5:
        assert bool((err.norm(dim=(-2, -1)) <= 1e-5 * norm + 1e-300).all())


def gradients(shape, dtype=torch.float32, seed=0, rank=None):
    g = torch.Generator().manual_seed(seed)
    *lead, m, n = shape
    r = rank or max(1, min(m, n) // 16)
    u = torch.randn(*lead, m, r, generator=g) @ torch.randn(*lead, r, n, generator=g) / math.sqrt(r)
    return (1e-3 * (u + 0.2 * torch.randn(*shape, generator=g))).to(dtype)


SHAPES = [(1, 1), (1, 7), (7, 1), (5, 3), (33, 63), (64, 64), (64, 65), (65, 64), (160, 64), (64, 1024), (1024, 64), (64, 1025),
          (2, 4000), (31, 257), (40, 513), (128, 128), (129, 257), (257, 70), (300, 900), (900, 300), (2, 9, 48, 24), (3, 100, 130)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_newton_schulz_against_64_bits(shape, dtype):
    from kan_sr.muon import newton_schulz
    u = gradients(shape, dtype, seed=sum(shape))
    compare(newton_schulz(u.cuda()), u, dtype is torch.float32 or (min(shape[-2:]) <= 64 and max(shape[-2:]) <= 1024))


@pytest.mark.parametrize("shape", [(1500, 1400), (1400, 1500), (1300, 2048)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_wide_tiles(shape, dtype):
    from kan_sr.muon import newton_schulz
    u = gradients(shape, dtype, seed=7)
    compare(newton_schulz(u.cuda()), u, dtype is torch.float32)


@pytest.mark.parametrize("shape,dtype", [((4, 1900, 1910), torch.bfloat16), ((4, 1910, 1900), torch.bfloat16),
                                         ((3, 1400, 1500), torch.bfloat16), ((3, 1400, 1500), torch.float32),
                                         ((3, 1500, 1400), torch.float32)])
def test_widest_tiles(shape, dtype):
    """Batches whose products take tiles of 128 for A and B, and the first two tiles of 256 for X with a last row and column of
    tiles that are cut off."""
    from kan_sr.muon import newton_schulz
    u = gradients(shape, dtype, seed=8)
    y = newton_schulz(u.cuda())
    for k in (0, shape[0] - 1):
        compare(y[k], u[k], dtype is torch.float32)


@pytest.mark.parametrize("shape", [(48, 80), (200, 150)])
def test_either_precision_for_either_type(shape):
    from kan_sr.muon import newton_schulz
    u = gradients(shape, torch.float32, seed=3)
    small = max(shape) <= 1024 and min(shape) <= 64
    compare(newton_schulz(u.cuda(), precision="fp32"), u, True)
    y = newton_schulz(u.cuda(), precision="bf16").double().cpu()
    ref = exact(u)
    assert float((y - ref).norm()) <= 8 * float((model(u, small) - ref).norm()) + 1e-5 * float(ref.norm())
    compare(newton_schulz(u.bfloat16().cuda(), precision="fp32"), u.bfloat16(), True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape", [(90, 30), (1000, 63), (1000, 62), (500, 60), (3, 70, 12), (900, 4)])
def test_tall_small_matrices(shape, dtype):
    """Rows that are, and are not, whole groups of four values; the same values behind an address that is not a multiple."""
    from kan_sr.muon import newton_schulz
    u = gradients(shape, dtype, seed=44)
    y = newton_schulz(u.cuda())
    compare(y, u, True)
    wide = torch.zeros(*shape[:-1], shape[-1] + 5, dtype=dtype, device="cuda")
    for lo in (1, 4):
        part = wide[..., lo:lo + shape[-1]]
        part.copy_(u)
        assert torch.equal(newton_schulz(part), y)


def test_strides_are_read_in_place():
    from kan_sr.muon import newton_schulz
    for m, n in ((40, 100), (150, 210)):
        u = gradients((3, m, n), seed=m)
        big = torch.full((3, m + 2, 2 * n + 3), float("nan")).cuda()
        view = big[:, 1:-1, 3::2]
        view.copy_(u)
        compare(newton_schulz(view), u, True)
        compare(newton_schulz(view.mT), u.mT, True)
        compare(newton_schulz(u.cuda()[:1].expand(3, m, n)), u[:1].expand(3, m, n), True)
    x = gradients((2, 3, 20, 30), seed=5)
    compare(newton_schulz(x.cuda().transpose(0, 1)), x.transpose(0, 1), True)


@pytest.mark.parametrize("shape", [(24, 40), (100, 140)])
def test_extreme_scales(shape):
    from kan_sr.muon import newton_schulz
    u = gradients(shape, seed=8) * 1e3
    for s in (1e-12, 1e-9, 1e-7, 1e30):
        v = (u.double() * s).float()
        y = newton_schulz(v.cuda()).double().cpu()
        ref = exact(v)
        assert float((y - ref).norm()) <= 1e-5 * float(ref.norm()), s
    # below the square root of the smallest fp32 number: the sum of squares is held in 64 bits
    y = newton_schulz((u * 1e-25).cuda(), eps=0.0).double().cpu()
    ref = exact((u * 1e-25), eps=0.0)
    assert float((y - ref).norm()) <= 1e-5 * float(ref.norm())
    assert float(newton_schulz(torch.zeros(shape).cuda()).abs().max()) == 0.0


@pytest.mark.parametrize("shape", [(24, 40), (100, 140)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_non_finite_matrix_is_nan_and_leaves_the_others(shape, bad):
    from kan_sr.muon import newton_schulz
    u = gradients((3,) + shape, seed=9)
    v = u.clone()
    v[1, 3, 5] = bad
    y, ref = newton_schulz(v.cuda()), newton_schulz(u.cuda())
    assert bool(torch.isnan(y[1]).all()) and torch.equal(y[0], ref[0]) and torch.equal(y[2], ref[2])


@pytest.mark.parametrize("shape", [(24, 40), (100, 140)])
def test_steps_coefficients_and_low_rank(shape):
    from kan_sr.muon import newton_schulz
    u = gradients(shape, seed=10)
    for steps in (1, 2, 7):
        compare(newton_schulz(u.cuda(), steps=steps), u, True, steps=steps)
    # the cubic iteration converges: after 30 steps the rows are orthonormal
    y = newton_schulz(u.cuda(), steps=30, coefficients=(1.5, -0.5, 0.0)).double()
    assert float((y @ y.mT - torch.eye(shape[0], device="cuda", dtype=torch.float64)).abs().max()) <= 64 * 2.0 ** -22
    low = gradients(shape, seed=11, rank=2)
    low -= 0.0
    g = torch.Generator().manual_seed(1)
    low = torch.randn(shape[0], 2, generator=g) @ torch.randn(2, shape[1], generator=g)
    y = newton_schulz(low.cuda()).double().cpu()
    sv = torch.linalg.svdvals(y)
    # rank 2 stays rank 2: what fp32 left of the other directions is at most 2^-24 of the norm, times 3.4445^5
    assert float(sv[1]) > 0.6 and float(sv[0]) < 1.3 and float(sv[2]) <= 485 * 16 * 2.0 ** -24


def test_bit_equal_from_run_to_run_and_on_a_side_stream():
    from kan_sr.muon import newton_schulz
    for shape, dtype in (((2, 64, 300), torch.float32), ((500, 700), torch.float32), ((500, 700), torch.bfloat16)):
        u = gradients(shape, dtype, seed=12).cuda()
        first = newton_schulz(u)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            second = newton_schulz(u)
        third = newton_schulz(u)                      # beside it
        torch.cuda.synchronize()
        assert torch.equal(first, second) and torch.equal(first, third)


def test_many_matrices_in_one_call():
    from kan_sr.muon import newton_schulz
    u = gradients((1000, 9, 20), seed=13)
    compare(newton_schulz(u.cuda()), u, True)
    u = gradients((70, 66, 100), torch.bfloat16, seed=14)
    compare(newton_schulz(u.cuda()), u, False)


def test_large_batches_run_in_parts():
    """More matrices of a shape than the workspace holds at once."""
    from kan_sr.muon import newton_schulz
    u = gradients((12, 1, 1), seed=15).expand(12, 96, 5000) * torch.rand(12, 96, 5000, generator=torch.Generator().manual_seed(2))
    y = newton_schulz(u.cuda().repeat(12, 1, 1))       # 144 x 8 MB of workspace
    assert torch.equal(y[:12], y[-12:])
    compare(y[:2].contiguous(), u[:2], True)


def test_calls_on_two_streams_at_once():
    from kan_sr.muon import newton_schulz
    us = [gradients((900, 1000), seed=40).cuda(), gradients((2, 300, 2500), torch.bfloat16, seed=41).cuda(), gradients((20, 64, 900), seed=42).cuda()]
    want = [newton_schulz(u) for u in us]
    streams = [torch.cuda.Stream() for _ in us]
    torch.cuda.synchronize()
    got = []
    for k in range(4):
        for u, st in zip(us, streams):
            with torch.cuda.stream(st):
                got.append(newton_schulz(u))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[k % 3]) for k, y in enumerate(got))


@pytest.mark.parametrize("rows", [40, 80])
def test_offsets_beyond_32_bits(rows):
    """Rows, then matrices, so far apart that the last one lies more than 2^31 elements (and 2^32 bytes) behind the first."""
    from kan_sr.muon import newton_schulz
    u = gradients((rows, 100), torch.bfloat16, seed=43)
    want = newton_schulz(u.cuda())
    step = (1 << 31) // (rows - 1) + 8
    big = torch.empty((rows - 1) * step + 100, dtype=torch.bfloat16, device="cuda")
    far = big.as_strided((rows, 100), (step, 1))
    far.copy_(u)
    assert torch.equal(newton_schulz(far), want)
    two = big.as_strided((2, rows, 100), ((rows - 1) * step - rows * 100, 100, 1))
    two.copy_(u.expand(2, rows, 100))
    y = newton_schulz(two)
    assert torch.equal(y[0], y[1]) and torch.equal(y, newton_schulz(u.cuda().expand(2, rows, 100)))


# ------------------------------------------------------------------------------------------------ the Muon update
LIST = [(192, 64), (64, 64), (32, 64), (64, 32), (64, 64, 1, 1), (160, 64, 1, 1), (8, 4, 3, 3), (70, 200), (200, 70), (70, 200), (64, 1, 3, 3)]


def reference_update(w, g, m, lr, momentum, nesterov, wd, scale, gs):
    shape = w.shape
    w, g, m = (t.double().reshape(shape[0], -1) for t in (w, g, m))
    g = g * gs
    m = momentum * m + g
    u = g + momentum * m if nesterov else m
    w = (1 - lr * wd) * w - lr * scale * max(w.shape) ** 0.5 * exact(u)
    return w.reshape(shape), m.reshape(shape)


@pytest.mark.parametrize("nesterov", [True, False])
def test_muon_update_of_a_list(nesterov):
    from kan_sr.muon import muon_update
    g = torch.Generator().manual_seed(20)
    ws = [torch.randn(s, generator=g) * 0.1 for s in LIST]
    ms = [torch.randn(s, generator=g) * 1e-3 for s in LIST]
    W, M = [w.cuda() for w in ws], [m.cuda() for m in ms]
    kw = dict(lr=0.02, momentum=0.9, nesterov=nesterov, weight_decay=0.1, scale=0.2)
    ref = [(w.double(), m.double()) for w, m in zip(ws, ms)]
    for k in range(3):
        gs = [gradients((s[0], max(1, math.prod(s[1:]))), seed=100 * k + i).reshape(s) for i, s in enumerate(LIST)]
        muon_update(W, [t.cuda() for t in gs], M, grad_scale=0.25, **kw)
        ref = [reference_update(w, t, m, kw["lr"], kw["momentum"], nesterov, kw["weight_decay"], kw["scale"], 0.25)
               for (w, m), t in zip(ref, gs)]
        for (w, m), a, b in zip(ref, W, M):
            # momentum: two roundings a step; weight: an update 1e-5 off (the bound of the orthogonalisation) and two roundings
            assert float((b.double().cpu() - m).norm()) <= (k + 1) * 4 * 2.0 ** -24 * float(m.norm())
            step = kw["lr"] * 0.2 * max(w.shape[0], w.numel() // w.shape[0]) ** 0.5 * min(w.shape[0], w.numel() // w.shape[0]) ** 0.5 * 1.3
            assert float((a.double().cpu() - w).norm()) <= (k + 1) * (1e-5 * step + 4 * 2.0 ** -24 * float(w.norm()))


@pytest.mark.parametrize("precision,shapes", [("fp32", [(1400, 1500), (1500, 1400), (66, 4000)]),
                                              ("bf16", [(1900, 1910), (1910, 1900), (1900, 1910), (1910, 1900)])])
def test_muon_update_of_wide_matrices(precision, shapes):
    from kan_sr.muon import muon_update
    g = torch.Generator().manual_seed(26)
    gs = [gradients(s, seed=30 + i) for i, s in enumerate(shapes)]
    ws = [torch.randn(s, generator=g) * 0.1 for s in shapes]
    W, M = [w.cuda() for w in ws], [torch.zeros(s, device="cuda") for s in shapes]
    muon_update(W, [t.cuda() for t in gs], M, lr=0.02, weight_decay=0.1, precision=precision)
    for k in (0, 1):
        u = gs[k].double() * 1.95                      # of a zero momentum: m = g, U = g + 0.95 g
        ref, rate = exact(u), 0.02 * 0.2 * max(shapes[k]) ** 0.5
        # 8 x the model's error as in `compare`, and four roundings of the weight
        tol = rate * (8 * (model(u, precision == "fp32") - ref).norm() + 32 * 2.0 ** -24 * ref.norm()) + 4 * 2.0 ** -24 * ws[k].norm()
        err = W[k].double().cpu() - ((1 - 0.02 * 0.1) * ws[k].double() - rate * ref)
        assert float(err.norm()) <= float(tol), (k, float(err.norm() / tol))
        assert torch.equal(M[k].cpu(), gs[k])


@pytest.mark.parametrize("lo", [1, 2, 4])
def test_parts_of_a_flat_buffer_at_any_offset(lo):
    from kan_sr.muon import muon_update
    g = torch.Generator().manual_seed(28)
    shapes = [(192, 64), (64, 192), (90, 30), (200, 72), (72, 200), (100, 99)]
    src = [[torch.randn(s, generator=g).cuda() for s in shapes] for _ in range(2)]
    grads = [1e-3 * torch.randn(s, generator=g).cuda() for s in shapes]
    W, M = ([t.clone() for t in part] for part in src)
    muon_update(W, grads, M, lr=0.02)
    flats = []
    for part in src + [grads]:
        flat, views, off = torch.zeros(lo + sum(t.numel() + 3 for t in part), device="cuda"), [], lo
        for t in part:
            views.append(flat[off:off + t.numel()].view(t.shape).copy_(t))
            off += t.numel() + 3
        flats.append((flat, views))
    muon_update(flats[0][1], flats[2][1], flats[1][1], lr=0.02)
    assert all(torch.equal(a, b) for a, b in zip(flats[0][1] + flats[1][1], W + M))
    for flat, views in flats[:2]:                      # what lies between the parts is left as it was
        for v in views:
            v.zero_()
        assert not bool(flat.any())


def test_long_lists_are_updated_like_their_entries():
    """More entries than a launch takes: 50 small and 30 large matrices of different shapes, mixed."""
    from kan_sr.muon import muon_update
    g = torch.Generator().manual_seed(27)
    shapes = [(8 + i, 40 + 7 * i) for i in range(50)] + [(66 + 3 * i, 150 - 2 * i) for i in range(30)]
    shapes = [shapes[(37 * i) % 80] for i in range(80)]
    w0 = [torch.randn(s, generator=g).cuda() for s in shapes]
    gs = [1e-3 * torch.randn(s, generator=g).cuda() for s in shapes]
    W, M = [t.clone() for t in w0], [torch.zeros_like(t) for t in w0]
    muon_update(W, gs, M, lr=0.02, weight_decay=0.1)
    for w, grad, a, b in zip(w0, gs, W, M):
        m = torch.zeros_like(w)
        muon_update([w], [grad], [m], lr=0.02, weight_decay=0.1)
        assert torch.equal(w, a) and torch.equal(m, b), tuple(w.shape)


def test_gradient_layouts_learning_rate_on_the_device_and_repeats():
    from kan_sr.muon import muon_update
    g = torch.Generator().manual_seed(21)
    shapes = [(48, 80), (80, 48), (150, 90), (16, 8, 3, 3)]
    w0 = [torch.randn(s, generator=g).cuda() for s in shapes]
    gs = [1e-3 * torch.randn(s, generator=g).cuda() for s in shapes]

    def run(grads, **kw):
        w, m = [t.clone() for t in w0], [torch.zeros_like(t) for t in w0]
        muon_update(w, grads, m, **kw)
        return w + m

    plain = run(gs, lr=0.01)
    odd = [t.t().contiguous().t() if t.dim() == 2 else t.contiguous(memory_format=torch.channels_last) for t in gs]
    assert all(torch.equal(a, b) for a, b in zip(run(odd, lr=0.01), plain))
    assert all(torch.equal(a, b) for a, b in zip(run(gs, lr=77.0, lr_dev=torch.full((1,), 0.01, device="cuda")), plain))


def test_captured_into_a_graph_and_replayed():
    from kan_sr.muon import muon_update
    g = torch.Generator().manual_seed(22)
    shapes = [(64, 64), (160, 64), (130, 140)]
    W = [torch.randn(s, generator=g).cuda() for s in shapes]
    M = [torch.zeros(s).cuda() for s in shapes]
    G = [1e-3 * torch.randn(s, generator=g).cuda() for s in shapes]
    We, Me = [t.clone() for t in W], [t.clone() for t in M]
    scratch = [t.clone() for t in W], [t.clone() for t in M]
    muon_update(scratch[0], G, scratch[1], lr=0.01)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        muon_update(W, G, M, lr=0.01)
    for k in range(4):
        for t in G:
            t.mul_(0.7).add_(1e-4 * k)
        graph.replay()
        torch.cuda.synchronize()
        muon_update(We, G, Me, lr=0.01)                # eager work between the replays
        assert all(torch.equal(a, b) for a, b in zip(W + M, We + Me)), k


def test_optimizer_state_versions_and_checkpoint():
    from kan_sr.muon import Muon, muon_update
    g = torch.Generator().manual_seed(23)
    shapes = [(64, 64), (32, 16, 3, 3)]
    params = [torch.nn.Parameter(torch.randn(s, generator=g).cuda()) for s in shapes] + [torch.nn.Parameter(torch.zeros(3, 3).cuda())]
    opt = Muon(params, lr=0.02, weight_decay=0.01)
    copies, momenta = [p.detach().clone() for p in params[:2]], [torch.zeros_like(p) for p in params[:2]]
    for k in range(2):
        for p in params[:2]:
            p.grad = 1e-3 * torch.randn(p.shape, generator=g).cuda()
        before = [p._version for p in params]
        opt.step()
        assert [p._version > v for p, v in zip(params, before)] == [True, True, False]
        muon_update(copies, [p.grad for p in params[:2]], momenta, lr=0.02, weight_decay=0.01)
    assert all(torch.equal(a, b) for a, b in zip(params, copies))
    again = Muon(params, lr=0.5)
    again.load_state_dict(opt.state_dict())
    assert again.param_groups[0]["lr"] == 0.02
    assert all(torch.equal(again.state[p]["momentum_buffer"], m) for p, m in zip(params, momenta))
    assert params[2] not in opt.state or not opt.state[params[2]]


def test_refusals_on_the_gpu():
    from kan_sr._lib import KsrError
    from kan_sr.muon import Muon, muon_update, newton_schulz
    w = torch.randn(8, 8, device="cuda")
    bad = [lambda: newton_schulz(w[0]), lambda: newton_schulz(w.double()), lambda: newton_schulz(w, steps=0),
           lambda: newton_schulz(w, steps=33), lambda: newton_schulz(w, coefficients=(9.0, 0.0, 0.0)),
           lambda: newton_schulz(w, precision="fp16"), lambda: newton_schulz(w.clone().requires_grad_()),
           lambda: newton_schulz(w, eps=-1.0),
           lambda: muon_update([w], [w, w], [w], lr=0.1), lambda: muon_update([w[0]], [w[0]], [w[1]], lr=0.1),
           lambda: muon_update([w], [w.clone()], [w], lr=0.1), lambda: muon_update([w, w], [w, w], [w.clone(), w.clone()], lr=0.1),
           lambda: muon_update([w], [w], [w.clone()], lr=0.1),
           lambda: muon_update([w[:5], w[3:]], [w[:5].clone(), w[3:].clone()], [w[:5].clone(), w[3:].clone()], lr=0.1),
           lambda: muon_update([w.t()[:, :4]], [w[:, :4]], [w.clone()[:, :4].contiguous()], lr=0.1),
           lambda: muon_update([w], [w.bfloat16()], [w.clone()], lr=0.1), lambda: muon_update([w], [w[:4]], [w.clone()], lr=0.1),
           lambda: Muon([torch.nn.Parameter(w[0].clone())]), lambda: Muon([torch.nn.Parameter(w.clone())], lr=-1.0)]
    for k, f in enumerate(bad):
        with pytest.raises(KsrError):
            f()
            print("call", k, "was not refused")
    assert newton_schulz(w[:0]).shape == (0, 8) and newton_schulz(w[:, :0]).shape == (8, 0)
    muon_update([], [], [], lr=0.1)
