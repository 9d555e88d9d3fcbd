"""Group norm and Muon where the package uses them: the UNet hyper-encoder with norm="group", TrainStep(optimizer="muon"), and
both together, against the oracle and against the Muon iteration in 64 bits."""
from ctypes import c_float, c_int, c_int64, c_void_p

import pytest
import torch

from conftest import rel_l2
from oracle import convsepkan_oracle as orc
from test_gpu_muon import exact
from test_gpu_unet import _check_grads

pytestmark = pytest.mark.gpu


def _perturb(m):
    with torch.no_grad():
        for mod in m.modules():
            if isinstance(mod, torch.nn.GroupNorm):
                mod.weight.uniform_(0.5, 1.5)
                mod.bias.normal_(0, 0.2)


def _model(groups=2, r=2, G=5):
    from kan_sr.module import ConvSepKan
    m = ConvSepKan([1], [r * r], [3], G, 3, 0.1, [-1, 1], r, backbone="unet", norm="group", norm_groups=groups)
    _perturb(m)
    return m


@pytest.mark.parametrize("B,H,W,P,groups", [(1, 16, 16, 40, 2), (3, 48, 80, 160, 1), (2, 40, 52, 64, 4), (2, 17, 31, 40, 2), (2, 128, 96, 160, 2)])
def test_unet_group_norm_vs_oracle(B, H, W, P, groups, monkeypatch):
    from kan_sr.unet import UNet
    torch.manual_seed(B * 100 + H)
    m = UNet(1, P, norm="group", norm_groups=groups).cuda()
    _perturb(m)
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in m.state_dict().items()}
    assert not any("running" in k for k in p)
    x, gy = torch.rand(B, 1, H, W), torch.randn(B, P, H, W)
    # ReLU's slope jumps at 0.  Where the 64-bit z is closer to 0 than fp32 resolves (here 1e-5: values of size 1 that are 18
    # convolutions and norms deep, 2e-6 off), either slope is the gradient of a function that close; the oracle takes the
    # kernels' side there, and only there.  (At 3 x 48 x 80 one z of 33 000 is -5.8e-8 and its slope changes the coarse levels'
    # gradients by 1e-2; every other value agrees.)
    tape = {}
    with torch.no_grad():
        m._run(x.cuda(), True, tape)
    sides = {f"{key}.double_conv.{i}.": (t[name] > 0).permute(0, 3, 1, 2).cpu() for key, t in tape.items() if "mid" in t
             for i, name in ((1, "mid"), (4, "out"))}
    plain = orc.group_norm_relu

    def on_the_kernels_side(h, q, prefix, groups, eps=1e-5):
        shift = 1e3                                   # relu(z + shift) - shift = z: the norm without its activation
        lifted = dict(q)
        lifted[prefix + "bias"] = q[prefix + "bias"] + shift
        z = plain(h, lifted, prefix, groups, eps) - shift
        side = sides[prefix]
        assert bool((z.detach().abs()[side != (z > 0)] <= 1e-5).all()), prefix
        return z * side

    rows, plain_rows = [], orc._l2_rows

    def recorded_rows(t, eps=1e-12):
        out = plain_rows(t, eps)
        out.retain_grad()
        rows.append((t.detach(), out))
        return out

    monkeypatch.setattr(orc, "group_norm_relu", on_the_kernels_side)
    monkeypatch.setattr(orc, "_l2_rows", recorded_rows)
    ref = orc.unet(x.double(), p, groups=groups)
    (ref * gy.double()).sum().backward()
    y = m.train()(x.cuda())
    # the tolerances of the BatchNorm form's tests
    assert bool(((y.detach().cpu() - ref.detach()).abs() <= 2e-5 + 1e-4 * ref.detach().abs()).all())
    y.backward(gy.cuda())
    rel = 1e-4 if (H // 16) * (W // 16) >= 16 else 1e-3
    # Where a row that is normalised is one pixel long (att4 at 16 x 16), q / |q| = +-1 has derivative 0: (u - q^ (q^ u)) / |q|
    # with q^ q^ = 1.  fp32 has q^ q^ within 2^-23 of 1, so up to 4 half steps of u / |q| remain, times what the weight's
    # gradient multiplies them with: the input, and for the two convolutions of `a` the other's weight, over 32 channels.
    left = max([float((out.grad.abs() / t.abs()).max()) for t, out in rows if t.shape[-1] == 1], default=0.0)
    x_max = float(max(t["out"].abs().max() for t in tape.values() if "mid" in t))
    zero = {n for n, q in p.items() if float(q.grad.norm()) < 1e-6 * max(1.0, q.numel() ** 0.5)}
    for n, q in m.named_parameters():
        if n in zero:
            assert n.startswith("att") and float(q.grad.abs().max()) <= max(1e-5, 4 * 2.0 ** -24 * left * x_max * 32 * B), n
    _check_grads({n: q.grad for n, q in m.named_parameters() if n not in zero}, {n: q.grad for n, q in p.items()}, rel=rel)
    with torch.no_grad():
        assert torch.equal(m.eval()(x.cuda()), y.detach())            # no running statistics: both modes are the same function
        one = m(x[:1].cuda())
    assert bool(((one.cpu() - ref[:1].detach()).abs() <= 2e-5 + 1e-4 * ref[:1].detach().abs()).all())    # images do not mix


def test_input_gradient_of_the_group_norm_model():
    torch.manual_seed(5)
    m = _model().cuda()
    p = {k: v.detach().cpu().double() for k, v in m.state_dict().items()}
    x = torch.rand(2, 3, 32, 48)
    xr = x.double().requires_grad_()
    ref = orc.conv_sep_kan_forward(xr, p, out_channels=[4], grid_size=5, spline_order=3, grid_range=[-1, 1], upscale=2, backbone="unet", norm_groups=2)
    gy = torch.randn(ref.shape)
    (ref * gy.double()).sum().backward()
    xg = x.cuda().requires_grad_()
    m(xg).backward(gy.cuda())
    assert rel_l2(xg.grad.cpu(), xr.grad) <= 1e-3


def test_adam_step_runs_is_adam_on_the_runs():
    from kan_sr._lib import check, lib, ptr, stream
    from kan_sr.train import flat_runs
    torch.manual_seed(1)
    n = 5000
    base = [torch.randn(n).cuda(), torch.randn(n).cuda(), torch.randn(n).cuda() * 0.1, torch.rand(n).cuda()]
    a, b = [t.clone() for t in base], [t.clone() for t in base]
    args = (c_float(1e-2), c_float(0.9), c_float(0.99), c_float(1e-8), c_float(0.1))
    check(lib().ksr_adam_step(*(ptr(t) for t in a), c_int64(n), *args, c_int(3), c_float(0.5), stream()), "adam")
    parts = [(0, 10), (10, 300), (400, 0), (700, 4000)] + [(4700 + 2 * k, 1) for k in range(140)]
    runs = flat_runs(parts)
    covered = torch.zeros(n, dtype=torch.bool)
    for o, k in parts:
        covered[o:o + k] = True
    assert sum(runs[1::2]) == int(covered.sum()) and len(runs) // 2 <= 143

    def step(t, lr, lr_dev, k, k_dev):
        check(lib().ksr_adam_step_runs(*(ptr(q) for q in t), runs, c_int(len(runs) // 2), c_float(lr), lr_dev, *args[1:], c_int(k),
                                       k_dev, c_float(0.5), stream()), "adam_runs")

    step(b, 1e-2, None, 3, None)
    c = covered.cuda()
    for got, want, old in zip(b, a, base):
        assert torch.equal(got[c], want[c]) and torch.equal(got[~c], old[~c])
    d = [t.clone() for t in base]
    lr_dev, k_dev = torch.full((1,), 1e-2, device="cuda"), torch.full((1,), 3, device="cuda", dtype=torch.int64)
    step(d, 9.0, ptr(lr_dev), 77, c_void_p(k_dev.data_ptr()))
    assert all(bool(((x - y).abs() <= 1e-6 * (1 + y.abs())).all()) for x, y in zip(d, b))


class _Reference:
    """torch.optim.Adam on the CPU in 64 bits for the vectors, the Muon update in 64 bits for the matrices."""

    def __init__(self, p, muon_names, lr, momentum=0.95):
        self.p = {n: v.double().requires_grad_() for n, v in p.items()}
        self.names, self.lr, self.mu = set(muon_names), lr, momentum
        self.adam = torch.optim.Adam([v for n, v in self.p.items() if n not in self.names], lr=lr)
        self.mom = {n: torch.zeros_like(self.p[n]) for n in self.names}

    def step(self, grads):
        for n, v in self.p.items():
            v.grad = grads[n].double().cpu()
        self.adam.step()
        with torch.no_grad():
            for n in self.names:
                g = self.p[n].grad
                self.mom[n] = self.mu * self.mom[n] + g
                u = (g + self.mu * self.mom[n]).reshape(g.shape[0], -1)
                self.p[n] -= exact(u).reshape(g.shape) * (self.lr * 0.2 * max(u.shape) ** 0.5)


@pytest.mark.parametrize("backbone", ["gazetr", "unet"])
def test_train_step_with_muon_vs_oracle(backbone):
    """Loss of every step against the oracle at the step's parameters; the parameters after every step against the updates in 64
    bits from the step's own gradients (held to the oracle elsewhere).  Adam and Newton-Schulz both enlarge what little a
    gradient that ought to be zero holds, so whole trajectories of two gradient computations say nothing."""
    from kan_sr.module import ConvSepKan
    from kan_sr.train import TrainStep
    torch.manual_seed(3)
    unet = backbone == "unet"
    m = _model() if unet else ConvSepKan([1], [4], [3], 5, 3, 0.1, [-1, 1], 2).eval()
    p0 = {n: v.detach().clone() for n, v in m.state_dict().items()}
    ts = TrainStep(m.cuda(), lr=1e-3, loss="l1+ssim", optimizer="muon")
    assert len(ts.muon_names) >= 8 and all(min(m.get_parameter(n).shape[0], m.get_parameter(n)[0].numel()) >= 16 for n in ts.muon_names)
    assert not any(k in n for n in ts.muon_names for k in ("feed", "reproj", "bias", "depthwise", "gate"))
    ref = _Reference(p0, ts.muon_names, 1e-3)
    for it in range(3):
        x, tgt = torch.rand(2, 3, 32, 48), torch.rand(2, 3, 64, 96)
        now = {n: v.detach().cpu() for n, v in m.state_dict().items()}
        y = orc.conv_sep_kan_forward(x, now, out_channels=[4], grid_size=5, spline_order=3, grid_range=[-1, 1], upscale=2,
                                     backbone=backbone, norm_groups=2 if unet else 0)
        loss = float(orc.training_loss(y, tgt))
        assert abs(float(ts.step(x.cuda(), tgt.cuda())) - loss) <= 1e-5 + 1e-4 * abs(loss)
        ref.step(ts.arena)
        for n, prm in m.named_parameters():
            # per step: an update 1e-5 off (the bound of the orthogonalisation; Adam's is smaller) and two roundings of the result
            want, have = ref.p[n].detach(), prm.detach().double().cpu()
            moved = float((want - p0[n].double()).norm())
            assert float((have - want).norm()) <= 2e-5 * moved + (it + 1) * 2.0 ** -23 * float(want.norm()), (it, n)


@pytest.mark.parametrize("backbone", ["gazetr", "unet"])
def test_captured_muon_step_equals_launched_step(backbone):
    """Together: the group-norm UNet (or GazeTR) trained by Muon, replayed from a graph and launched, with a change of the
    learning rate and of the input shape in between: bit-equal."""
    from kan_sr.module import ConvSepKan
    from kan_sr.train import TrainStep
    runs = []
    for capture in (False, True):
        torch.manual_seed(33)
        m = (_model() if backbone == "unet" else ConvSepKan([1], [4], [3], 5, 3, 0.1, [-1, 1], 2).eval()).cuda()
        ts = TrainStep(m, lr=1e-3, loss="l1+ssim", capture=capture, optimizer="muon", device_state=backbone == "gazetr" or None)
        gen = torch.Generator().manual_seed(7)
        losses = []
        for it in range(9):
            h, w = (32, 48) if it < 5 else (40, 36)
            if it == 4:
                ts.set_epoch(100)
            x, tgt = torch.rand(2, 3, h, w, generator=gen).cuda(), torch.rand(2, 3, 2 * h, 2 * w, generator=gen).cuda()
            losses.append(float(ts.step(x, tgt)))
        if capture:
            assert ts._graph is not None
        runs.append((losses, ts.flat_p.clone(), ts.exp_avg.clone()))
    assert runs[0][0] == runs[1][0] and torch.equal(runs[0][1], runs[1][1]) and torch.equal(runs[0][2], runs[1][2])


def test_recorded_while_an_eager_graph_of_the_parameters_lives():
    from kan_sr.train import TrainStep
    runs = []
    for keep in (False, True):
        torch.manual_seed(35)
        m = _model().cuda()
        gen = torch.Generator().manual_seed(9)
        x0 = torch.rand(2, 3, 32, 32, generator=gen).cuda()
        alive = m(x0) if keep else None
        ts = TrainStep(m, lr=1e-3, optimizer="muon", capture=True)
        for it in range(5):
            ts.step(torch.rand(2, 3, 32, 32, generator=gen).cuda(), torch.rand(2, 3, 64, 64, generator=gen).cuda())
        assert ts._graph is not None and (alive is None or alive.requires_grad)
        runs.append((ts.flat_p.clone(), ts.exp_avg.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


def test_changed_momentum_is_not_replayed_from_an_old_graph():
    from kan_sr.module import ConvSepKan
    from kan_sr.train import TrainStep
    runs = []
    for capture in (False, True):
        torch.manual_seed(34)
        m = ConvSepKan([1], [4], [3], 5, 3, 0.1, [-1, 1], 2).eval().cuda()
        ts = TrainStep(m, lr=1e-3, optimizer="muon", capture=capture, device_state=True)
        gen = torch.Generator().manual_seed(8)
        for it in range(8):
            if it == 4:
                ts.muon_momentum, ts.betas = 0.5, (0.8, 0.99)
            ts.step(torch.rand(2, 3, 32, 32, generator=gen).cuda(), torch.rand(2, 3, 64, 64, generator=gen).cuda())
        runs.append((ts.flat_p.clone(), ts.exp_avg.clone()))
    assert torch.equal(runs[0][0], runs[1][0]) and torch.equal(runs[0][1], runs[1][1])


def test_muon_checkpoint_resumes_and_does_not_mix_with_adam(tmp_path):
    from kan_sr._lib import KsrError
    from kan_sr.checkpoint import load_checkpoint, save_checkpoint
    from kan_sr.train import TrainStep
    torch.manual_seed(11)
    xs, tg = [torch.rand(2, 3, 32, 32).cuda() for _ in range(4)], [torch.rand(2, 3, 64, 64).cuda() for _ in range(4)]
    m = _model().cuda()
    ts = TrainStep(m, lr=1e-3, optimizer="muon", muon_momentum=0.8)
    for it in range(3):
        ts.step(xs[it], tg[it])
    path = str(tmp_path / "last.ckpt")
    save_checkpoint(m, path, epoch=3, global_step=3, train_step=ts)
    m2 = _model().cuda()
    ts2 = TrainStep(m2, lr=5.0, optimizer="muon")
    load_checkpoint(m2, path, train_step=ts2)
    assert ts2.muon_momentum == 0.8
    a, b = float(ts.step(xs[3], tg[3])), float(ts2.step(xs[3], tg[3]))
    assert a == b and torch.equal(ts.flat_p, ts2.flat_p) and torch.equal(ts.exp_avg, ts2.exp_avg)
    m3 = _model().cuda()
    with pytest.raises(KsrError, match="Muon"):
        load_checkpoint(m3, path, train_step=TrainStep(m3, lr=1e-3))
    save_checkpoint(m3, path, train_step=TrainStep(m3, lr=1e-3))
    with pytest.raises(KsrError, match="Muon"):
        load_checkpoint(m2, path, train_step=ts2)


def test_muon_optimizer_on_the_autograd_path_keeps_the_unets_weights_fresh():
    """torch-style training of the module: the kernel-layout weight copies of the UNet follow updates written by the kernels."""
    from kan_sr.muon import Muon
    from kan_sr.train import takes_muon
    torch.manual_seed(4)
    m = _model().cuda()
    enc = m.layers[-1].encoder.encoder
    params = [p for n, p in enc.named_parameters() if takes_muon(n, p.shape)]
    opt = Muon(params, lr=0.05)
    x = torch.rand(2, 3, 32, 32).cuda()
    for _ in range(2):
        opt.zero_grad()
        m(x)[:, :1].square().mean().backward()
        opt.step()
        with torch.no_grad():
            y = m(x)
            enc.invalidate_prepared()
            assert torch.equal(m(x), y)


def test_refusals():
    from kan_sr._lib import KsrError
    from kan_sr.module import ConvSepKan
    from kan_sr.train import TrainStep
    from kan_sr.unet import UNet
    m = _model().cuda()
    for bad in (lambda: TrainStep(m, optimizer="sgd"), lambda: TrainStep(m, optimizer="muon", muon_params=lambda n, s: False),
                lambda: TrainStep(m, optimizer="muon", muon_momentum=1.0), lambda: UNet(1, 40, norm="layer"),
                lambda: UNet(1, 40, norm="group", norm_groups=3),
                lambda: ConvSepKan([1], [4], [3], 5, 3, 0.1, [-1, 1], 2, norm="group")):
        with pytest.raises(KsrError):
            bad()
