"""Group norm + activation (kan_sr.ops.group_norm_act) in calls of the largest numbers of groups, traces, forward mode, streams."""
import pytest
import torch

from test_gpu_group_norm import U32, formula, z_error

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B,S,C,G", [((1 << 21) + 3, 2, 32, 8),            # 2^24 + 24 workgroups of 256 threads in one pass
                                     ((1 << 20) + 1, 1, 64, 32)])          # a pixel per image: group norm per token, 2^25 groups
def test_more_groups_than_one_launch_holds(B, S, C, G):
    """2^32 threads are more than a launch takes: the images go in ranges."""
    from kan_sr.ops import group_norm_act
    g = torch.Generator("cuda").manual_seed(B)
    x = torch.randn(B, S, C, device="cuda", generator=g)
    w, b = 1 + 0.3 * torch.randn(C, device="cuda", generator=g), 0.3 * torch.randn(C, device="cuda", generator=g)
    dy = torch.randn(B, S, C, device="cuda", generator=g)
    args = [t.clone().requires_grad_() for t in (x, w, b)]
    y = group_norm_act(args[0], G, args[1], args[2], activation="silu")
    dx, dw, db = torch.autograd.grad(y, args, dy)
    # the first, the last and the images around the borders of ranges
    some = torch.cat([torch.arange(k, k + 40) for k in (0, B // 4 - 20, B // 3 - 20, B // 2 - 20, 2 * B // 3 - 20, 3 * B // 4 - 20, B - 40)]).cuda()
    x64, w64, b64 = x[some].double().requires_grad_(), w.double().requires_grad_(), b.double().requires_grad_()
    y64, xhat, z, mean, rstd = formula(x64, w64, b64, G, 1e-5, "silu")
    y64.backward(dy[some].double())
    with torch.no_grad():
        ez = z_error(x64, w64, b64, xhat, z, mean, rstd)
        assert bool(((y[some].double() - y64).abs() <= 1.2 * ez + 16 * U32 * (z.abs() + 1)).all())
        # dx: three terms of dz and xhat, each with ez and a few dozen roundings of values of at most |w dz| (1 + |xhat|) rstd
        size = rstd * (1 + xhat.abs()) ** 2 * (w64.abs().max() + 1) * dy[some].double().abs().amax(dim=(1, 2), keepdim=True)
        assert bool(((dx[some].double() - x64.grad).abs() <= size * (4 * ez.amax(dim=(1, 2), keepdim=True) + 256 * U32)).all())
        # dw, db: of all images, in 64 bits part by part; at most B S / 4 + 64 roundings of the sums of absolute values
        ref, total = torch.zeros(2, C, dtype=torch.float64, device="cuda"), torch.zeros(2, C, dtype=torch.float64, device="cuda")
        for lo in range(0, B, 1 << 18):
            p, d = x[lo:lo + (1 << 18)].double(), dy[lo:lo + (1 << 18)].double()
            _, xh, zz, _, _ = formula(p, w.double(), b.double(), G, 1e-5, "silu")
            s = torch.sigmoid(zz)
            dz = d * s * (1 + zz * (1 - s))
            for k, t in enumerate((dz, dz * xh)):
                ref[k] += t.sum(dim=(0, 1))
                total[k] += t.abs().sum(dim=(0, 1))
        tol = (B * S / 4 + 64) * U32 * total + 64 * U32 * total
        assert bool(((torch.stack([db, dw]).double() - ref).abs() <= tol).all())


@pytest.mark.filterwarnings("ignore")
def test_traced_calls_run_the_kernels():
    from kan_sr.ops import group_norm_act
    x = torch.randn(2, 30, 16, device="cuda")
    w, b = torch.randn(16, device="cuda"), torch.randn(16, device="cuda")
    for grad in (False, True):
        with torch.set_grad_enabled(grad):
            traced = torch.jit.trace(lambda t: group_norm_act(t, 4, w, b, activation="silu"), (x,))
            for k in range(2):
                u = torch.randn(2, 30, 16, device="cuda")
                assert torch.equal(traced(u), group_norm_act(u, 4, w, b, activation="silu"))


@pytest.mark.parametrize("which", [0, 1, 2])
def test_forward_mode_is_refused_not_dropped(which):
    from torch.autograd import forward_ad
    from kan_sr.ops import group_norm_act
    args = [torch.randn(2, 30, 16, device="cuda"), torch.randn(16, device="cuda"), torch.randn(16, device="cuda")]
    plain = group_norm_act(args[0], 4, *args[1:])
    for grad in (False, True):
        with torch.set_grad_enabled(grad), forward_ad.dual_level():
            assert torch.equal(group_norm_act(args[0], 4, *args[1:]), plain)          # nothing dual: an ordinary call
            dual = list(args)
            dual[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
            with pytest.raises((RuntimeError, NotImplementedError)):
                group_norm_act(dual[0], 4, *dual[1:])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("shape,G", [((3, 200, 16), 4), ((2, 300, 24), 6), ((2, 60, 60, 90), 9), ((1, 130, 127, 320), 32), ((2, 400, 8), 4)])
def test_relu_has_one_mask(shape, G, dtype):
    """Values at the edge: every channel's bias is -w xhat of the values that half of its elements have, so that z is what rounding
    leaves.  The gradient of the bias counts the positive results, exactly (dy = 1, fewer than 2^24 of them)."""
    from kan_sr.ops import group_norm_act
    g = torch.Generator().manual_seed(7)
    C = shape[-1]
    x = torch.randn(shape, generator=g)
    level = torch.randn(C, generator=g)
    x = torch.where(torch.rand(shape, generator=g) < 0.5, level.expand(shape), x).to(dtype)
    w = 1 + 0.3 * torch.randn(C, generator=g)
    _, xhat, _, _, _ = formula(x.double(), torch.ones(C, dtype=torch.float64), torch.zeros(C, dtype=torch.float64), G, 1e-5, "none")
    edge = xhat[0].reshape(-1, C)[(x[0] == level.to(dtype)).reshape(-1, C).int().argmax(dim=0), torch.arange(C)]
    b = (-(w.double() * edge)).float()
    x, w, b = x.cuda().requires_grad_(), w.cuda().requires_grad_(), b.cuda().requires_grad_()
    y = group_norm_act(x, G, w, b, activation="relu")
    assert float((y.detach().float().reshape(-1, C)[(x.detach() == level.to(dtype).cuda()).reshape(-1, C).any(dim=1)]).min()) == 0.0
    db, = torch.autograd.grad(y, (b,), torch.ones_like(y))
    assert torch.equal(db, (y > 0).reshape(-1, C).sum(dim=0).float())


def test_calls_that_overlap_on_three_streams():
    """Forward and backward of several hundred microseconds each, queued behind one event and then let go together: a workspace that
    two calls shared would mix their sums."""
    from kan_sr.ops import group_norm_act
    args = []
    for k, (shape, G, dtype) in enumerate([((3, 256, 256, 320), 32, torch.bfloat16), ((4, 300, 300, 90), 9, torch.float32),
                                           ((24, 128, 128, 256), 32, torch.float32)]):
        g = torch.Generator("cuda").manual_seed(k)
        x, dy = ((torch.randn(shape, device="cuda", generator=g) + k).to(dtype) for _ in range(2))
        w, b = (torch.randn(shape[-1], device="cuda", generator=g) for _ in range(2))
        args.append((x.requires_grad_(), w.requires_grad_(), b.requires_grad_(), dy, G))

    def run(x, w, b, dy, G):
        y = group_norm_act(x, G, w, b, activation="silu")
        return (y.detach(),) + torch.autograd.grad(y, (x, w, b), dy)

    want = [run(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    gate, go = torch.randn(8192, 8192, device="cuda"), torch.cuda.Event()
    torch.cuda.synchronize()
    got = []
    for _ in range(6):                                  # about 50 ms, while the calls are queued
        gate = gate @ gate * 1e-2
    go.record()
    for st in streams:
        st.wait_event(go)
    for k in range(4):
        for a, st in zip(args, streams):
            with torch.cuda.stream(st):
                got.append(run(*a))
    torch.cuda.synchronize()
    for k, out in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(out, want[k % 3])), k


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_saved_tensors_that_come_back_with_other_strides(dtype):
    """save_on_cpu stores a channel slice densely: its strides of the forward would reach beyond it in the backward."""
    from kan_sr.ops import group_norm_act
    big = torch.randn(2, 30, 20, 64, device="cuda").to(dtype)
    dy = torch.randn(2, 30, 20, 24, device="cuda").to(dtype)
    w, b = torch.randn(24, device="cuda", requires_grad=True), torch.randn(24, device="cuda", requires_grad=True)
    for x in (big[..., 8:32], big[..., 3:27], big[:1, :1, :1, :24].expand(2, 30, 20, 24)):
        x = x.detach().requires_grad_()
        want = torch.autograd.grad(group_norm_act(x, 4, w, b, activation="gelu"), (x, w, b), dy)
        with torch.autograd.graph.save_on_cpu():
            y = group_norm_act(x, 4, w, b, activation="gelu")
        for p, q in zip(torch.autograd.grad(y, (x, w, b), dy), want):
            # other vectors, another order of the sums: at most 64 roundings of each of two terms of the largest gradient's size; a
            # bfloat16 result may end one step away
            tol = 128 * U32 * q.abs().max() + (torch.finfo(dtype).eps * q.abs() if q.dtype is torch.bfloat16 else 0)
            assert bool(((p - q).abs() <= tol).all())
