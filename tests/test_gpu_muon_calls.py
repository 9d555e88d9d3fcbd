"""What else a call holds makes no difference to a matrix; calls of the largest sizes, traces and forward mode (kan_sr.muon)."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def randn(*shape, seed=1):
    return torch.randn(*shape, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))


# alone these run in tiles of 64, or with tiles cut along k; in the batch in tiles of 128 (256), whole and cut ones beside each other
BATCHES = [((777, 2051), 5), ((1536, 1536), 3), ((1500, 1400), 6), ((2100, 2100), 2), ((600, 3000), 12), ((1900, 1910), 4), ((130, 5000), 9)]


@pytest.mark.parametrize("shape,n", BATCHES)
def test_fp32_results_do_not_depend_on_the_rest_of_a_batch(shape, n):
    from kan_sr.muon import newton_schulz
    u = randn(*shape)
    alone = newton_schulz(u)
    y = newton_schulz(u.expand(n, *shape))
    assert all(torch.equal(y[k], alone) for k in range(n))


@pytest.mark.parametrize("shape,n", BATCHES)
def test_bf16_results_do_not_depend_on_the_rest_of_a_batch(shape, n):
    """Sums of single operands end in the same bits however the tiles are cut and whatever their size."""
    from kan_sr.muon import newton_schulz
    u = randn(*shape).bfloat16()
    alone = newton_schulz(u)
    y = newton_schulz(u.expand(n, *shape))
    assert all(torch.equal(y[k], alone) for k in range(n))


@pytest.mark.parametrize("precision", ["fp32", "bf16"])
def test_lists_of_large_matrices_are_updated_like_their_entries(precision):
    from kan_sr.muon import muon_update
    shapes = [(777, 2051), (1536, 1536), (100, 600), (1500, 1400), (300, 3000), (1536, 1536), (900, 70), (2051, 777)]
    w0, gs = [randn(*s, seed=k) for k, s in enumerate(shapes)], [1e-3 * randn(*s, seed=50 + k) for k, s in enumerate(shapes)]
    W, M = [t.clone() for t in w0], [torch.zeros_like(t) for t in w0]
    muon_update(W, gs, M, lr=0.02, precision=precision)
    for w, g, a, b in zip(w0, gs, W, M):
        m = torch.zeros_like(w)
        muon_update([w], [g], [m], lr=0.02, precision=precision)
        assert torch.equal(w, a) and torch.equal(m, b), tuple(w.shape)


def test_more_small_matrices_than_one_launch_holds():
    """2^22 workgroups of 512 threads run together, the rest of the batch in the next launches."""
    from kan_sr.muon import newton_schulz
    n = (1 << 23) + 3                                  # of 2^32 threads and more a launch is invalid
    u = randn(n, 1, 2)
    y = newton_schulz(u, steps=1)
    x = u.double() / (u.double().norm(dim=(1, 2), keepdim=True) + 1e-7)
    a, b, c = 3.4445, -4.7750, 2.0315
    A = x.square().sum(dim=2, keepdim=True)
    ref = (a + b * A + c * A * A) * x
    # operands of 22 bits: three products of a few units of 2^-22 each, of values of at most 3.4445 + 4.775 + 2.0315
    assert float((y.double() - ref).abs().max()) <= 4 * (a - b + c) * 2.0 ** -22
    for k in (0, (1 << 22) - 1, 1 << 22, n - 1):
        assert torch.equal(newton_schulz(u[k], steps=1), y[k])


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("shape", [(24, 40), (3, 100, 140)])
def test_traced_calls_run_the_kernels(shape):
    from kan_sr.muon import newton_schulz
    traced = torch.jit.trace(lambda t: newton_schulz(t), (randn(*shape),))
    for k in range(2):
        u = randn(*shape, seed=10 + k)
        assert torch.equal(traced(u), newton_schulz(u))


@pytest.mark.filterwarnings("ignore")
def test_forward_mode_and_traced_updates_are_refused_not_dropped():
    from torch.autograd import forward_ad
    from kan_sr._lib import KsrError
    from kan_sr.muon import muon_update, newton_schulz
    a, b, c = (randn(24, 40, seed=k) for k in range(3))
    before = [t.clone() for t in (a, b, c)]
    with forward_ad.dual_level():
        assert torch.equal(newton_schulz(a), newton_schulz(a.clone()))              # nothing dual: an ordinary call
        dual = forward_ad.make_dual(a, torch.ones_like(a))
        for grad in (False, True):
            with torch.set_grad_enabled(grad):
                with pytest.raises(KsrError, match="differentiable"):
                    newton_schulz(dual)
        for args in ((dual, b, c), (b, dual, c), (b, c, dual)):
            with pytest.raises(KsrError, match="differentiated"):
                muon_update(*([t] for t in args), lr=0.1)

    def update(t):
        muon_update([a], [t], [c], lr=0.1)
        return a + t

    with pytest.raises(KsrError, match="traced"):
        torch.jit.trace(update, (b,))
    assert all(torch.equal(t, u) for t, u in zip((a, b, c), before))


def test_gradients_that_overlap_what_is_written_are_refused():
    """The matrices of a call run side by side: one's weight may be written while another still reads it as its gradient."""
    from kan_sr._lib import KsrError
    from kan_sr.muon import muon_update
    a, b, m, n = (randn(8, 8, seed=k) for k in range(4))
    buf = randn(200, seed=9)
    w, far = buf[8:72].view(8, 8), buf[120:184].view(8, 8)
    before = [t.clone() for t in (a, b, m, n, buf)]
    for ws, gs, ms in (([a, b], [b, a], [m, n]),                                   # crossed
                       ([a, b], [randn(8, 8), m], [m, n]),                         # another entry's momentum
                       ([w], [buf[0:64].view(8, 8)], [m]), ([w], [buf[71:135].view(8, 8)], [m]),        # partly its own weight
                       ([a], [buf[60:124].view(8, 8)], [far]),                     # partly its own momentum
                       ([w], [buf[:160:20].expand(8, 8)], [m]), ([w], [buf[:64].view(8, 8).t()], [m]),  # by its strides
                       ([buf[8:72].view(4, 16)], [buf[72:136].view(4, 16)], [buf[135:199].view(4, 16)])):
        with pytest.raises(KsrError, match="overlap"):
            muon_update(ws, gs, ms, lr=0.1)
    assert all(torch.equal(t, u) for t, u in zip((a, b, m, n, buf), before))
    # neighbours in one buffer, and gradients that share memory, are fine
    g = randn(8, 8, seed=10)
    muon_update([w], [buf[72:136].view(8, 8)], [buf[136:200].view(8, 8)], lr=0.1)
    muon_update([a, b], [g, g.t()], [m, n], lr=0.1)
    muon_update([b], [g[:1].expand(8, 8)], [n], lr=0.1)


def test_tensors_made_in_inference_mode():
    """They have no version counter to bump: the update of all, and the counters of the others, are as ever."""
    from kan_sr.muon import muon_update
    g = [1e-3 * randn(24, 40, seed=2), 1e-3 * randn(70, 30, seed=3)]
    with torch.inference_mode():
        w = [randn(24, 40)]
    w.append(randn(70, 30))
    m = [torch.zeros(24, 40, device="cuda"), torch.zeros(70, 30, device="cuda")]
    copies = [t.clone() for t in w], [t.clone() for t in m]
    before = [t._version for t in (w[1], *m)]
    muon_update(w, g, m, lr=0.1)
    assert all(t._version > v for t, v in zip((w[1], *m), before))
    muon_update(copies[0], g, copies[1], lr=0.1)
    assert all(torch.equal(a, b) for a, b in zip(w + m, copies[0] + copies[1]))
