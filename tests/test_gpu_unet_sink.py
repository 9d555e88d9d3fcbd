"""The UNet's gradients when its gradient sink changes between forward and backward."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("norm", ["batch", "group"])
def test_a_sink_that_is_gone_is_an_error_not_a_lost_gradient(norm):
    from kan_sr._lib import KsrError
    from kan_sr.unet import UNet
    torch.manual_seed(3)
    net = UNet(1, 40, norm=norm).cuda()
    x, gy = torch.rand(2, 1, 32, 48, device="cuda"), torch.randn(2, 40, 32, 48, device="cuda")
    net(x).backward(gy)
    want = {n: p.grad.clone() for n, p in net.named_parameters()}
    net.zero_grad(set_to_none=True)
    sink = {n: torch.zeros_like(p) for n, p in net.named_parameters()}

    def into_the_sink():
        net.grad_sink = sink
        net(x).backward(gy)
        assert all(p.grad is None for p in net.parameters()) and all(torch.equal(sink[n], w) for n, w in want.items())

    into_the_sink()
    y = net(x)
    net.grad_sink = None                                # recorded with it, gone at the backward
    with pytest.raises(KsrError, match="grad_sink"):
        y.backward(gy)
    assert all(p.grad is None for p in net.parameters())
    del y
    net(x).backward(gy)                                 # recorded without: the parameters have their gradients again
    assert all(torch.equal(p.grad, want[n]) for n, p in net.named_parameters())
    net.zero_grad(set_to_none=True)
    for t in sink.values():
        t.zero_()
    into_the_sink()
