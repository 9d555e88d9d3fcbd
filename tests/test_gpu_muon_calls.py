"""What else a call holds makes no difference to a matrix, and calls of the largest sizes (kan_sr.muon)."""
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
