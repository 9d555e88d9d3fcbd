"""Adam over runs (ksr_adam_step_runs) of the greatest length."""
from ctypes import c_float, c_int, c_int64

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_run_of_almost_two_to_the_31_elements():
    from kan_sr._lib import check, lib, ptr, stream
    first, n, tail = 3, (1 << 31) - 1, 70000            # the last steps of the threads pass 2^31
    total = first + n + tail
    p, g, m, v = (torch.full((total,), value, device="cuda") for value in (2.0, 0.5, 0.0, 0.0))
    args = (c_float(0.1), None, c_float(0.9), c_float(0.99), c_float(1e-8), c_float(0.0), c_int(1), None, c_float(1.0), stream())
    small = [torch.full((5,), value, device="cuda") for value in (2.0, 0.5, 0.0, 0.0)]
    check(lib().ksr_adam_step_runs(*(ptr(t) for t in small), (c_int64 * 2)(0, 5), c_int(1), *args), "adam_runs")
    check(lib().ksr_adam_step_runs(ptr(p), ptr(g), ptr(m), ptr(v), (c_int64 * 2)(first, n), c_int(1), *args), "adam_runs")
    for t, want, old in zip((p, m, v), (small[0], small[2], small[3]), (2.0, 0.0, 0.0)):
        assert float(t[first:first + n].min()) == float(want[0]) == float(t[first:first + n].max()) != old
        assert bool((t[:first] == old).all()) and bool((t[first + n:] == old).all())
