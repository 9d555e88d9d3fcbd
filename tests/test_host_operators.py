"""CPU tests of the operators' refusals: every call below ends before anything is launched."""
import ctypes
from ctypes import c_float, c_int, c_int64, c_void_p

import pytest
import torch


def test_group_norm_refuses_what_it_cannot_take():
    from kan_sr._lib import KsrError
    from kan_sr.ops import group_norm_act
    x = torch.randn(2, 3, 3, 8)
    for bad in (lambda: group_norm_act(x, 2),                                     # CPU tensor
                lambda: group_norm_act(x, 2, activation="tanh"),
                lambda: group_norm_act(torch.randn(8), 2)):
        with pytest.raises(KsrError):
            bad()


def test_group_norm_refuses_at_the_abi():
    from kan_sr import _lib
    L = _lib.lib()
    fake = c_void_p(1 << 20)                    # never read: the argument checks come first

    def fwd(x=fake, B=2, S=9, C=8, G=2, eps=1e-5, act=0, stride=8, ws=fake):
        return L.ksr_group_norm_fwd(x, c_int64(72), c_int64(stride), None, None, fake, fake, ws, c_int64(B), c_int64(S), c_int(C),
                                    c_int(G), c_float(eps), c_int(act), c_int(0), None)

    assert fwd(x=None) == -1 and b"null pointer" in L.ksr_last_error()
    assert fwd(ws=None) == -1 and fwd(C=9) == -1 and fwd(G=0) == -1 and fwd(B=-1) == -1 and fwd(S=-1) == -1
    assert fwd(act=4) == -1 and b"activation" in L.ksr_last_error()
    assert fwd(eps=float("nan")) == -1 and fwd(stride=-8) == -1
    assert fwd(x=c_void_p((1 << 20) + 2)) == -1 and b"misaligned" in L.ksr_last_error()
    assert fwd(B=1 << 40) == -2
    assert fwd(B=0) == 0 and fwd(S=0) == 0       # nothing to do
    assert L.ksr_group_norm_ws_floats(c_int64(2), c_int64(9), c_int(8), c_int(3), c_int(0)) == -1
    assert L.ksr_group_norm_ws_floats(c_int64(0), c_int64(9), c_int(8), c_int(2), c_int(0)) == 0


@pytest.mark.parametrize("shape,stride,want", [
    ((2, 3, 5, 8), None, (120, 8)), ((1, 8), None, (0, 0)), ((4, 8), None, (8, 0)), ((2, 1, 5, 8), None, (40, 8)),
    ((2, 3, 5, 8), (15 * 20, 5 * 20, 20, 1), (300, 20)),           # a channel slice
    ((2, 3, 5, 8), (0, 0, 0, 1), (0, 0)),                          # expanded pixels
    ((2, 3, 5, 1), (15 * 4, 20, 4, 7), (60, 4)),                   # one channel: its stride says nothing
    ((2, 3, 5, 8), (200, 48, 8, 1), None), ((2, 3, 5, 8), (120, 1, 3, 15), None)])
def test_pixel_rows(shape, stride, want):
    from kan_sr.ops import _pixel_rows
    t = torch.arange(2000.0).as_strided(shape, stride) if stride else torch.zeros(shape)
    u, ib, ip, S = _pixel_rows(t)
    n = 1
    for k in shape[1:-1]:
        n *= k
    assert S == n and torch.equal(u, t)
    if want is None:
        assert u.is_contiguous() and (ib, ip) == (n * shape[-1], shape[-1])
    else:
        assert (ib, ip) == want and u.data_ptr() == t.data_ptr()
