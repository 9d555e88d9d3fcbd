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


def test_muon_refuses_what_it_cannot_take():
    from kan_sr._lib import KsrError
    from kan_sr.muon import Muon, as_matrix, muon_update, newton_schulz
    w = torch.randn(4, 4)
    for bad in (lambda: newton_schulz(w), lambda: newton_schulz(w, steps=0), lambda: newton_schulz(w, coefficients=(1.0, 2.0)),
                lambda: muon_update([w], [w], [w.clone()], lr=0.1), lambda: Muon([torch.nn.Parameter(w[0])]),
                lambda: Muon([torch.nn.Parameter(w.double())]), lambda: Muon([torch.nn.Parameter(w)], momentum=1.0),
                lambda: Muon([torch.nn.Parameter(w)], precision="fp64")):
        with pytest.raises(KsrError):
            bad()
    assert as_matrix((64, 32, 3, 3)) == (64, 288) and as_matrix((5,)) is None and as_matrix((5, 7)) == (5, 7)


def test_muon_refuses_at_the_abi():
    from kan_sr import _lib
    from kan_sr.muon import MATRIX_WORDS, _matrix
    L = _lib.lib()
    A = 1 << 20                                  # addresses that are never read: the checks come first

    def one(src=A, dst=A, mom=A, rs=8, rows=8, cols=8, batch=1):
        return (c_int64 * MATRIX_WORDS)(*_matrix(src or 0, dst or 0, mom or 0, rs, 1, 0, rows & 0xffffffff, cols, batch))

    def call(mats, bf16=0, muon=1, steps=5, coef=(3.4445, -4.775, 2.0315), eps=1e-7, ws=None, ws_bytes=0, count=1):
        return L.ksr_muon_batch(mats, c_int(count), c_int(bf16), c_int(1), c_int(muon), c_int(steps), *(c_float(v) for v in coef),
                                c_float(eps), c_float(0.9), c_int(1), c_float(1.0), c_float(0.1), None, c_float(0.0), c_float(0.2),
                                ws, c_int64(ws_bytes), None)

    assert call(one(src=None)) == -1 and call(one(dst=None)) == -1 and call(one(mom=None)) == -1
    assert b"null pointer" in L.ksr_last_error()
    assert call(None) == -1 and call(one(rows=-1)) == -1 and call(one(rs=-8)) == -1 and call(one(src=A + 2)) == -1
    assert call(one(), bf16=1) == -1 and call(one(), steps=0) == -1 and call(one(), steps=33) == -1
    assert call(one(), eps=float("nan")) == -1 and call(one(), eps=float("inf")) == -1
    assert call(one(), coef=(9.0, 0.0, 0.0)) == -2 and b"coefficients" in L.ksr_last_error()
    assert call(one(), coef=(float("nan"), 0.0, 0.0)) == -2
    assert call(one(rows=1 << 21)) == -2 and call(one(rows=1 << 16, cols=1 << 16)) == -2 and call(one(batch=1 << 25)) == -2
    assert call(one(rows=100, cols=100)) == -1 and b"workspace" in L.ksr_last_error()
    need = L.ksr_muon_ws_bytes(one(rows=100, cols=100), c_int(1), c_int(1))
    assert need > 0 and L.ksr_muon_ws_bytes(one(rows=64, cols=1024), c_int(1), c_int(1)) == 0
    assert call(one(rows=100, cols=100), ws=c_void_p(A + 8), ws_bytes=need) == -1
    assert call(one(rows=0)) == 0 and call(None, count=0) == 0


def test_flat_runs_and_the_matrices_that_muon_takes():
    from kan_sr.train import flat_runs, takes_muon
    assert list(flat_runs([(0, 4), (4, 6), (12, 1), (13, 2)])) == [0, 10, 12, 3] and len(flat_runs([])) == 0
    pick = [("ffn3.pointwise1.weight", (64, 64, 1, 1), True), ("ffn3.depthwise.weight", (64, 1, 3, 3), False), ("feed.weight", (160, 64, 1, 1), False),
            ("encoder.layers.0.linear1.weight", (32, 64), True), ("encoder.norm.weight", (64,), False), ("ffn1.pointwise2.weight", (64, 1, 1, 1), False),
            ("reproj.conv.weight", (160, 4, 1, 1), False), ("down4.maxpool_conv.1.double_conv.0.weight", (64, 32, 3, 3), True)]
    assert all(takes_muon(n, torch.Size(s)) == want for n, s, want in pick)


def test_adam_runs_refusals():
    from kan_sr import _lib
    L, fake = _lib.lib(), c_void_p(1 << 20)

    def call(runs, n, step=1, lr_dev=None, step_dev=None):
        return L.ksr_adam_step_runs(fake, fake, fake, fake, runs, c_int(n), c_float(1.0), lr_dev, c_float(0.9), c_float(0.9), c_float(1e-8),
                                    c_float(0.0), c_int(step), step_dev, c_float(1.0), None)

    two = (c_int64 * 2)(0, 4)
    assert call(None, 1) == -1 and call(two, -1) == -1 and call(two, 1, step=0) == -1 and call(two, 1, lr_dev=fake) == -1
    assert call((c_int64 * 2)(-1, 4), 1) == -1 and call((c_int64 * 2)(0, 1 << 31), 1) == -1
    assert call(two, 0) == 0 and call((c_int64 * 2)(0, 0), 1) == 0
    assert call((c_int64 * 4)(0, 4, 3, 2), 2) == -1 and call((c_int64 * 4)(4, 2, 0, 2), 2) == -1 and call((c_int64 * 4)(7, 0, 7, 0), 2) == 0


def test_group_norm_unet_has_the_batch_norm_keys_without_running_statistics():
    from kan_sr.unet import UNet
    batch, group = UNet(1, 40).state_dict(), UNet(1, 40, norm="group").state_dict()
    assert set(group) == {k for k in batch if "running" not in k and "num_batches" not in k}
    assert all(group[k].shape == batch[k].shape for k in group)


def test_group_norm_limits_of_an_image():
    from kan_sr import _lib
    L = _lib.lib()

    def ws(B, S, C, G):
        return L.ksr_group_norm_ws_floats(c_int64(B), c_int64(S), c_int(C), c_int(G), c_int(0))

    # 2^32 threads and more in a launch: images in ranges, one image's groups have to fit
    assert ws(1 << 20, 1, 512, 32) > 0 and ws(1 << 23, 2, 8, 8) > 0
    assert ws(1, 2, 1 << 23, 1 << 23) > 0 and ws(1, 300, 1 << 23, 1 << 23) == -1 and b"launch limits" in L.ksr_last_error()
    assert ws(1, 2, 1 << 25, 1 << 25) == -1
