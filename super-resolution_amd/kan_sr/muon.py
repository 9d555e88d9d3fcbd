"""Newton-Schulz orthogonalisation of matrices and the Muon optimiser on the HIP path.

Muon replaces a weight matrix's momentum by the nearest (semi-)orthogonal matrix, approximately: with X = U / |U|_F a few
steps of X <- a X + (b A + c A A) X, A = X X^T, drive every singular value towards 1.  The products, the momentum update before
them and the weight update after them are kernels of libksr (ksr_muon_batch); matrices with a shorter side of up to 64, which
is all this package's hyper-encoders have, run in one launch for the whole list.
"""
from __future__ import annotations

from array import array
from typing import Iterable, Optional, Sequence

import torch

from ._lib import KsrError, check, has_tangent, lib, on_device_of, stream

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
MATRIX_WORDS = 8                                  # KsrMatrix of include/ksr.h as 64-bit words


def _matrix(src: int, dst: int, momentum: int, row_stride: int, col_stride: int, batch_stride: int, rows: int, cols: int,
            batch: int) -> tuple:
    """One KsrMatrix: three addresses, three strides, rows | cols and batch | 0 as pairs of 32 bits."""
    return src, dst, momentum, row_stride, col_stride, batch_stride, rows | cols << 32, batch


def _run(words: Sequence[int], device_of: torch.Tensor, bf16: bool, split: bool, steps: int, coefficients, eps: float, muon: bool = False,
         momentum: float = 0.0, nesterov: bool = False, grad_scale: float = 1.0, lr: float = 0.0,
         lr_dev: Optional[torch.Tensor] = None, weight_decay: float = 0.0, scale: float = 0.0) -> None:
    L = lib()
    held, n = array("q", words), len(words) // MATRIX_WORDS
    mats = held.buffer_info()[0]
    with on_device_of(device_of):
        nbytes = L.ksr_muon_ws_bytes(mats, n, split)
        if nbytes < 0:
            check(int(nbytes), "ksr_muon_ws_bytes")
        ws = torch.empty(nbytes, device=device_of.device, dtype=torch.uint8) if nbytes else None
        a, b, c = coefficients
        check(L.ksr_muon_batch(mats, n, bf16, split, muon, steps, a, b, c, eps, momentum, nesterov, grad_scale, lr,
                               lr_dev.data_ptr() if lr_dev is not None else None, weight_decay, scale,
                               ws.data_ptr() if nbytes else None, nbytes, stream()), "ksr_muon_batch")


def _steps_and_coefficients(steps, coefficients):
    if not 1 <= int(steps) <= 32:
        raise KsrError(f"newton_schulz: {steps} steps (1 to 32)")
    if len(coefficients) != 3:
        raise KsrError(f"newton_schulz: three coefficients (a, b, c), got {coefficients!r}")
    return int(steps), tuple(float(v) for v in coefficients)


def _split(precision: Optional[str], dtype: torch.dtype) -> bool:
    if precision not in (None, "fp32", "bf16"):
        raise KsrError(f"precision must be 'fp32' or 'bf16', got {precision!r}")
    return dtype is torch.float32 if precision is None else precision == "fp32"


def newton_schulz(g: torch.Tensor, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7,
                  precision: Optional[str] = None) -> torch.Tensor:
    """Orthogonalises the matrices g [..., rows, cols] (float32 or bfloat16, any strides): a dense tensor of g's shape and type.

    X = g / (|g|_F + eps), then `steps` times X <- a X + (b A + c A A) X with A = X X^T (of the transposed matrix where
    rows > cols).  precision: "fp32" (default for float32) forms the products to fp32 accuracy (operands of 22 bits); "bf16"
    (default for bfloat16) takes a third of the matrix work with operands of 11 bits: 2e-4 to 9e-4 of the result before it is
    rounded to bfloat16, which is 1.7e-3 by itself; pass "fp32" where bfloat16 results have to be those of fp32 products.  A
    matrix's result does not depend on what else is in the call.  Not differentiable."""
    steps, coefficients = _steps_and_coefficients(steps, coefficients)
    if g.dim() < 2:
        raise KsrError(f"newton_schulz: g must be [..., rows, cols], got {tuple(g.shape)}")
    if not g.is_cuda:
        raise KsrError("libksr ops need GPU tensors (the HIP path is the only path)")
    if g.dtype not in (torch.float32, torch.bfloat16):
        raise KsrError(f"newton_schulz: g must be float32 or bfloat16, got {g.dtype}")
    if g.requires_grad and torch.is_grad_enabled() or has_tangent(g):
        raise KsrError("newton_schulz is not differentiable: detach g")
    split = _split(precision, g.dtype)
    if torch.jit.is_tracing():                       # a trace records the call, not the allocation of its result alone
        return _NewtonSchulz.apply(g, split, steps, coefficients, eps)
    return _newton_schulz(g, split, steps, coefficients, eps)


def _newton_schulz(g: torch.Tensor, split: bool, steps: int, coefficients, eps: float) -> torch.Tensor:
    out = torch.empty(g.shape, device=g.device, dtype=g.dtype)
    if g.numel() == 0:
        return out
    u = g.detach()
    u = u.unsqueeze(0) if u.dim() == 2 else u.reshape(-1, *u.shape[-2:])
    if max(u.shape) > 1 << 24:
        raise KsrError(f"newton_schulz: {tuple(g.shape)} is too large")
    batch, rows, cols = u.shape
    bs, rs, cs = u.stride()
    _run(_matrix(u.data_ptr(), out.data_ptr(), 0, rs, cs, bs, rows, cols, batch), g, g.dtype is torch.bfloat16, split, steps, coefficients, eps)
    return out


class _NewtonSchulz(torch.autograd.Function):
    @staticmethod
    def forward(ctx, g, split, steps, coefficients, eps):
        return _newton_schulz(g, split, steps, coefficients, eps)

    @staticmethod
    def backward(ctx, *grads):
        raise KsrError("newton_schulz is not differentiable: detach g")


def as_matrix(shape: Sequence[int]):
    """(rows, cols) of a parameter: the first dimension against all others, so a convolution's [out, in, kh, kw] is
    [out, in * kh * kw].  None for vectors and scalars, which Muon does not take."""
    if len(shape) < 2:
        return None
    cols = 1
    for n in shape[1:]:
        cols *= n
    return shape[0], cols


def muon_update(weights, grads, momenta, lr: float, momentum: float = 0.95, nesterov: bool = True, weight_decay: float = 0.0,
                steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7, scale: float = 0.2,
                grad_scale: float = 1.0, precision: Optional[str] = None, lr_dev: Optional[torch.Tensor] = None) -> None:
    """One Muon update of a list of float32 GPU tensors, in place, in few launches:

        m <- momentum m + grad_scale g;   U = grad_scale g + momentum m (nesterov) or m;   O = newton_schulz(U)
        w <- (1 - lr weight_decay) w - lr scale sqrt(max(rows, cols)) O

    Nothing that is written (weights, momenta) may lie between the first and the last element of anything else in the call;
    gradients may be views of each other.  scale = 0.2 gives an update the root mean square of a typical Adam step, so that one learning rate serves both.  lr_dev: a
    one-element float32 GPU tensor that replaces lr (recorded graphs)."""
    steps, coefficients = _steps_and_coefficients(steps, coefficients)
    weights, grads, momenta = list(weights), list(grads), list(momenta)
    if not len(weights) == len(grads) == len(momenta):
        raise KsrError(f"muon_update: {len(weights)} weights, {len(grads)} gradients, {len(momenta)} momenta")
    if not weights:
        return
    device = weights[0].device
    if device.type != "cuda":
        raise KsrError("libksr ops need GPU tensors (the HIP path is the only path)")
    if torch.jit.is_tracing() or has_tangent(*weights, *grads, *momenta):
        raise KsrError("muon_update works in place on plain tensors: it can be neither traced nor differentiated")
    f32 = torch.float32
    if lr_dev is not None and (lr_dev.dtype is not f32 or lr_dev.numel() != 1 or lr_dev.device != device):
        raise KsrError("muon_update: lr_dev must be one float32 on the weights' device")
    every = weights + grads + momenta
    if {t.dtype for t in every} != {f32} or set(map(torch.Tensor.get_device, every)) != {device.index}:
        raise KsrError(f"muon_update: every weight, gradient and momentum must be float32 on {device}")
    # methods mapped over lists: a call's time is the host's (every tensor's attributes in turn: 5 us more for 16 matrices)
    T = torch.Tensor
    shapes = list(map(T.size, weights))
    if not (shapes == list(map(T.size, grads)) == list(map(T.size, momenta)) and all(map(T.is_contiguous, weights + momenta))):
        i = next(i for i, (w, g, m) in enumerate(zip(weights, grads, momenta))
                 if not w.shape == g.shape == m.shape or not w.is_contiguous() or not m.is_contiguous())
        raise KsrError(f"muon_update: tensor {i}: gradient and momentum must have the weight's shape {tuple(shapes[i])}, weight "
                       "and momentum be contiguous")
    words, held, spans = [], [], []
    for shape, g, wp, mp in zip(shapes, grads, map(T.data_ptr, weights), map(T.data_ptr, momenta)):
        if len(shape) == 2:
            rows, cols = shape
            rs, cs = g.stride()
        elif len(shape) > 2:
            rows, cols = as_matrix(shape)
            g, rs, cs = g.contiguous(), cols, 1
            held.append(g)
        else:
            raise KsrError(f"muon_update: a tensor is {tuple(shape)}: matrices only (vectors belong to Adam)")
        if rows > 1 << 24 or cols > 1 << 24:
            raise KsrError(f"muon_update: a tensor is {tuple(shape)}: too large")
        gp = g.data_ptr()
        if wp:
            nbytes = 4 * rows * cols
            spans += (wp, wp + nbytes, True), (mp, mp + nbytes, True), (gp, gp + 4 * ((rows - 1) * rs + (cols - 1) * cs + 1), False)
        words += gp, wp, mp, rs, cs, 0, rows | cols << 32, 1                # _matrix(...)
    spans.sort()
    written = read = 0                                          # where what is written, and read, so far ends
    for first, last, write in spans:                            # the matrices of a call run side by side
        if first < written or write and first < read:
            raise KsrError("muon_update: weights or momenta of the list overlap each other or a gradient, or one is in it twice")
        if write:
            written = last
        elif last > read:
            read = last
    _run(words, weights[0], False, _split(precision, f32), steps, coefficients, eps, True, momentum, nesterov, grad_scale, lr,
         lr_dev, weight_decay, scale)
    # the kernels write behind torch's back: whoever keys on the version counters (autograd, the UNet's kernel-layout weights) sees it
    try:
        torch.autograd.graph.increment_version(weights + momenta)
    except RuntimeError:                             # tensors made in inference mode have no counter, the others still need theirs
        torch.autograd.graph.increment_version([t for t in weights + momenta if not t.is_inference()])


class Muon(torch.optim.Optimizer):
    """torch optimiser over muon_update for parameters of two or more dimensions (convolutions as [out, in * kh * kw]);
    vectors (biases, norms) belong to another optimiser.  Keeps one fp32 momentum per parameter (state "momentum_buffer")."""

    def __init__(self, params: Iterable, lr: float = 1e-3, momentum: float = 0.95, nesterov: bool = True,
                 weight_decay: float = 0.0, steps: int = 5, coefficients: Sequence[float] = COEFFICIENTS, eps: float = 1e-7,
                 scale: float = 0.2, precision: Optional[str] = None):
        steps, coefficients = _steps_and_coefficients(steps, coefficients)
        if lr < 0 or weight_decay < 0 or not 0 <= momentum < 1 or eps < 0:
            raise KsrError(f"Muon: lr = {lr}, momentum = {momentum}, weight_decay = {weight_decay}, eps = {eps}")
        _split(precision, torch.float32)
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, weight_decay=weight_decay, steps=steps,
                                      coefficients=coefficients, eps=eps, scale=scale, precision=precision))
        for group in self.param_groups:
            for p in group["params"]:
                if p.dim() < 2 or p.dtype is not torch.float32:
                    raise KsrError(f"Muon takes float32 parameters of two or more dimensions, got {p.dtype} {tuple(p.shape)}")

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            weights, grads, momenta = [], [], []
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                m = self.state[p].get("momentum_buffer")
                if m is None:
                    m = self.state[p]["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.contiguous_format)
                weights.append(p)
                grads.append(g)
                momenta.append(m)
            muon_update(weights, grads, momenta, group["lr"], group["momentum"], group["nesterov"], group["weight_decay"],
                        group["steps"], group["coefficients"], group["eps"], group["scale"], precision=group["precision"])
        return loss
