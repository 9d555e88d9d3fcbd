"""CPU oracle for the ConvSepKAN hot path.  TEST INFRASTRUCTURE ONLY.

This file is the checker, never the product: only tests/, __graft_entry__.smoke()
and bench.py's cpu_baseline leg may import it.  It is a from-scratch functional
restatement (plain torch ops on CPU tensors, fp32 or fp64) of the algorithm the
reference implements with nn.Modules.  Parity is PINNED: tests/test_oracle_golden.py
checks every function below against golden vectors produced by importing the
reference itself (tests/golden/make_golden.py).

Every function takes a flat ``params`` dict that uses the reference's own
state_dict key names (e.g. ``layers.0.encoder.encoder.ffn2.gate.weight``), so a
reference checkpoint is directly usable.

Reference map (paths relative to the reference repository root):
  knot_vector          conv_sep_kan/kan_layer.py:14-29   generate_control_points
  bspline_basis        conv_sep_kan/bspline.py:4-28      compute_bspline
  kan_eval             conv_sep_kan/kan_layer.py:68-84, 106-118, 153-162
  kan_cell             conv_sep_kan/conv_sep_kan_cells.py:123-156
  pixel_shuffle        conv_sep_kan/conv_sep_kan.py:18,38 (nn.PixelShuffle)
  ffn                  conv_sep_kan/unet_blocks.py:212-241
  gated_ffn            conv_sep_kan/unet_blocks.py:244-275
  batch_tx_layer       conv_sep_kan/gazetr.py:35-66 (+ nn.MultiheadAttention, batch_first)
  gazetr               conv_sep_kan/gazetr.py:100-119
  bilinear_up          conv_sep_kan/conv_sep_kan.py:33-34 (F.interpolate bilinear)
  conv_sep_kan_forward conv_sep_kan/conv_sep_kan.py:29-42
  double_conv          conv_sep_kan/unet_blocks.py:9-31   (conv3x3 -> BatchNorm2d -> ReLU, twice)
  anchor_attention     conv_sep_kan/unet_blocks.py:91-178 SelfAttention
  unet                 conv_sep_kan/unet.py:7-42, unet_blocks.py:34-88
"""
from __future__ import annotations

import math
from typing import Dict, Optional, Sequence

import torch
import torch.nn.functional as F

Params = Dict[str, torch.Tensor]


# --------------------------------------------------------------------------- spline
def knot_vector(grid_size: int, spline_order: int, grid_range: Sequence[float],
                dtype=torch.float32) -> torch.Tensor:
    """Uniform knots t_j = j*h + lo, j = -k .. G+k, ALWAYS evaluated in fp32 as
    (float32(j) * float32(h)) + lo (one rounding after the multiply, one after the
    add) and only then cast to ``dtype``: the fp32 rounding of the knots is part of
    the algorithm (e.g. t_6 = 0.20000005 for G=5), also for an fp64 evaluation."""
    lo, hi = grid_range[0], grid_range[1]
    h = (hi - lo) / grid_size
    j = torch.arange(-spline_order, grid_size + spline_order + 1)
    return (j * h + lo).to(dtype)   # int64 tensor * python float -> float32


def bspline_basis(x: torch.Tensor, t: torch.Tensor, k: int) -> torch.Tensor:
    """Cox-de Boor recursion on one shared knot vector.

    x: [N, I]; t: [G+2k+1]; returns [N, I, G+k].  The order-0 indicator is the
    half-open test t_j <= x < t_{j+1}; outside [t_0, t_last) every basis is 0.
    The indicator carries no gradient; d/dx flows through the (x-t)/(dt) factors.
    """
    xe = x.unsqueeze(-1)                                   # [N, I, 1]
    b = ((xe >= t[:-1]) & (xe < t[1:])).to(x.dtype)        # [N, I, M-1]
    m = t.numel()
    for p in range(1, k + 1):
        n = m - (p + 1)
        left = (xe - t[:n]) / (t[p:-1] - t[:n])
        right = (t[p + 1:] - xe) / (t[p + 1:] - t[1:n + 1])
        b = left * b[..., :-1] + right * b[..., 1:]
    return b


def kan_eval(x: torch.Tensor, coef: torch.Tensor, uw: torch.Tensor, rw: torch.Tensor,
             t: torch.Tensor, k: int) -> torch.Tensor:
    """Per-sample KAN layer.  x [N,I]; coef [N,O,I,K]; uw, rw [N,O,I] -> [N,O].

    out[n,o] = sum_i ( rw[n,o,i]*silu(x[n,i]) + uw[n,o,i]*sum_g B_g(x[n,i])*coef[n,o,i,g] )
    """
    basis = bspline_basis(x, t, k)                          # [N, I, K]
    spline = (basis.unsqueeze(1) * coef).sum(-1)            # [N, O, I]
    phi = rw * F.silu(x).unsqueeze(1) + uw * spline
    return phi.sum(-1)


def kan_param_count(in_dim: int, out_dim: int, grid_size: int, spline_order: int) -> int:
    """P = O*I*(G+k) coefficients + O*I spline weights + O*I residual weights."""
    return out_dim * in_dim * (grid_size + spline_order + 2)


def kan_cell(x: torch.Tensor, w: torch.Tensor, out_dim: int, grid_size: int,
             spline_order: int, grid_range: Sequence[float]) -> torch.Tensor:
    """x [B,I,H,W], w [B,P,H,W] -> [B,O,H,W].  Channel layout of w at each pixel:
    [coef (o-major, then i, then g) | uw (o,i) | rw (o,i)]."""
    B, I, H, W = x.shape
    O, K = out_dim, grid_size + spline_order
    wn = w.permute(0, 2, 3, 1).reshape(B * H * W, -1)
    xn = x.permute(0, 2, 3, 1).reshape(B * H * W, I)
    n_coef = O * I * K
    coef = wn[:, :n_coef].reshape(-1, O, I, K)
    uw = wn[:, n_coef:n_coef + O * I].reshape(-1, O, I)
    rw = wn[:, n_coef + O * I:n_coef + 2 * O * I].reshape(-1, O, I)
    t = knot_vector(grid_size, spline_order, grid_range, dtype=x.dtype)
    y = kan_eval(xn, coef, uw, rw, t, spline_order)
    return y.reshape(B, H, W, O).permute(0, 3, 1, 2)


def pixel_shuffle(y: torch.Tensor, r: int) -> torch.Tensor:
    """out[b, c, h*r+i, w*r+j] = y[b, c*r*r + i*r + j, h, w]."""
    B, C, H, W = y.shape
    c = C // (r * r)
    return y.reshape(B, c, r, r, H, W).permute(0, 1, 4, 2, 5, 3).reshape(B, c, H * r, W * r)


# --------------------------------------------------------------------------- convs
def ffn(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """pointwise1 -> depthwise 3x3 (zero pad 1, groups=C) -> ReLU -> pointwise2."""
    h = F.conv2d(x, p[prefix + "pointwise1.weight"], p[prefix + "pointwise1.bias"])
    h = F.conv2d(h, p[prefix + "depthwise.weight"], p[prefix + "depthwise.bias"],
                 padding=1, groups=h.shape[1])
    h = torch.relu(h)
    return F.conv2d(h, p[prefix + "pointwise2.weight"], p[prefix + "pointwise2.bias"])


def gated_ffn(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """t = relu(fn_1(x)) [2C]; value = t[:C]; gate = dw3x3(t[C:]); fn_2(value*gate)."""
    t = torch.relu(F.conv2d(x, p[prefix + "fn_1.0.weight"], p[prefix + "fn_1.0.bias"]))
    c = t.shape[1] // 2
    val, g = t[:, :c], t[:, c:]
    g = F.conv2d(g, p[prefix + "gate.weight"], p[prefix + "gate.bias"], padding=1, groups=c)
    return F.conv2d(val * g, p[prefix + "fn_2.weight"], p[prefix + "fn_2.bias"])


# --------------------------------------------------------------------------- transformer over the batch axis
def batch_tx_layer(s: torch.Tensor, p: Params, prefix: str, nhead: int = 2) -> torch.Tensor:
    """Post-LN encoder layer, eval mode (dropout off).  s: [L, S, E] where L indexes
    pixels and S is the (local) batch: attention mixes the S images at one pixel."""
    L, S, E = s.shape
    hd = E // nhead
    qkv = s @ p[prefix + "self_attn.in_proj_weight"].t() + p[prefix + "self_attn.in_proj_bias"]
    q, k, v = qkv.split(E, dim=-1)
    q = q.reshape(L, S, nhead, hd).transpose(1, 2)           # [L, h, S, hd]
    k = k.reshape(L, S, nhead, hd).transpose(1, 2)
    v = v.reshape(L, S, nhead, hd).transpose(1, 2)
    att = torch.softmax((q @ k.transpose(-1, -2)) / math.sqrt(hd), dim=-1)
    ctx = (att @ v).transpose(1, 2).reshape(L, S, E)
    a = ctx @ p[prefix + "self_attn.out_proj.weight"].t() + p[prefix + "self_attn.out_proj.bias"]
    s = F.layer_norm(s + a, (E,), p[prefix + "norm1.weight"], p[prefix + "norm1.bias"])
    m = torch.relu(s @ p[prefix + "linear1.weight"].t() + p[prefix + "linear1.bias"])
    m = m @ p[prefix + "linear2.weight"].t() + p[prefix + "linear2.bias"]
    return F.layer_norm(s + m, (E,), p[prefix + "norm2.weight"], p[prefix + "norm2.bias"])


def gazetr_features(x: torch.Tensor, p: Params, prefix: str, num_layers: int = 2) -> torch.Tensor:
    """Hyper-encoder trunk up to (not including) the `feed` 1x1 conv. x [B,1,H,W] -> [B,64,H,W]."""
    h = ffn(x, p, prefix + "ffn1.")
    h = torch.sigmoid(gated_ffn(h, p, prefix + "ffn2."))
    h = ffn(h, p, prefix + "ffn3.")
    h = torch.sigmoid(gated_ffn(h, p, prefix + "ffn4."))
    B, C, H, W = h.shape
    s = h.permute(2, 3, 0, 1).reshape(H * W, B, C)          # (h w) b c
    for i in range(num_layers):
        s = batch_tx_layer(s, p, f"{prefix}encoder.layers.{i}.")
    s = F.layer_norm(s, (C,), p[prefix + "encoder.norm.weight"], p[prefix + "encoder.norm.bias"])
    return s.reshape(H, W, B, C).permute(2, 3, 0, 1)


def gazetr(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    feat = gazetr_features(x, p, prefix)
    return F.conv2d(feat, p[prefix + "feed.weight"], p[prefix + "feed.bias"])


# --------------------------------------------------------------------------- channel attention
def chan_attention(x: torch.Tensor, p: Params, prefix: str, q=None, k=None, v=None) -> torch.Tensor:
    """ConvSepKanAttention.forward (conv_sep_kan/conv_sep_kan_attention.py:48-71): q, k, v = dw3x3(pw(x));
    q, k L2-normalised over the H*W axis (F.normalize, eps 1e-12); a = softmax(q k^T) over the [mid, mid]
    channel-by-channel scores (no temperature); a_proj(a v).  a_dw is a parameter the forward never uses."""
    B, C, H, W = x.shape

    def branch(n):
        t = F.conv2d(x, p[prefix + n + "_proj.weight"], p[prefix + n + "_proj.bias"])
        return F.conv2d(t, p[prefix + n + "_dw.weight"], p[prefix + n + "_dw.bias"], padding=1, groups=t.shape[1])

    q = branch("q") if q is None else q
    k = branch("k") if k is None else k
    v = branch("v") if v is None else v
    q, k, v = (t.reshape(B, t.shape[1], H * W) for t in (q, k, v))
    q = q / q.norm(dim=-1, keepdim=True).clamp_min(1e-12)
    k = k / k.norm(dim=-1, keepdim=True).clamp_min(1e-12)
    a = torch.softmax(q @ k.transpose(-2, -1), dim=-1)
    y = (a @ v).reshape(B, -1, H, W)
    return F.conv2d(y, p[prefix + "a_proj.weight"], p[prefix + "a_proj.bias"])


# --------------------------------------------------------------------------- chroma
def bilinear_up(x: torch.Tensor, r: int) -> torch.Tensor:
    """Bilinear upsample by integer factor r, align_corners=False, no antialias.
    src = (dst + 0.5)/r - 0.5 clamped at 0; i0 = floor(src); i1 = min(i0+1, size-1)."""
    B, C, H, W = x.shape

    def axis(n_in: int):
        d = torch.arange(n_in * r, dtype=x.dtype)
        src = ((d + 0.5) * (1.0 / r) - 0.5).clamp(min=0)
        i0 = src.floor().long().clamp(max=n_in - 1)
        i1 = (i0 + 1).clamp(max=n_in - 1)
        lam = src - i0.to(x.dtype)
        return i0, i1, lam

    y0, y1, ly = axis(H)
    x0, x1, lx = axis(W)
    rows0, rows1 = x[:, :, y0, :], x[:, :, y1, :]
    top = rows0[..., x0] * (1 - lx) + rows0[..., x1] * lx
    bot = rows1[..., x0] * (1 - lx) + rows1[..., x1] * lx
    return top * (1 - ly)[:, None] + bot * ly[:, None]


# --------------------------------------------------------------------------- training loss
def ssim(pred: torch.Tensor, tgt: torch.Tensor, sigma: float = 1.5, k1: float = 0.01, k2: float = 0.03) -> torch.Tensor:
    """torchmetrics' StructuralSimilarityIndexMeasure(data_range=(0, 1)) with its defaults, restated from the
    published definition (torchmetrics is neither installed nor part of the reference tree: parity unpinned).
    Inputs clamped to [0,1]; 11 x 11 Gaussian window; variances clamped at 0; only windows entirely inside the image
    (the library reflect-pads by 5 and then crops 5 from every border of the result, which keeps exactly these);
    mean over pixels and channels per image, then over images."""
    p, t = pred.clamp(0.0, 1.0), tgt.clamp(0.0, 1.0)
    ks = int(3.5 * sigma + 0.5) * 2 + 1
    d = torch.arange((1 - ks) / 2, (1 + ks) / 2, 1, dtype=p.dtype)
    g = torch.exp(-(d / sigma) ** 2 / 2)
    g = g / g.sum()
    C = p.shape[1]
    k2d = (g[:, None] * g[None, :]).expand(C, 1, ks, ks).contiguous()
    stack = torch.cat([p, t, p * p, t * t, p * t])
    out = F.conv2d(stack, k2d, groups=C).split(p.shape[0])
    mu_p, mu_t = out[0], out[1]
    var_p = (out[2] - mu_p * mu_p).clamp_min(0.0)
    var_t = (out[3] - mu_t * mu_t).clamp_min(0.0)
    cov = out[4] - mu_p * mu_t
    c1, c2 = k1 ** 2, k2 ** 2
    s = ((2 * mu_p * mu_t + c1) * (2 * cov + c2)) / ((mu_p * mu_p + mu_t * mu_t + c1) * (var_p + var_t + c2))
    return s.reshape(s.shape[0], -1).mean(-1).mean()


def training_loss(pred: torch.Tensor, tgt: torch.Tensor) -> torch.Tensor:
    """DefaultPipeline.training_step (src/ml/pipelines/default.py:75-84): L1 on the Y plane + 0.15 (1 - SSIM)."""
    return (pred[:, :1] - tgt[:, :1]).abs().mean() + (1.0 - ssim(pred, tgt)) * 0.15


def cosine_warm_restarts_lr(base_lr: float, epoch: int, T_0: int = 500, eta_min: float = 1e-5) -> float:
    """CosineAnnealingWarmRestarts(T_0=500, T_mult=1, eta_min=1e-5) (default.py:66-68), stepped once per epoch."""
    t_cur = epoch % T_0
    return eta_min + (base_lr - eta_min) * (1 + math.cos(math.pi * t_cur / T_0)) / 2


# --------------------------------------------------------------------------- colour
YCBCR_O = torch.tensor([16., 128., 128.]) / 255.
YCBCR_T = torch.tensor([[0.256788235294118, 0.504129411764706, 0.097905882352941],
                        [-0.148223529411765, -0.290992156862745, 0.439215686274510],
                        [0.439215686274510, -0.367788235294118, -0.071427450980392]]).T


def rgb_to_ycbcr(image: torch.Tensor) -> torch.Tensor:
    """src/ml/utils/colors/ycbcr.py:13-41: per pixel ycbcr = rgb @ T + O (SDTV range), shape (*, 3, H, W)."""
    x = image.to(torch.float32)
    rgb = x.reshape(-1, 3, x.shape[-2], x.shape[-1]).permute(0, 2, 3, 1)
    return (rgb @ YCBCR_T + YCBCR_O).permute(0, 3, 1, 2).reshape(x.shape)


def ycbcr_to_rgb(image: torch.Tensor) -> torch.Tensor:
    """src/ml/utils/colors/ycbcr.py:44-73: per pixel rgb = (ycbcr - O) @ T^-1."""
    x = image.to(torch.float32)
    ycc = x.reshape(-1, 3, x.shape[-2], x.shape[-1]).permute(0, 2, 3, 1)
    return ((ycc - YCBCR_O) @ YCBCR_T.inverse()).permute(0, 3, 1, 2).reshape(x.shape)


# --------------------------------------------------------------------------- whole model
def conv_sep_kan_forward(x: torch.Tensor, p: Params, *, out_channels: Sequence[int],
                         grid_size: int, spline_order: int, grid_range: Sequence[float],
                         upscale: int, in_channels: Sequence[int] = (1,), attention: bool = False,
                         backbone: str = "gazetr", train: bool = False, stats: Optional[dict] = None,
                         norm_groups: int = 0) -> torch.Tensor:
    """x [B,3,H,W] (Y,Cb,Cr) -> [B,3,rH,rW].  Every layer sees the Y plane; only the
    last layer's output survives (the reference's loop overwrites y).
    attention=True: the `feed` 1x1 conv is replaced by chan_attention (parameters under `...feed.`), a wiring
    the reference itself does not contain (its ConvSepKanAttention is a stand-alone module).
    backbone="unet": the hyper-encoder is `unet` (conv_sep_kan_encoder.py:7,17 with UNet in place of GazeTR); `train`
    and `stats` are its BatchNorm mode and running-statistics output; norm_groups > 0: its GroupNorm form."""
    n_layers = len(out_channels)
    li = n_layers - 1
    prefix = f"layers.{li}.encoder.encoder."
    yplane = x[:, :1]
    if backbone == "unet":
        w = unet(yplane, p, prefix, train, stats, norm_groups)
    elif attention:
        w = chan_attention(gazetr_features(yplane, p, prefix), p, prefix + "feed.")
    else:
        w = gazetr(yplane, p, prefix)
    y = kan_cell(yplane, w, out_channels[li], grid_size, spline_order, grid_range)
    y = pixel_shuffle(y, upscale)
    cb = bilinear_up(x[:, 1:2], upscale)
    cr = bilinear_up(x[:, 2:3], upscale)
    return torch.cat([y, cb, cr], dim=1)


def init_like_training_setup(p: Params, seed: int = 0) -> Params:
    """Restates the weight re-initialisation the training pipeline applies before
    fitting (src/ml/pipelines/default.py:36-57): conv weights kaiming-normal
    (fan_out, relu) with zero bias; nn.Linear weights N(0, 0.01) with zero bias
    (this covers out_proj / linear1 / linear2 but NOT in_proj_weight/in_proj_bias,
    which are plain Parameters, nor the LayerNorms)."""
    g = torch.Generator().manual_seed(seed)
    out = {}
    for name, v in p.items():
        v = v.clone()
        if v.dim() == 4 and name.endswith(".weight"):
            fan_out = v.shape[0] * v.shape[2] * v.shape[3]
            v.normal_(0.0, math.sqrt(2.0 / fan_out), generator=g)
        elif name.endswith(".bias") and (name[:-5] + ".weight") in p and p[name[:-5] + ".weight"].dim() == 4:
            v.zero_()
        elif any(name.endswith(s) for s in ("out_proj.weight", "linear1.weight", "linear2.weight")):
            v.normal_(0.0, 0.01, generator=g)
        elif any(name.endswith(s) for s in ("out_proj.bias", "linear1.bias", "linear2.bias")):
            v.zero_()
        out[name] = v
    return out


def param_shapes(out_dim: int, grid_size: int, spline_order: int, in_dim: int = 1,
                 layer: int = 0) -> Dict[str, tuple]:
    """Names and shapes of the 52 tensors of one ConvSepKanLayer, in state_dict order."""
    P = kan_param_count(in_dim, out_dim, grid_size, spline_order)
    pre = f"layers.{layer}.encoder.encoder."
    C = 64
    s: Dict[str, tuple] = {}

    def conv(name, co, ci, kh):
        s[pre + name + ".weight"] = (co, ci, kh, kh)
        s[pre + name + ".bias"] = (co,)

    conv("ffn1.pointwise1", in_dim, in_dim, 1)
    conv("ffn1.depthwise", in_dim, 1, 3)
    conv("ffn1.pointwise2", C, in_dim, 1)
    for g in ("ffn2", "ffn4"):
        conv(g + ".fn_1.0", 2 * C, C, 1)
        conv(g + ".fn_2", C, C, 1)
        conv(g + ".gate", C, 1, 3)
        if g == "ffn2":
            conv("ffn3.pointwise1", C, C, 1)
            conv("ffn3.depthwise", C, 1, 3)
            conv("ffn3.pointwise2", C, C, 1)
    for l in range(2):
        q = f"{pre}encoder.layers.{l}."
        s[q + "self_attn.in_proj_weight"] = (3 * C, C)
        s[q + "self_attn.in_proj_bias"] = (3 * C,)
        s[q + "self_attn.out_proj.weight"] = (C, C)
        s[q + "self_attn.out_proj.bias"] = (C,)
        s[q + "linear1.weight"] = (32, C)
        s[q + "linear1.bias"] = (32,)
        s[q + "linear2.weight"] = (C, 32)
        s[q + "linear2.bias"] = (C,)
        for n in ("norm1", "norm2"):
            s[q + n + ".weight"] = (C,)
            s[q + n + ".bias"] = (C,)
    s[pre + "encoder.norm.weight"] = (C,)
    s[pre + "encoder.norm.bias"] = (C,)
    conv("feed", P, C, 1)
    return s


def random_params(out_dim: int, grid_size: int, spline_order: int, seed: int = 0,
                  scale: float = 1.0, dtype=torch.float32) -> Params:
    """Deterministic, non-degenerate parameters (non-zero biases, non-unit LayerNorm
    gains) for parity tests; NOT any initialisation the reference uses."""
    g = torch.Generator().manual_seed(seed)
    out: Params = {}
    for name, shp in param_shapes(out_dim, grid_size, spline_order).items():
        fan_in = 1
        for d in shp[1:]:
            fan_in *= d
        if "norm" in name and name.endswith(".weight"):
            v = 1.0 + 0.1 * torch.randn(shp, generator=g)
        elif name.endswith("bias"):
            v = 0.1 * torch.randn(shp, generator=g)
        else:
            v = scale * torch.randn(shp, generator=g) / math.sqrt(max(fan_in, 1))
        out[name] = v.to(dtype)
    return out


# --------------------------------------------------------------------------- UNet hyper-encoder
def batch_norm_relu(x: torch.Tensor, p: Params, prefix: str, train: bool, stats: Optional[dict] = None,
                    momentum: float = 0.1, eps: float = 1e-5) -> torch.Tensor:
    """BatchNorm2d + ReLU.  train: statistics of this batch (biased variance for the normalisation); the
    running statistics move by `momentum` towards the batch mean and the UNBIASED batch variance and are
    returned through `stats` (key -> new value) instead of being written in place."""
    if train:
        n = x.numel() // x.shape[1]
        mean = x.mean(dim=(0, 2, 3))
        var = ((x - mean[None, :, None, None]) ** 2).mean(dim=(0, 2, 3))
        if stats is not None:
            stats[prefix + "running_mean"] = (1 - momentum) * p[prefix + "running_mean"] + momentum * mean
            stats[prefix + "running_var"] = (1 - momentum) * p[prefix + "running_var"] + momentum * var * n / max(n - 1, 1)
            stats[prefix + "num_batches_tracked"] = p[prefix + "num_batches_tracked"] + 1
    else:
        mean, var = p[prefix + "running_mean"], p[prefix + "running_var"]
    scale = p[prefix + "weight"] / torch.sqrt(var + eps)
    shift = p[prefix + "bias"] - mean * scale
    return torch.relu(x * scale[None, :, None, None] + shift[None, :, None, None])


def group_norm_relu(x: torch.Tensor, p: Params, prefix: str, groups: int, eps: float = 1e-5) -> torch.Tensor:
    """GroupNorm + ReLU (not in the reference): statistics over the pixels and the channels of a group of one image."""
    B, C, H, W = x.shape
    v = x.reshape(B, groups, -1)
    d = v - v.mean(dim=-1, keepdim=True)
    xh = (d / torch.sqrt((d * d).mean(dim=-1, keepdim=True) + eps)).reshape(x.shape)
    return torch.relu(xh * p[prefix + "weight"][None, :, None, None] + p[prefix + "bias"][None, :, None, None])


def double_conv(x: torch.Tensor, p: Params, prefix: str, train: bool, stats: Optional[dict] = None, groups: int = 0) -> torch.Tensor:
    """prefix ends in 'double_conv.': Sequential indices 0 conv, 1 BN, 3 conv, 4 BN (unet_blocks.py:16-28).
    groups > 0: GroupNorm in the place of both BatchNorms."""
    h = F.conv2d(x, p[prefix + "0.weight"], None, padding=1)
    if groups:
        h = F.conv2d(group_norm_relu(h, p, prefix + "1.", groups), p[prefix + "3.weight"], None, padding=1)
        return group_norm_relu(h, p, prefix + "4.", groups)
    h = batch_norm_relu(h, p, prefix + "1.", train, stats)
    h = F.conv2d(h, p[prefix + "3.weight"], None, padding=1)
    return batch_norm_relu(h, p, prefix + "4.", train, stats)


def _reflect_conv_s2(x, w, b=None, groups=1):
    return F.conv2d(F.pad(x, (1, 1, 1, 1), mode="reflect"), w, b, stride=2, groups=groups)


def _l2_rows(t: torch.Tensor, eps: float = 1e-12) -> torch.Tensor:
    return t / t.norm(dim=-1, keepdim=True).clamp_min(eps)


def anchor_attention(x: torch.Tensor, p: Params, prefix: str, heads: int) -> torch.Tensor:
    """SelfAttention.forward (unet_blocks.py:131-178).  The line `b, c, h, w = x.shape` rebinds the optional
    argument `w` to the image WIDTH, so the test `w is not None` always holds and v is multiplied by the width
    (an int): that factor is part of the reference's function and is kept."""
    B, C, H, W = x.shape
    q = _reflect_conv_s2(x, p[prefix + "q_proj.weight"], groups=C)
    k = _reflect_conv_s2(x, p[prefix + "k_proj.weight"])
    v = F.conv2d(x, p[prefix + "v_proj.weight"]) * W
    a = F.conv2d(_reflect_conv_s2(x, p[prefix + "a_proj.0.weight"], groups=C), p[prefix + "a_proj.1.weight"],
                 p[prefix + "a_proj.1.bias"])
    split = lambda t: t.reshape(B, heads, t.shape[1] // heads, -1)      # 'b (head c) h w -> b head c (h w)'
    q, k, v, a = _l2_rows(split(q)), _l2_rows(split(k)), split(v), _l2_rows(split(a))
    attn_a = torch.softmax((q @ a.transpose(-2, -1)) * p[prefix + "temperature_a"], dim=-1)
    attn_k = torch.softmax((a @ k.transpose(-2, -1)) * p[prefix + "temperature_v"], dim=-1)
    out = attn_a @ (attn_k @ v)
    return F.conv2d(out.reshape(B, C, H, W), p[prefix + "project_out.weight"])


UNET_HEADS = {"att1": 2, "att2": 2, "att3": 4, "att4": 4}                    # unet.py:23-26


def unet(x: torch.Tensor, p: Params, prefix: str = "", train: bool = False, stats: Optional[dict] = None,
         groups: int = 0) -> torch.Tensor:
    """UNet(in, P).forward (unet.py:30-42): x [B,1,H,W] -> [B,P,H,W]; H, W >= 16 (sizes that are not multiples of 16:
    the pooling floors and the upsampled tensor is zero-padded to the skip's size)."""
    xs = [double_conv(x, p, prefix + "proj.double_conv.", train, stats, groups)]
    for i in range(1, 5):
        xs.append(double_conv(F.max_pool2d(xs[-1], 2), p, prefix + f"down{i}.maxpool_conv.1.double_conv.", train, stats, groups))
    y = xs[4]
    for i in range(1, 5):
        skip = anchor_attention(xs[4 - i], p, prefix + f"att{5 - i}.", UNET_HEADS[f"att{5 - i}"])
        up = F.conv_transpose2d(y, p[prefix + f"up{i}.up.weight"], p[prefix + f"up{i}.up.bias"], stride=2)
        dy, dx = skip.shape[2] - up.shape[2], skip.shape[3] - up.shape[3]          # unet_blocks.py:68-73
        up = F.pad(up, [dx // 2, dx - dx // 2, dy // 2, dy - dy // 2])
        y = double_conv(torch.cat([skip, up], dim=1), p, prefix + f"up{i}.conv.double_conv.", train, stats, groups)
    return F.conv2d(y, p[prefix + "reproj.conv.weight"], p[prefix + "reproj.conv.bias"])


# --------------------------------------------------------------------------- SeemoRe blocks (conv_sep_kan/seemore.py)
# The top class SeemoRe (seemore.py:13-77) and its RME / ResGroup (:84-107, :162-181) cannot be constructed (RME passes
# mlp_ratio= to a GatedFFN that has no such argument, :176 vs :355-358); the blocks below can, and are pinned on fixtures
# generated from the reference's own modules (tests/golden/seemore.npz).  Forward only.
def sm_layer_norm_cf(x: torch.Tensor, p: Params, prefix: str, eps: float = 1e-6) -> torch.Tensor:
    """LayerNorm(data_format='channels_first') (seemore.py:386-410): per pixel over the channel axis of [B,C,H,W],
    biased variance, eps inside the square root."""
    mu = x.mean(dim=1, keepdim=True)
    var = ((x - mu) ** 2).mean(dim=1, keepdim=True)
    xh = (x - mu) / torch.sqrt(var + eps)
    return xh * p[prefix + "weight"][None, :, None, None] + p[prefix + "bias"][None, :, None, None]


def sm_striped_conv(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """StripedConv2d(depthwise=True) (seemore.py:325-341): 1 x ks then ks x 1 depthwise convolutions, zero padding ks // 2."""
    C = x.shape[1]
    w0, w1 = p[prefix + "conv.0.weight"], p[prefix + "conv.1.weight"]
    ks = w0.shape[-1]
    h = F.conv2d(x, w0, p[prefix + "conv.0.bias"], padding=(0, ks // 2), groups=C)
    return F.conv2d(h, w1, p[prefix + "conv.1.bias"], padding=(ks // 2, 0), groups=C)


def sm_gated_ffn(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """seemore.py's GatedFFN with GELU (:354-382): t = gelu(fn_1(x)) [2C]; value, gate = halves; gelu(fn_2(value * dw3x3(gate)))."""
    t = F.gelu(F.conv2d(x, p[prefix + "fn_1.0.weight"], p[prefix + "fn_1.0.bias"]))
    c = t.shape[1] // 2
    val, g = t[:, :c], t[:, c:]
    ks = p[prefix + "gate.weight"].shape[-1]
    g = F.conv2d(g, p[prefix + "gate.weight"], p[prefix + "gate.bias"], padding=ks // 2, groups=c)
    return F.gelu(F.conv2d(val * g, p[prefix + "fn_2.0.weight"], p[prefix + "fn_2.0.bias"]))


def sm_striped_conv_former(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """StripedConvFormer (seemore.py:134-155): q, v = halves of gelu(to_qv(x)); proj(striped(q) * v)."""
    t = F.gelu(F.conv2d(x, p[prefix + "to_qv.0.weight"], p[prefix + "to_qv.0.bias"]))
    c = t.shape[1] // 2
    q = sm_striped_conv(t[:, :c], p, prefix + "attn.")
    return F.conv2d(q * t[:, c:], p[prefix + "proj.weight"], p[prefix + "proj.bias"])


def sm_sme(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """SME (seemore.py:114-129): x + block(norm_1(x)), then + ffn(norm_2(.))."""
    x = x + sm_striped_conv_former(sm_layer_norm_cf(x, p, prefix + "norm_1."), p, prefix + "block.")
    return x + sm_gated_ffn(sm_layer_norm_cf(x, p, prefix + "norm_2."), p, prefix + "ffn.")


def sm_expert(x: torch.Tensor, k: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """Expert (seemore.py:289-302): conv_3(conv_2(k) * conv_1(x)), all 1x1, through a low-dimensional space."""
    a = F.conv2d(x, p[prefix + "conv_1.weight"], p[prefix + "conv_1.bias"])
    b = F.conv2d(k, p[prefix + "conv_2.weight"], p[prefix + "conv_2.bias"])
    return F.conv2d(a * b, p[prefix + "conv_3.weight"], p[prefix + "conv_3.bias"])


def sm_router(x: torch.Tensor, p: Params, prefix: str) -> torch.Tensor:
    """Router (seemore.py:305-318): global average pool, then a bias-free linear map to one logit per expert."""
    return x.mean(dim=(2, 3)) @ p[prefix + "body.2.weight"].t()


def sm_moe_layer(x: torch.Tensor, k: torch.Tensor, p: Params, prefix: str, topk: int) -> torch.Tensor:
    """MoELayer (seemore.py:261-285): per image, softmax over the router's logits, the top-k experts weighted by their
    probabilities (not renormalised) added to the input.  The reference's train branch evaluates every expert and zeroes
    the others' weights, its eval branch (one image) only the selected ones: the same sum."""
    n_exp = p[prefix + "gate.body.2.weight"].shape[0]
    w = torch.softmax(sm_router(x, p, prefix + "gate."), dim=1)
    top = torch.topk(w, topk, dim=1).indices
    mask = torch.zeros_like(w).scatter_(1, top, 1.0)
    out = x.clone()
    for e in range(n_exp):
        we = (w * mask)[:, e]
        if bool((we != 0).any()):
            out = out + sm_expert(x, k, p, f"{prefix}experts.{e}.") * we[:, None, None, None]
    return out


def sm_moe_block(x: torch.Tensor, p: Params, prefix: str, topk: int, recursive: int, use_shuffle: bool = False) -> torch.Tensor:
    """MoEBlock (seemore.py:188-258): conv_1 (3x3, GELU, 1x1 to 2C) -> [optional channel shuffle in 2 groups] -> halves x, k;
    x = gelu(striped3(x)); k = k + bilinear(conv(agg_conv^recursive(k))) (agg_conv: depthwise 4x4 stride 4 + GELU; conv:
    depthwise 3x3 then 1x1); proj(moe_layer(x, k))."""
    t = F.conv2d(x, p[prefix + "conv_1.0.weight"], p[prefix + "conv_1.0.bias"], padding=1)
    t = F.conv2d(F.gelu(t), p[prefix + "conv_1.2.weight"], p[prefix + "conv_1.2.bias"])
    B, C2, H, W = t.shape
    if use_shuffle:
        t = t.reshape(B, 2, C2 // 2, H, W).transpose(1, 2).reshape(B, C2, H, W)
    c = C2 // 2
    xs, k = t[:, :c], t[:, c:]
    xs = F.gelu(sm_striped_conv(xs, p, prefix + "conv_2.0."))
    a = k
    for _ in range(recursive):
        a = F.gelu(F.conv2d(a, p[prefix + "agg_conv.0.weight"], p[prefix + "agg_conv.0.bias"], stride=4, groups=c))
    a = F.conv2d(a, p[prefix + "conv.0.weight"], p[prefix + "conv.0.bias"], padding=1, groups=c)
    a = F.conv2d(a, p[prefix + "conv.1.weight"], p[prefix + "conv.1.bias"])
    k = k + F.interpolate(a, size=(H, W), mode="bilinear", align_corners=False)
    y = sm_moe_layer(xs, k, p, prefix + "moe_layer.", topk)
    return F.conv2d(y, p[prefix + "proj.weight"], p[prefix + "proj.bias"])
