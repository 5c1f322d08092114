"""Pure-PyTorch reference implementations of every sodkit op.

These serve two roles:
  1. the CPU execution path (the [BJ:7] plumbing config runs with no GPU);
  2. the fp32 numerics oracle the HIP kernels are unit-tested against
     (SURVEY §4.2.1).

They are differentiable torch code — autograd provides the CPU backward.
On a GPU device, sodkit ops never route here: the HIP extension is required
and fails loudly if missing (no silent eager fallback).
"""

from __future__ import annotations

import math
from typing import Optional

import torch
import torch.nn.functional as F



def _fp(x: torch.Tensor) -> torch.Tensor:
    """Upcast to fp32 compute precision, but keep fp64 (gradcheck) intact."""
    return x if x.dtype == torch.float64 else x.float()

# ---------------------------------------------------------------------------
# Convolution.  sodkit stores conv weights in KRSC layout [Cout, R, S, Cin]
# (torch's channels-last weight layout): the MFMA implicit-GEMM A-operand is
# then W[cout][(r,s,cin)] row-major — coalesced LDS staging with no transpose.
# The reference path permutes to torch's [Cout, Cin, R, S].
# ---------------------------------------------------------------------------

def conv2d(x: torch.Tensor, w_krsc: torch.Tensor, bias: Optional[torch.Tensor],
           stride: int, padding: int, dilation: int) -> torch.Tensor:
    w = w_krsc.permute(0, 3, 1, 2)  # [Cout, Cin, R, S]
    return F.conv2d(x, w, bias, stride=stride, padding=padding, dilation=dilation)


# ---------------------------------------------------------------------------
# Fused BatchNorm(+residual add)(+ReLU).  Training-mode batch stats with
# optional cross-rank stats all-reduce (SyncBN).
# ---------------------------------------------------------------------------

class _SyncSum(torch.autograd.Function):
    """Autograd-correct cross-rank sum: forward all-reduces the stats,
    backward all-reduces the incoming gradient (the C4 backward-stats
    reduction real SyncBN needs — a transparent all_reduce under autograd
    would silently drop the cross-rank gradient terms)."""

    @staticmethod
    def forward(ctx, x, pg):
        ctx.pg = pg
        y = x.clone()
        torch.distributed.all_reduce(y, group=pg)
        return y

    @staticmethod
    def backward(ctx, g):
        g = g.contiguous().clone()
        torch.distributed.all_reduce(g, group=ctx.pg)
        return g, None


def bn_act(x: torch.Tensor, gamma: torch.Tensor, beta: torch.Tensor,
           running_mean: torch.Tensor, running_var: torch.Tensor,
           training: bool, momentum: float, eps: float,
           relu: bool = True, residual: Optional[torch.Tensor] = None,
           process_group=None) -> torch.Tensor:
    xf = _fp(x)
    if training:
        n = x.numel() // x.shape[1]
        dims = [0, 2, 3]
        s = xf.sum(dim=dims)
        ss = (xf * xf).sum(dim=dims)
        cnt = torch.full((1,), float(n), device=x.device)
        if process_group is not None and torch.distributed.is_initialized() \
                and torch.distributed.get_world_size(process_group) > 1:
            packed = _SyncSum.apply(torch.cat([s, ss, cnt]), process_group)
            s, ss, cnt = packed[: s.numel()], packed[s.numel():-1], packed[-1:]
        n_tot = cnt.item()
        mean = s / n_tot
        # clamp: the two-pass form can go slightly negative by cancellation
        var = (ss / n_tot - mean * mean).clamp_min(0.0)
        with torch.no_grad():
            unbiased = var * (n_tot / max(n_tot - 1.0, 1.0))
            running_mean.mul_(1 - momentum).add_(mean.detach(), alpha=momentum)
            running_var.mul_(1 - momentum).add_(unbiased.detach(), alpha=momentum)
    else:
        mean, var = running_mean, running_var
    invstd = torch.rsqrt(var.clamp_min(0.0) + eps)
    y = (xf - mean.view(1, -1, 1, 1)) * (invstd * gamma).view(1, -1, 1, 1) \
        + beta.view(1, -1, 1, 1)
    if residual is not None:
        y = y + _fp(residual)
    if relu:
        y = F.relu(y)
    return y.to(x.dtype)


# ---------------------------------------------------------------------------
# Bilinear resize (+ optional fused add) — `cus_sample` / `upsample_add`
# parity (SURVEY §2.1 utils/tensor_ops.py).
# ---------------------------------------------------------------------------

def bilinear2d(x: torch.Tensor, out_h: int, out_w: int,
               add: Optional[torch.Tensor] = None,
               align_corners: bool = False) -> torch.Tensor:
    y = F.interpolate(_fp(x), size=(out_h, out_w), mode="bilinear",
                      align_corners=align_corners)
    if add is not None:
        y = y + _fp(add)
    return y.to(x.dtype)


# ---------------------------------------------------------------------------
# Dynamic (spatially-variant) 3x3 filtering — HDFNet DDPM (K10).
# ---------------------------------------------------------------------------

def dynamic_filter(x: torch.Tensor, kernels: torch.Tensor,
                   dilation: int) -> torch.Tensor:
    """x [N,C,H,W], kernels [N,9,H,W] -> sum_e k_e * shift_e(x), zero pad."""
    n, c, h, w = x.shape
    cols = F.unfold(x.contiguous(), 3, dilation=dilation, padding=dilation)
    cols = cols.view(n, c, 9, h * w)
    k = kernels.reshape(n, 1, 9, h * w)
    return (cols * k).sum(dim=2).view(n, c, h, w)


# ---------------------------------------------------------------------------
# Hybrid pixel-wise loss: BCE-with-logits + soft IoU + SSIM (the [BJ:5]
# generalized loss; the reference's CEL/HEL family, SURVEY §2.1 loss/).
# All math in fp32.  Per-image IoU and SSIM, averaged over the batch.
# ---------------------------------------------------------------------------

_SSIM_WIN = 11
_SSIM_SIGMA = 1.5
_SSIM_C1 = 0.01 ** 2
_SSIM_C2 = 0.03 ** 2


def _gaussian_window(device, dtype=torch.float32):
    half = _SSIM_WIN // 2
    g = torch.tensor(
        [math.exp(-((i - half) ** 2) / (2 * _SSIM_SIGMA ** 2)) for i in range(_SSIM_WIN)],
        device=device, dtype=dtype)
    g = g / g.sum()
    w2d = torch.outer(g, g)
    return w2d.view(1, 1, _SSIM_WIN, _SSIM_WIN)


def ssim_map(p: torch.Tensor, t: torch.Tensor) -> torch.Tensor:
    """Per-pixel SSIM between probability map p and target t, both [N,1,H,W]
    fp32 in [0,1].  11x11 gaussian window, reflection-free (same padding via
    conv with zero pad is wrong at edges; use valid region weighting by
    renormalizing the window mass — implemented by dividing by the window sum
    of a ones image)."""
    w = _gaussian_window(p.device, p.dtype)
    pad = _SSIM_WIN // 2
    ones = torch.ones_like(p)
    wsum = F.conv2d(ones, w, padding=pad)            # window mass inside image
    mu_p = F.conv2d(p, w, padding=pad) / wsum
    mu_t = F.conv2d(t, w, padding=pad) / wsum
    s_pp = F.conv2d(p * p, w, padding=pad) / wsum - mu_p * mu_p
    s_tt = F.conv2d(t * t, w, padding=pad) / wsum - mu_t * mu_t
    s_pt = F.conv2d(p * t, w, padding=pad) / wsum - mu_p * mu_t
    num = (2 * mu_p * mu_t + _SSIM_C1) * (2 * s_pt + _SSIM_C2)
    den = (mu_p * mu_p + mu_t * mu_t + _SSIM_C1) * (s_pp + s_tt + _SSIM_C2)
    return num / den


def hybrid_loss(logits: torch.Tensor, target: torch.Tensor,
                w_bce: float = 1.0, w_iou: float = 1.0,
                w_ssim: float = 1.0) -> torch.Tensor:
    z = _fp(logits)
    t = _fp(target)
    loss = z.new_zeros(())
    if w_bce:
        loss = loss + w_bce * F.binary_cross_entropy_with_logits(z, t)
    p = torch.sigmoid(z)
    if w_iou:
        inter = (p * t).sum(dim=[1, 2, 3])
        union = p.sum(dim=[1, 2, 3]) + t.sum(dim=[1, 2, 3]) - inter
        iou = (inter + 1.0) / (union + 1.0)
        loss = loss + w_iou * (1.0 - iou).mean()
    if w_ssim:
        loss = loss + w_ssim * (1.0 - ssim_map(p, t).mean())
    return loss


# ---------------------------------------------------------------------------
# SGD with momentum + fp32 master weights (reference math for the fused
# multi-tensor kernel K11).  Operates in-place; grad scale folds in the
# 1/world_size gradient average and any loss-scale.
# ---------------------------------------------------------------------------

@torch.no_grad()
def sgd_step(param, grad, master32, momentum_buf32, lr: float, momentum: float,
             weight_decay: float, grad_scale: float, nesterov: bool = False):
    g = grad.float() * grad_scale
    if weight_decay:
        g = g.add(master32, alpha=weight_decay)
    momentum_buf32.mul_(momentum).add_(g)
    if nesterov:
        g = g.add(momentum_buf32, alpha=momentum)
    else:
        g = momentum_buf32
    master32.add_(g, alpha=-lr)
    param.copy_(master32.to(param.dtype))


# ---------------------------------------------------------------------------
# Global gradient norm -> clip multiplier, overflow skip, dynamic loss scale.
# ---------------------------------------------------------------------------

_TINY32 = torch.finfo(torch.float32).tiny


@torch.no_grad()
def grad_norm(grads, prescale: float, max_norm: float, loss_scale=None,
              good_steps=None, skips=None, growth_interval: int = 500):
    for g in grads:
        if g.device != grads[0].device or g.layout != torch.strided:
            raise ValueError("gradients must be dense and on one device")
        if g.dtype not in (torch.float32, torch.bfloat16, torch.float16):
            raise ValueError(f"gradients must be float32, bfloat16 or "
                             f"float16, got {g.dtype}")
    total = sum(g.double().square().sum() for g in grads)
    scale = (loss_scale.double() if loss_scale is not None
             else torch.ones_like(total))
    norm = (total.sqrt() * prescale / scale).float()
    finite = torch.isfinite(norm)
    clip = torch.ones_like(total)
    if max_norm > 0:
        clip = (max_norm / (norm.double() + 1e-6)).clamp(max=1.0)
    # 0 means "skip the step": a finite norm never rounds to it
    mult = torch.where(finite, (clip / scale).float().clamp(min=_TINY32),
                       torch.zeros_like(norm))
    if good_steps is not None:
        good = torch.where(finite, good_steps + 1.0, torch.zeros_like(norm))
        grow = good >= float(growth_interval)
        up = torch.where(grow, (loss_scale * 2.0).clamp(max=65536.0),
                         loss_scale)
        loss_scale.copy_(torch.where(finite, up,
                                     (loss_scale * 0.5).clamp(min=1.0)))
        good_steps.copy_(torch.where(grow, torch.zeros_like(good), good))
        skips += (~finite).float()
    return norm, mult


# ---------------------------------------------------------------------------
# AdamW, moments in 32 or in 8 bits, on the flat elements of one tensor.  The
# operations and their order are the kernel's (csrc/adamw.hip), each rounded
# to float32 by itself.  `gs` is a float32 scalar tensor.
# ---------------------------------------------------------------------------

ADAMW_BLOCK = 256
_M32 = 0xFFFFFFFF


def _adamw_moments(grad, m, v, betas, gs):
    b1, b2 = betas
    g = grad.float() * gs
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    return m, v


def _root(v):
    """The float32 root to the last bit, which torch's own on the CPU is not (one
    in six is a unit off): the root in 64 bits, rounded."""
    return v.double().sqrt().float()


def _power(b: float, step: int) -> float:
    """b^step by squaring, each product rounded to float64 as in the kernel.
    A squaring doubles the error that it gets, so the error grows with step:
    under step * 2^-53, relative.  `**` is nearer, but not the same bits, and
    1 - b^step takes the difference into the last bit of a float32 now and
    then where b is near one."""
    p = 1.0
    while step:
        if step & 1:
            p *= b
        b *= b
        step >>= 1
    return p


def _adamw_weight(param, w, m, r, lr, step, betas, eps, weight_decay):
    b1, b2 = betas
    rate = lr / (1 - _power(b1, step))
    den = r * (1 / math.sqrt(1 - _power(b2, step))) + eps
    new = w * (1 - lr * weight_decay) - (m / den) * rate
    w.copy_(new)
    if param.dtype == torch.float16:      # saturates, as every kernel's cast
        big = torch.finfo(torch.float16).max
        new = new.clamp(-big, big)
    param.copy_(new)


@torch.no_grad()
def adamw_step(param, grad, w, exp_avg, exp_avg_sq, lr: float, step: int,
               betas, eps: float, weight_decay: float, gs):
    m, v = _adamw_moments(grad, exp_avg, exp_avg_sq, betas, gs)
    exp_avg.copy_(m)
    exp_avg_sq.copy_(v)
    _adamw_weight(param, w, m, _root(v), lr, step, betas, eps, weight_decay)


def _mix32(h):
    """The finalizer of MurmurHash3 (Appleby, public domain) on int64 tensors
    or ints that hold 32 bits."""
    h = h ^ (h >> 16)
    h = (h * 0x85EBCA6B) & _M32
    h = h ^ (h >> 13)
    h = (h * 0xC2B2AE35) & _M32
    return h ^ (h >> 16)


def adamw8_noise(places: int, seed: int, step: int, tensor: int,
                 first: int = 0):
    """The 32 random bits of each element from `first` on: the upper half rounds
    m, the lower half r."""
    key = _mix32((seed + step * 0x9E3779B9) & _M32)
    key = _mix32((key + tensor) & _M32)
    i = torch.arange(first, first + places, dtype=torch.int64)
    key = _mix32((key + (i >> 32)) & _M32)
    return _mix32(((i & _M32) + key) & _M32)


def _adamw8_grid(code, bias: int, shift: int):
    bits = torch.where(code > 0, (code + bias) << shift, torch.zeros_like(code))
    return bits.view(torch.float32)


def adamw8_decode(code_m, code_r, scales):
    """(m, r) in float32: the values of the codes of whole blocks."""
    cm, cr = code_m.to(torch.int32), code_r.to(torch.int32)
    m = _adamw8_grid(cm & 127, 889, 20).view(-1, ADAMW_BLOCK) * scales[:, :1]
    m = torch.where((cm > 127).view_as(m), -m, m)
    r = _adamw8_grid(cr, 1777, 19).view(-1, ADAMW_BLOCK) * scales[:, 1:]
    return m.reshape(-1), r.reshape(-1)


def adamw8_encode(m, r, noise):
    """(code_m, code_r, scales) of whole blocks, rounded by the noise."""
    def codes(x, top, noise16, bias, shift):
        inv = 1.0 / top.clamp(min=2.0 ** -100)
        bits = (x * inv).view(torch.int32) & 0x7FFFFFFF
        bits = bits.clamp(max=0x3F800000)
        return ((bits + (noise16 << (shift - 16))) >> shift) - bias

    m, r = m.view(-1, ADAMW_BLOCK), r.view(-1, ADAMW_BLOCK)
    noise = noise.view(-1, ADAMW_BLOCK)
    sm, sr = m.abs().amax(1, keepdim=True), r.amax(1, keepdim=True)
    # a square past float32 leaves m finite beside an r that stops every step:
    # neither moment of such a block is finite, as in the kernel
    sm = torch.where(torch.isfinite(sr), sm, sr)
    cm = codes(m.abs(), sm, (noise >> 16).to(torch.int32), 889, 20).clamp(min=0)
    cm = torch.where(torch.signbit(m), cm + 128, cm)
    cr = codes(r, sr, (noise & 0xFFFF).to(torch.int32), 1777, 19).clamp(min=1)
    cr = torch.where(r > 0, cr, torch.zeros_like(cr))
    return (cm.to(torch.uint8).view(-1), cr.to(torch.uint8).view(-1),
            torch.cat([sm, sr], 1))


@torch.no_grad()
def adamw8_step(param, grad, w, code_m, code_r, scales, lr: float, step: int,
                betas, eps: float, weight_decay: float, gs, seed: int,
                tensor: int):
    n, places = param.numel(), code_m.numel()
    m, r = adamw8_decode(code_m, code_r, scales)
    m, v = _adamw_moments(F.pad(grad.float(), (0, places - n)), m, r * r,
                          betas, gs)
    r = _root(v)
    _adamw_weight(param, w, m[:n], r[:n], lr, step, betas, eps, weight_decay)
    for dst, src in zip((code_m, code_r, scales),
                        adamw8_encode(m, r, adamw8_noise(places, seed, step, tensor))):
        dst.copy_(src)
