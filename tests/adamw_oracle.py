"""The AdamW step and the gradient norm in 64 bits, from their definitions, and
the bounds that rounding to float32 allows around them."""

import math

import torch

U = 2.0 ** -24      # half a step of float32, relative


def step64(w, g, m, v, t, lr, betas, eps, wd, gs):
    """float64 in, (w, m, v) and elementwise bounds of their float32 errors out.

    m: the gradient's scale (1 for the product, 1 for its own rounding), both
    products, 1-b1 and b1 as float32 and the sum: under 8 half steps of the
    terms.  v: the same with the gradient twice, all terms positive: under 10
    of the sum.  The update inherits m's error over its own size and half of
    v's, and adds the rounded root, its scale, eps' sum, the quotient, the
    rate and the product: 16 more; w adds the decay, its product and the sum."""
    b1, b2 = betas
    g = g * gs
    m1 = b1 * m + (1 - b1) * g
    v1 = b2 * v + (1 - b2) * g * g
    em = 8 * U * ((b1 * m).abs() + ((1 - b1) * g).abs()) + 2.0 ** -148
    ev = 10 * U * v1 + 2.0 ** -145
    rate = lr / (1 - b1 ** t)
    bc2 = math.sqrt(1 - b2 ** t)
    den = v1.sqrt() / bc2 + eps
    # tiny v: its absolute error of 2^-145 moves the root by at most 2^-72
    upd = rate * m1 / den
    w1 = w * (1 - lr * wd) - upd
    eu = rate * em / den + upd.abs() * (16 * U + 5 * U + 2.0 ** -72 / (bc2 * eps))
    ew = eu + 4 * U * (w.abs() + w1.abs())
    return w1, m1, v1, em, ev, ew


def param_bound(w, ew, dtype):
    """A parameter is its weight rounded to nearest: half a step of its type, or
    half of the smallest number."""
    if dtype == torch.float32:
        return ew
    f = torch.finfo(dtype)
    return ew + (w.abs() + ew) * (f.eps / 2) + f.smallest_normal * f.eps / 2


def check(got, want, bound, what):
    """Elementwise, with the worst excess in the message."""
    d = (got.double() - want).abs() - bound
    assert torch.isfinite(got.double()).all(), what
    assert (d <= 0).all(), f"{what}: over its bound by {d.max().item():.3g}"


def level(c, top, steps):
    """What code c stands for: c steps, `steps` an octave, below `top`, which is 1."""
    c = c.double()
    down = top - c
    octave = torch.ceil(down / steps)
    return torch.where(c > 0, torch.exp2(-octave) * (1 + (octave * steps - down) / steps),
                       torch.zeros_like(c))


def decode64(code_m, code_r, scales):
    blk = torch.arange(code_m.numel(), device=code_m.device) // 256
    m = level(code_m % 128, 127, 8) * scales.double()[blk, 0]
    return torch.where(code_m >= 128, -m, m), level(code_r, 255, 16) * scales.double()[blk, 1]
