"""Elementwise bounds of the dense operators' kernels, tight enough that one wrong element shows.

u is half a step of the type (2^-8 bf16, 2^-11 f16), LAMBDA = 8. Roundings are taken as independent
with mean zero (the signs of the random operands make them so): a sum of terms t_k, each rounded
once, is off by more than LAMBDA u sqrt(sum t_k^2) with probability 2 exp(-LAMBDA^2 / 2) = 2.5e-14
(Hoeffding), 2e-6 over the 10^8 elements of these tests. That holds for the weights' rounding of the
tensor-core form and for roundings carried from one product into the next. The rest is counted at
its worst:
  sums in fp32. An MMA adds 16 products and the sum so far, each cut off at 2^-24 of the largest at
    worst: 17 2^-24 of the sum of magnitudes. Tensor cores: K / 16 of them, up to 8 splits of K and
    their operand pairs, on |x| |w|. Few tokens (M <= 32): up to 8 per group, then 3 operations for
    each of the K / G groups and 16 warps, on |x| (31 |s| + |b|), since its factors are 16 + q <= 31;
  the result's rounding, u |y|, and in f16 2^-25 for results (weights: LAMBDA 2^-25 sqrt(sum x^2))
    below the normal range.
"""
from __future__ import annotations

import torch

import dense_ref as R

LAMBDA = 8.0


def product(x, q, transpose=True, few=None):
    """(y, bound) of the 4-bit product in float64; x [M, K] as the kernel has it."""
    return sums([(x, q)], transpose, few)


def sums(pairs, transpose, few=None):
    """(y, bound) of a sum of 4-bit products with one rounding at its end."""
    y = var = mag = off = sub = 0.0
    dt = pairs[0][0].dtype
    K = pairs[0][0].shape[-1] * len(pairs)
    for x, q in pairs:
        x, w, s = x.double(), q.dense(), q.spread(31.0)
        if transpose:
            w, s = w.t(), s.t()
        y, var, mag = y + x @ w, var + x.square() @ w.square(), mag + x.abs() @ w.abs()
        if few if few is not None else (transpose and x.shape[0] <= 32):
            off = off + x.abs() @ s
        sub = sub + x.square().sum(-1, keepdim=True)
    u = R.U[dt]
    G = pairs[0][1].group
    acc = (17 * K / 16 + 16) * 2.0 ** -24 * mag + (17 * 8 + 3 * K / G + 16) * 2.0 ** -24 * off
    bound = LAMBDA * u * var.sqrt() + acc
    if dt == torch.float16:
        bound = bound + LAMBDA * 2.0 ** -25 * sub.sqrt() + 2.0 ** -25
    return y, bound * (1 + 2 * u) + u * y.abs()


def act_error(g, kind):
    """What the activation in fp32 may be off by, g float64. It is g sigmoid(z), z = g or
    2 GELU_C (g + 0.044715 g^3): z log2(e) takes up to 4 roundings, so that the exponential, and for
    z < 0 with it the result, is off by |z| 4 2^-24 relative, the hardware's base-2 exponential and
    reciprocal by 2^-22 each, the product by 2^-24. The 64-bit form's 0.5 g (1 + tanh) itself is off
    by 2^-53 |g| where tanh is near -1 (there its bound would otherwise be zero, and the kernel is
    the more exact of the two)."""
    z = g if kind == "silu" else 2 * R.GELU_C * (g + 0.044715 * g ** 3)
    return R.act(g, kind)[0].abs() * (z.abs() + 4) * 2.0 ** -22 + 2.0 ** -52 * g.abs()


def block(g, u, down, kind, residual=None, few=False):
    """(y, bound) of the block's output, given g and u as the kernel stored them. It forms h from the
    sums before their rounding (each off by up to u) and rounds it once; those errors pass through
    the down product."""
    dt, half = g.dtype, R.U[g.dtype]
    gd, ud = g.double(), u.double()
    a, da = R.act(gd, kind)
    h = a * ud
    # the slope at the unrounded g: |act''| < 1.13, which adds half |g| of it
    slope = da.abs() + 1.13 * half * gd.abs()
    eh = half * (slope * (gd * ud).abs() + h.abs() * (1 + half) + h.abs()) + act_error(gd, kind) * ud.abs()
    if dt == torch.float16:
        eh = eh + 2.0 ** -25
    y, bound = product(_As(h, dt), down, True, few)
    w2 = down.dense().square().t()
    bound = bound + LAMBDA * (eh.square() @ w2).sqrt() * (1 + 2 * half)
    if residual is not None:
        y2 = y + residual.double()
        bound, y = bound + half * (y2.abs() - y.abs()), y2
    return y, bound


def gradients(g, u, dy, gate, up, down, kind):
    """[(dg, bound), (du, bound)] at g and u as the kernel reads them."""
    half = R.U[g.dtype]
    gd, ud = g.double(), u.double()
    a, da = R.act(gd, kind)
    dh, b = product(dy, down, transpose=False)
    b = b - half * dh.abs()  # dh itself is not rounded
    out = []
    for f, err in ((ud * da, 2.0 ** -20 * (1 + gd.abs()) * ud.abs()), (a, act_error(gd, kind))):
        v = dh * f
        e = (b * f.abs() + err * (dh.abs() + b)) * (1 + half) + half * v.abs()
        out.append((v, e + 2.0 ** -25 if g.dtype == torch.float16 else e))
    return out


class _As:
    """float64 values that stand for a tensor of another type."""

    def __init__(self, t, dtype):
        self.t, self.dtype, self.shape = t, dtype, t.shape

    def double(self):
        return self.t
