"""The dense operators in 64 bits (torch, any device), and the bounds their kernels are held to.

u is half a step of the activations' type (2^-8 bf16, 2^-11 f16). A 4-bit product y = x W^T
may round each weight once (the tensor-core path: |dw| <= u |w|), accumulates K terms in fp32,
and rounds the result once:
    |dy| <= u |x| |W|^T + acc + u |y|,   acc = (K + 16) 2^-23 * |x| (|s| off + |b|)^T,
where off bounds the integers the small-batch path multiplies by (its weight fields are
offset by 128 in bf16, 1024 in f16), so that acc covers either path. f16 weights below 2^-14
are rounded to 2^-25 at worst; that adds 2^-25 |x|.
"""
from __future__ import annotations

import math

import torch

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
OFFSET = {torch.bfloat16: 144.0, torch.float16: 1040.0}
GELU_C = math.sqrt(2.0 / math.pi)


class QW:
    """A random packed matrix with zero points of its own per group."""

    def __init__(self, gen, rows, cols, group, dtype, biases=True, device="cpu", scale=0.02):
        self.group = group
        self.w = torch.randint(-2 ** 31, 2 ** 31, (rows, cols // 8), dtype=torch.int32, generator=gen).to(device)
        s = (torch.randn(rows, cols // group, generator=gen) * scale).abs() + 1e-3 * scale
        self.scales = s.to(dtype).to(device)
        z = 7.0 + 2.0 * torch.rand(rows, cols // group, generator=gen)
        self.biases = (-z * s).to(dtype).to(device) if biases else None

    def dense(self):
        """[rows, cols] float64."""
        q = torch.stack([(self.w >> (4 * i)) & 15 for i in range(8)], -1).reshape(self.w.shape[0], -1).double()
        w = q * self.scales.double().repeat_interleave(self.group, 1)
        return w if self.biases is None else w + self.biases.double().repeat_interleave(self.group, 1)

    def spread(self, off):
        """|s| off + |b| per element, float64."""
        m = self.scales.double().abs() * off
        if self.biases is not None:
            m = m + self.biases.double().abs()
        return m.repeat_interleave(self.group, 1)


def rand(gen, *shape, dtype, device="cpu"):
    return torch.randn(*shape, generator=gen).to(dtype).to(device)


def qmm(x, q, transpose=True):
    """(y, bound) of the 4-bit product."""
    x64, w = x.double(), q.dense()
    dt, K = x.dtype, x.shape[-1]
    s = q.spread(OFFSET[dt])
    if transpose:
        w, s = w.t(), s.t()
    y = x64 @ w
    bound = U[dt] * (x64.abs() @ w.abs()) + (K + 16) * 2.0 ** -23 * (x64.abs() @ s) + U[dt] * y.abs()
    if dt == torch.float16:
        bound = bound + 2.0 ** -25 * x64.abs().sum(-1, keepdim=True) + 2.0 ** -25
    return y, bound * (1 + 2 * U[dt])


def act(g, kind):
    """The activation and its derivative."""
    if kind == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    t = torch.tanh(GELU_C * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * GELU_C * (1 + 3 * 0.044715 * g * g)


def ffn(x, gate, up, down, kind, residual=None):
    wg, wu, wd = gate.dense(), up.dense(), down.dense()
    g, u = x.double() @ wg.t(), x.double() @ wu.t()
    y = (act(g, kind)[0] * u) @ wd.t()
    return (y if residual is None else y + residual.double()), g, u


def ffn_vjp(g, u, dy, gate, up, down, kind):
    """Gradients at the given g and u (float64)."""
    a, da = act(g, kind)
    dh = dy.double() @ down.dense()
    dg, du = dh * u * da, dh * a
    return dg @ gate.dense() + du @ up.dense(), dg, du


def rel(got, want):
    """2-norm of the difference over the 2-norm of the result."""
    return float((got.double() - want).norm() / want.norm())


def rope(x, dims, traditional=False, base=10000.0, scale=1.0, offset=0, freqs=None, mscale=1.0, inverse=False):
    """[B, H, L, D] in float64."""
    B, H, L, D = x.shape
    off = offset.double() if isinstance(offset, torch.Tensor) else torch.full((B,), float(offset), dtype=torch.float64)
    pos = off.to(x.device)[:, None] + torch.arange(L, device=x.device)
    i = torch.arange(0, dims, 2, dtype=torch.float64, device=x.device)
    wave = freqs.double() if freqs is not None else base ** (i / dims)
    ang = (pos * scale)[:, None, :, None] / wave
    if inverse:
        ang = -ang
    c, s, v = torch.cos(ang) * mscale, torch.sin(ang) * mscale, x[..., :dims].double()
    if traditional:
        a, b = v[..., 0::2], v[..., 1::2]
        r = torch.stack([a * c - b * s, a * s + b * c], -1).flatten(-2)
        big = torch.stack([a.abs() + b.abs()] * 2, -1).flatten(-2)
    else:
        a, b = v[..., :dims // 2], v[..., dims // 2:]
        r = torch.cat([a * c - b * s, a * s + b * c], -1)
        big = torch.cat([a.abs() + b.abs()] * 2, -1)
    tail = x[..., dims:].double()
    # cos and sin in fp32 (a few steps of 2^-24, the reduced angle's rounding among them), two
    # products and a sum in fp32, one rounding to the type
    bound = 8 * 2.0 ** -24 * abs(mscale) * big + U[x.dtype] * r.abs() * (1 + 2.0 ** -20)
    if x.dtype == torch.float16:
        bound = bound + 2.0 ** -25
    return torch.cat([r, tail], -1), torch.cat([bound, torch.zeros_like(tail)], -1)
