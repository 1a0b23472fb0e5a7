"""Float64 restatement of what a decoder block computes around its attention (test infrastructure
only), from the definitions in ``include/dsalt_b200.h``: the 8-bit form of activations, the norm and
rotation of heads, the gated feed-forward block, and their gradients."""
from __future__ import annotations

import math

import torch

GROUP = 32


# --------------------------------------------------------------------------- 8 bits
def pack(x):
    """``(codes, exps)`` of ``x [rows, n]`` (float64 holding values of the input type)."""
    rows, n = x.shape
    groups = -(-n // GROUP)
    b = torch.cat([x, x.new_zeros(rows, groups * GROUP - n)], 1).view(rows, groups, GROUP)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    # exponent field of the largest magnitude as fp32 (0 below the normal range)
    field = torch.where(bad, top.new_zeros(()), top).float().view(torch.int32) >> 23
    s = (field - 6).clamp(min=1)
    step = torch.exp2((s - 127).double())[..., None]
    codes = torch.round(torch.where(bad[..., None], b.new_zeros(()), b) / step).clamp(-127, 127)
    s = torch.where(bad, torch.full_like(s, 255), s)
    return codes.view(rows, -1)[:, :n].to(torch.int8), s.to(torch.uint8)


def unpack(codes, exps):
    scale = torch.exp2(exps.double() - 127)
    scale = torch.where(exps == 255, torch.full_like(scale, math.nan), scale)
    return codes.double() * scale.repeat_interleave(GROUP, 1)[:, :codes.shape[1]]


def held(x):
    return unpack(*pack(x))


# --------------------------------------------------------------------------- heads
def rope(x, w, cos, sin, eps):
    """``x [T, H, D]``, ``cos, sin [T, D/2]``; ``w [D]`` or None."""
    half = x.shape[-1] // 2
    n = x if w is None else w * x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    a, b, c, s = n[..., :half], n[..., half:], cos[:, None], sin[:, None]
    return torch.cat([a * c - b * s, b * c + a * s], -1)


def rope_grad(x, w, cos, sin, eps, d):
    """``(dx, dw)`` for the output's gradient ``d``."""
    half = x.shape[-1] // 2
    a, b, c, s = d[..., :half], d[..., half:], cos[:, None], sin[:, None]
    dn = torch.cat([a * c + b * s, b * c - a * s], -1)
    if w is None:
        return dn, None
    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    xr = x * r
    dw = (dn * xr).sum((0, 1))
    dn = dn * w
    return r * (dn - xr * (dn * xr).mean(-1, keepdim=True)), dw


# --------------------------------------------------------------------------- feed-forward
def share(g, act):
    """``(p, p')`` with ``act(g) = g p(g)``."""
    if act == "silu":
        p = torch.sigmoid(g)
        return p, p * (1 - p)
    return 0.5 * torch.erfc(-g / math.sqrt(2.0)), torch.exp(-0.5 * g * g) / math.sqrt(2 * math.pi)


def ffn(x, wg, wu, wd, act):
    g, u = x @ wg.T, x @ wu.T
    return (g * share(g, act)[0] * u) @ wd.T


def ffn_grad(x, wg, wu, wd, act, dy, g=None, u=None):
    """``(dx, dwg, dwu, dwd)``; ``g`` and ``u`` (and ``x`` in the weights' gradients) as they were held."""
    if g is None:
        g, u = x @ wg.T, x @ wu.T
    p, dp = share(g, act)
    dh = dy @ wd
    dg, du = dh * u * (p + g * dp), dh * g * p
    return dg @ wg + du @ wu, dg.T @ x, du.T @ x, dy.T @ (g * p * u)
