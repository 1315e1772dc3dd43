"""Rotary positions in 64 bits, for the tests (not collected)."""
import torch


def rotate(x, cos, sin, R, pairs, back=False):
    """x [..., T, D] float64; cos, sin broadcast to [..., T, R / 2]"""
    one, two = (slice(0, R, 2), slice(1, R, 2)) if pairs == "interleaved" else (slice(0, R // 2), slice(R // 2, R))
    s = -sin if back else sin
    a, b = x[..., one], x[..., two]
    out = x.clone()
    out[..., one] = a * cos - b * s
    out[..., two] = a * s + b * cos
    return out


def forward(x, gamma, cos, sin, R, pairs, eps):
    """x [B, H, T, D]; gamma [D] or None -> y, rstd or None"""
    r = rotate(x, cos, sin, R, pairs)
    if gamma is None:
        return r, None
    rstd = (r.square().mean(-1) + eps).rsqrt()
    return r * rstd[..., None] * gamma, rstd


def tables(cos, sin, positions, T):
    """[B or 1, 1, T, R / 2] float64 on the CPU"""
    c, s = cos.double().cpu(), sin.double().cpu()
    if positions is None:
        return c[None, None, :T], s[None, None, :T]
    at = positions.long().cpu()
    return c[at][:, None], s[at][:, None]
