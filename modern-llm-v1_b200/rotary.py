"""Rotary positions in other layouts for q and k, forward and backward (csrc/rotary.cuh).

rope_norm.py has the reference's one form (all of a head, neighbouring pairs, the token's index, the norm always).  Models trained
elsewhere differ: pairs of the head's halves, only part of the head, positions of their own per token (padded or packed batches),
no QK-norm, and frequencies scaled for contexts longer than those trained on.  A QK-norm is behind the rotation, as the reference has it;
a model with the norm in front of it (and a gamma that differs within a pair) normalises first and passes no gammas here.  The caller allocates every tensor; outputs are
overwritten except ``d_gamma_*``, which are accumulated into as in rope_qknorm_backward.  Bad arguments raise ValueError, CUDA
failures RuntimeError; there is no CPU or PyTorch fallback.
"""
from __future__ import annotations

import torch

from . import _lib


def make_rotary_cache(T_max, rotary_dim, base=10000.0, scaling="none", factor=1.0, trained=None, turns_fast=32.0, turns_slow=1.0,
                      device="cuda"):
    """cos, sin [T_max, rotary_dim / 2] FP32 on `device`, from angles in 64 bits: position * base^(-2i / rotary_dim), scaled by

    "linear"  every frequency divided by `factor`
    "base"    the base grown so that the slowest pair is slowed by `factor` and the fastest not at all
    "parts"   pairs that turn more than `turns_fast` times within `trained` positions kept, those that turn less than
              `turns_slow` times divided by `factor`, those between in proportion

    (A sharper softmax that goes with a scaling is the caller's softmax_scale.)"""
    if scaling not in _lib.SCALINGS:
        raise ValueError("make_rotary_cache: scaling must be one of " + ", ".join(_lib.SCALINGS))
    if T_max <= 0 or rotary_dim <= 0 or rotary_dim % 2 != 0:
        raise ValueError("make_rotary_cache: T_max must be positive and rotary_dim even")
    if scaling == "parts" and trained is None:
        raise ValueError("make_rotary_cache: trained is needed to scale by parts")
    cos = torch.empty((T_max, rotary_dim // 2), dtype=torch.float32, device=device)
    sin = torch.empty_like(cos)
    _lib.host().rotary_table(T_max, rotary_dim, float(base), _lib.SCALINGS[scaling], float(factor), float(trained or 0.0), float(turns_fast),
                             float(turns_slow), cos, sin)
    return cos, sin


def rotary_forward(xq, xk, cos, sin, gamma_q, gamma_k, eps, yq, yk, rstd_q, rstd_k, B, T, Hq, Hkv, D, rotary_dim, pairs="interleaved",
                   positions=None, x_layout="BTHD", y_layout="BHTD"):
    """yq, yk (BF16 in y_layout, ready for flash_attn_forward_gqa) = q and k (BF16 or FP32 in x_layout) with the first rotary_dim
    elements of every head rotated, in "interleaved" pairs (x[2i], x[2i+1]) or "half" ones (x[i], x[i + rotary_dim / 2]).  positions:
    [B, T] int32 rows of cos and sin [n, rotary_dim / 2], or None for 0 .. T-1; a token whose position is no row of the tables is
    skipped and reported by device_status.  With gamma_q, gamma_k (FP32 [D]) each row is normalised behind the rotation and 1 / rms
    goes to rstd_q, rstd_k (FP32 [B, H, T]); without them (None) all four are None."""
    _lib.host().rotary_fwd(xq, xk, cos, sin, gamma_q, gamma_k, eps, yq, yk, rstd_q, rstd_k, B, T, Hq, Hkv, D, rotary_dim, pairs, positions,
                           x_layout, y_layout)


def rotary_backward(d_yq, d_yk, xq, xk, cos, sin, gamma_q, gamma_k, rstd_q, rstd_k, d_xq, d_xk, d_gamma_q, d_gamma_k, B, T, Hq, Hkv, D,
                    rotary_dim, pairs="interleaved", positions=None, x_layout="BTHD", y_layout="BHTD"):
    """d_xq, d_xk (BF16 or FP32 in x_layout, overwritten) from d_yq, d_yk (BF16 in y_layout); with the norm also d_gamma_q, d_gamma_k
    (FP32 [D], accumulated into) from the forward's inputs and rstd.  Without it xq, xk, gammas, rstds and d_gammas are None (xq and xk
    may be given and are not read)."""
    _lib.host().rotary_bwd(d_yq, d_yk, xq, xk, cos, sin, gamma_q, gamma_k, rstd_q, rstd_k, d_xq, d_xk, d_gamma_q, d_gamma_k, B, T, Hq, Hkv,
                           D, rotary_dim, pairs, positions, x_layout, y_layout)
