"""Rotary positions of queries and keys on MI355X, alone (``rotary``) or behind a norm of each head in the same pass (``qk_norm_rotary``),
both with their backward.  The scan's C and B are its queries and keys, (batch, seqlen, ngroups, dstate): they are turned as they lie.
Checks, argument blocks, allocation and the autograd node are compiled (csrc/host_ops.cpp); all arithmetic runs in libissm_hip.so."""
from __future__ import annotations

import math

import torch

from . import _lib as L


def rotary_table(length, dim, base=10000.0, scaling=None, factor=1.0, original_length=None, beta_fast=32.0, beta_slow=1.0, device="cuda"):
    """(length, dim) fp32: for each position the cosines of its dim / 2 angles, then their sines.  Angles are position * base ** (-2 j / dim),
    computed in 64 bits.  For contexts longer than a model was trained for (`factor` times `original_length`):

    * scaling="linear": positions are divided by factor
    * scaling="base": the base grows so that the slowest angle is divided by factor and the fastest stays
    * scaling="parts": angles that turn more than beta_fast times within original_length stay, those that turn fewer than beta_slow times
      are divided by factor, with a ramp between them; cosines and sines are scaled by 0.1 log(factor) + 1
    """
    if length < 1 or dim < 2 or dim % 2:
        raise ValueError(f"a table of {length} positions and {dim} features: at least one, and an even number")
    if not (base > 1.0 and factor >= 1.0):
        raise ValueError(f"base {base} has to be above 1 and factor {factor} at least 1")
    if scaling not in (None, "linear", "base", "parts"):
        raise ValueError(f"scaling {scaling!r}: None, 'linear', 'base' or 'parts'")
    j = torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim
    if scaling == "base":
        base = base * factor ** (dim / max(dim - 2, 1))
    speed, size = torch.pow(torch.full_like(j, base), -j), 1.0
    if scaling == "linear":
        speed = speed / factor
    elif scaling == "parts":
        if original_length is None or original_length < 1 or not beta_fast > beta_slow > 0:
            raise ValueError("scaling='parts' takes original_length, and beta_fast > beta_slow > 0")
        # the ramp is linear in the angle's index; the angle that turns n times has the index at which base ** (-2 j / dim) is 2 pi n / original_length
        at = [dim * math.log(original_length / (2 * math.pi * n)) / (2 * math.log(base)) for n in (beta_fast, beta_slow)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), dim - 1)
        ramp = ((torch.arange(dim // 2, device=device, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0.0, 1.0)
        speed = speed * (1.0 - ramp) + speed / factor * ramp
        size = 0.1 * math.log(factor) + 1.0
    angle = torch.arange(length, device=device, dtype=torch.float64)[:, None] * speed
    return torch.cat([size * angle.cos(), size * angle.sin()], dim=1).float()


def rotary(q, k, table, positions=None, interleaved=False):
    """
    Argument:
        q: (batch, seqlen, heads, headdim), k: (batch, seqlen, kv_heads, headdim) or None; features contiguous, other strides as they are.
            headdim up to 1024, batch * seqlen * (heads + kv_heads) below 2^31, heads + kv_heads up to 2^20.
            bfloat16 where both are, else computed in float32; each is returned in its own type
        table: (rows, rot) of rotary_table; the first rot <= headdim features of a head are turned, the others returned as they are
        positions: (batch, seqlen) or (seqlen,) int32 or int64, rows of the table, or None: 0, 1, ... along the sequence.  A position
            outside the table makes its token's turned features NaN.
        interleaved: pairs of features (2j, 2j + 1) instead of (j, j + rot / 2)
    Return:
        the turned q and k (q alone where k is None)
    """
    res = L.host().rotary(q, k, None, None, table, positions, 0.0, bool(interleaved))
    return (res[0], res[1]) if k is not None else res[0]


def qk_norm_rotary(q, k, q_weight, k_weight, table, positions=None, eps=1e-6, interleaved=False):
    """rotary(q / rms(q) * q_weight, k / rms(k) * k_weight) with rms over each head's features, sqrt(mean(x^2) + eps), in one pass.
    q_weight, k_weight: (headdim,), k and k_weight may be None.  First derivatives for q, k, q_weight and k_weight."""
    if q_weight is None or (k is None) != (k_weight is None):
        raise ValueError("qk_norm_rotary takes q_weight, and k_weight where there is a k")
    res = L.host().rotary(q, k, q_weight, k_weight, table, positions, float(eps), bool(interleaved))
    return (res[0], res[1]) if k is not None else res[0]
