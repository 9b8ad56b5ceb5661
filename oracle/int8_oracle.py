"""Eight-bit Linear layers from their definition, in float64 on the CPU, with the bound of the f32 epilogue."""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def quantize_rows(x: torch.Tensor):
    """(q f64, scale f64): the scale is the f32 nearest to max|x| / 127 and at least 2^-126.  The division of two f32
    values in 64 bits keeps them on the right side of every border between two steps: x and (k + 1/2) s differ by at
    least 2^-33 relative where they differ (24 and 32 bits), the quotient is off by 2^-53."""
    x = x.double()
    bad = ~torch.isfinite(x).all(1)
    amax = torch.where(bad, 1.0, x.abs().amax(1))
    s = (amax.float() / 127.0).clamp_min(torch.finfo(torch.float32).tiny).double()
    q = torch.round(x / s[:, None]).clamp(-127, 127)
    q[bad] = 0.0
    s[bad] = math.nan
    return q, s


def linear(x, weight, weight_scale, bias=None, out_dtype=None):
    """(y f64, bound).  Epilogue: the integer sum to f32, times the token's scale, times the channel's, plus the bias: three
    roundings of the product and one of the result, then the output type."""
    q, s = quantize_rows(x)
    prod = (q @ weight.double().t()) * s[:, None] * weight_scale.double()[None, :]
    y = prod if bias is None else prod + bias.double()
    tol = 3 * U * prod.abs() + U * y.abs() + 2.0 ** -126   # (the token's part alone may fall below the normal range)
    half = torch.finfo(out_dtype or x.dtype).eps / 2
    return y, tol + half * (y.abs() + tol)
