"""64-bit statements of the answer scores and the distillation loss, with the error bounds of an f32 evaluation.

Everything is computed on the CPU in float64 from the definitions; bounds are returned beside the values.  The bounds
count roundings for arithmetic in units u = 2^-24 (half an f32 step, relative):

  exponent   t = (x - m) log2(e) / T: the difference (1 u |t|), the product (1 u |t|): an error of 2 |t| u in t is one of
             2 ln2 |t| u < 2 |t| u in e = 2^t; the hardware exponential adds one step, 2 u
  sums       up to eight f32 additions in a row for S (8 u), the rest in f64; so S is off by at most (2 E|t| + 10) u,
             relative, with E|t| the mean of |t| under p; sum e t: a product, up to 16 additions in a row and six levels
             over a wave
  logarithm  of the sum as f32: one step of the result, 2 u |log S|
  products   u each
  underflow  the hardware exponential gives 0 below 2^-126, so e (and p = e / S, S >= 1) may be off by 2^-126 absolutely;
             a gradient multiplies that by the factor that p has in it
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24
FLUSH = 2.0 ** -126


def _half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def _tiny(dtype: torch.dtype) -> float:
    """An absolute allowance for results below the normal range."""
    return 2 * torch.finfo(dtype).tiny


def distribution(logits: torch.Tensor, temperature: float):
    """(m, log p (R,C), p, |t|, empty, broken) in f64."""
    x = logits.double()
    m = torch.where(torch.isnan(x), -math.inf, x).amax(1, keepdim=True)
    broken = (torch.isnan(x) | (x == math.inf)).any(1)
    empty = (m[:, 0] == -math.inf) & ~broken
    z = (x - m) / temperature
    z = torch.where(empty[:, None], 0.0, z)
    s = torch.exp(z).sum(1, keepdim=True)
    lp = z - torch.log(s)
    lp[broken] = math.nan
    p = torch.exp(lp)
    t = torch.where(p > 0, z.abs() / math.log(2.0), 0.0)
    lp[empty] = -math.inf
    p[empty] = 0.0
    return m, lp, p, t, empty, broken


def sum_bound(p, t):
    """Relative bound of S, an absolute one of log S (the logarithm's own step included)."""
    log_s = -torch.log(p.amax(1).clamp_min(1e-300))   # the largest term of S is 1
    return (2 * (p * t).sum(1) + 10 + 2 * log_s) * U


def entropy(lp, p):
    return -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(1) + torch.where(torch.isnan(p).any(1), math.nan, 0.0)


def entropy_bound(h, p, t):
    """H = log S - ln2 W / S, W = sum e t: each term e t is off by (2 |t| + 2 + 2) u relative, the sums add 22 u, the
    quotient and its factor 4 u."""
    w = (p * t * (2 * t + 30)).sum(1) * math.log(2.0) * U
    return sum_bound(p, t) * (1 + math.log(2.0) * (p * t).sum(1)) + w + 2 * U * h.abs() + 4 * U


def order(logits: torch.Tensor, top: int) -> torch.Tensor:
    """Indices of the `top` largest, ties by the lowest index, NaN above everything."""
    x = logits.double() + 0.0
    x = torch.where(torch.isnan(x), torch.full_like(x, math.inf), x)
    first = torch.isnan(logits)
    # two stable sorts: by value, then NaN before the rest
    idx = torch.sort(x, dim=1, descending=True, stable=True).indices
    nan = torch.take_along_dim(first, idx, 1).to(torch.int8)
    again = torch.sort(nan, dim=1, descending=True, stable=True).indices
    return torch.take_along_dim(idx, again, 1)[:, :top]


def _f32_range(v):
    """What lies past the f32 range is infinite in an f32 result."""
    return torch.where(v < -torch.finfo(torch.float32).max, -math.inf, v)


def token_logprobs(logits, targets=None, top=0, temperature=1.0):
    """dict of values and of "<name>_tol" bounds."""
    m, lp, p, t, empty, broken = distribution(logits, temperature)
    C = logits.shape[1]
    tol = sum_bound(p, t)[:, None]
    out = {"entropy": torch.where(empty, 0.0, entropy(lp, p))}
    out["entropy_tol"] = entropy_bound(out["entropy"], p, t)
    if targets is not None:
        tg = targets.reshape(logits.shape[0], -1)
        v = torch.take_along_dim(lp, tg.clamp(0, C - 1), 1)
        v = torch.where(tg < 0, 0.0, torch.where(tg >= C, math.nan, v))
        v = _f32_range(v)
        out["logprobs"], out["logprobs_tol"] = v, tol + 2 * U * v.abs()
    if top:
        out["top_indices"] = order(logits, top)
        v = _f32_range(torch.take_along_dim(lp, out["top_indices"], 1))
        out["top_logprobs"], out["top_logprobs_tol"] = v, tol + 2 * U * v.abs()
    return out


def token_logprobs_grad(logits, temperature, targets=None, g_logprobs=None, g_entropy=None, top_indices=None, g_top=None):
    """(gradient, bound) of sum(g_logprobs logprobs) + sum(g_entropy entropy) + sum(g_top top_logprobs)."""
    m, lp, p, t, empty, broken = distribution(logits, temperature)
    R, C = logits.shape
    g, size = torch.zeros(R, C, dtype=torch.float64), torch.zeros(R, C, dtype=torch.float64)
    a, amag = torch.zeros(R, dtype=torch.float64), torch.zeros(R, dtype=torch.float64)
    for idx, up in ((targets, g_logprobs), (top_indices, g_top)):
        if up is None:
            continue
        idx, up = idx.reshape(R, -1), up.double().reshape(R, -1)
        live = idx >= 0
        up = torch.where(live, up, 0.0)
        up = torch.where(idx >= C, math.nan, up)
        a, amag = a + up.sum(1), amag + up.abs().sum(1)
        at = torch.where(live & (idx < C), idx, 0)
        add = torch.where(live & (idx < C), up, 0.0)
        g.scatter_add_(1, at, add)
        size.scatter_add_(1, at, add.abs())
    h = torch.zeros(R, dtype=torch.float64) if g_entropy is None else g_entropy.double()
    H = torch.where(empty, 0.0, entropy(lp, p))
    lpf = torch.where(p > 0, lp, 0.0)
    g = g - p * (a[:, None] + h[:, None] * (lpf + H[:, None]))
    mag = p * (amag[:, None] + h.abs()[:, None] * (lpf.abs() + H.abs()[:, None]))
    # p is off by (2|t| + 2 + 2) u plus S's bound; log p by 2 |t| u (its own exponent) plus S's bound and 2 u of log S;
    # H comes as the f32 that the forward returned; six more products, sums and the roundings of A
    S = sum_bound(p, t)[:, None]
    tol = mag * ((2 * t + 14) * U + S)
    tol = tol + p * h.abs()[:, None] * (2 * t * U + S + 3 * U * lpf.abs() + entropy_bound(H, p, t)[:, None])
    tol = tol + size * 160 * U   # up to 128 + 32 terms added one by one
    tol = tol + FLUSH * (amag[:, None] + h.abs()[:, None] * (torch.where(lp > -math.inf, lp, 0.0).abs() + H.abs()[:, None]))
    g, tol = g / temperature, tol / temperature + 4 * U * (g / temperature).abs()
    g[empty] = 0.0
    tol[empty] = 0.0
    g[broken] = math.nan
    return g, tol + _half_step(logits.dtype) * (g.abs() + tol) + _tiny(logits.dtype)


def distill(logits, teacher, indices, temperature=1.0, tail=False):
    """(row losses, bounds, gradient of their sum, bounds); rows in f64."""
    m, lp, p, t, empty, broken = distribution(logits, temperature)
    R, C = logits.shape
    live = (indices >= 0) & (indices < C)
    beyond = (indices >= C).any(1)
    v = torch.where(live, teacher.double(), -math.inf)
    if not tail:
        top = v.amax(1, keepdim=True)
        v = v - torch.where(top == -math.inf, 0.0, torch.logsumexp(v, 1, keepdim=True))
    q = torch.exp(v)
    at = torch.where(live, indices, 0)
    target = torch.zeros(R, C, dtype=torch.float64).scatter_add_(1, at, q)
    lpk = torch.take_along_dim(lp, at, 1)
    loss = torch.where(q > 0, q * (v - lpk), 0.0).sum(1)
    mass = q.sum(1)
    rest = torch.zeros(R, dtype=torch.float64)
    outside = torch.ones(R, C, dtype=torch.float64)
    outside = torch.where(torch.zeros(R, C, dtype=torch.float64).scatter_add_(1, at, live.double()) > 0, 0.0, outside)
    shared = torch.zeros(R, C, dtype=torch.float64)   # rest times each class's share of what the list leaves
    t_out, held_bound = t, torch.zeros(R, dtype=torch.float64)
    if tail:
        rest = 1.0 - mass
        some = (rest > 2.0 ** -20) & (outside.sum(1) > 0) & live.any(1)
        rest = torch.where(some, rest, 0.0)
        # relative to their own maximum, and in logarithms: what the student leaves outside the list may lie below every
        # number
        x = logits.double()
        xo = torch.where(outside > 0, x, -math.inf)
        mo = torch.where(torch.isnan(xo), -math.inf, xo).amax(1, keepdim=True)
        zo = (xo - torch.where(mo == -math.inf, 0.0, mo)) / temperature
        so = torch.exp(zo).sum(1, keepdim=True)
        share = torch.where(so > 0, torch.exp(zo) / so, 0.0)
        held = (mo - m)[:, 0] / temperature + torch.log(so[:, 0]) + lp.amax(1)   # (the largest is -log S)
        t_out = torch.where(share > 0, zo.abs() / math.log(2.0), 0.0)
        held_bound = (2 * (share * t_out).sum(1) + 10) * U
        loss = loss + torch.where(some, rest * (torch.log(rest) - held), 0.0)
        shared = rest[:, None] * share
    total = mass + rest
    g = p * total[:, None] - shared - target
    tol_s = sum_bound(p, t)
    loss_tol = total * tol_s + rest * (held_bound + tol_s) + 2.0 ** -36 * (1 + (q * v.clamp_min(-1e3).abs()).sum(1))
    # rounding to f32 once, and the f32 of a row that a mean reads
    t2 = temperature * temperature
    loss, loss_tol = loss * t2, loss_tol * t2 + 2 * U * (loss * t2).abs()
    loss = torch.where(loss > torch.finfo(torch.float32).max, math.inf, loss)
    # on the list, or without a tail: p as above, mass to f32; q to f32, summed where an answer is named again, subtracted,
    # scaled
    off = outside if tail else torch.zeros_like(outside)
    tol = (1.0 - off) * p * total[:, None] * ((2 * t + 10) * U + tol_s[:, None]) + target * 140 * U
    # elsewhere one exponential times one factor, the difference of the two parts' factors, formed in 64 bits: the
    # exponential is off by its argument's difference, factor and product, 3 ln2 |t| u (2 |t| u and, as it is 0 past
    # |t| = 126, another 10 u), the factor by what its two sums are, and as f32
    tol = tol + off * ((p * total[:, None] - shared).abs() * (2 * t_out + 20) * U
                       + (p * total[:, None]) * (tol_s + 2 * U)[:, None] + shared * (held_bound + 2 * U)[:, None])
    tol = tol + FLUSH * (total + rest)[:, None]
    g, tol = g * temperature, tol * temperature + 4 * U * (g * temperature).abs()
    none = ~live.any(1)
    loss, loss_tol = torch.where(none, 0.0, loss), torch.where(none, 0.0, loss_tol)
    loss = torch.where(empty & (total > 0) & ~none, math.inf, loss)
    for bad in (beyond, broken & ~none):
        loss = torch.where(bad, math.nan, loss)
    zero = empty | none
    g[zero], tol[zero] = 0.0, 0.0
    g[beyond] = math.nan
    g[broken & ~none] = math.nan
    return loss, loss_tol, g, tol
