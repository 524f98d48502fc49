"""Plain 64-bit forms of the attention operators, and how far a kernel may be from them."""
from __future__ import annotations

import math

import torch


def attend(q, k, v, scale, limit=None):
    """One sequence: q [n, Hq, D], k / v [m, Hkv, D] -> (out, A, slack, P) in float64.

    ``limit [n]``: the keys each query sees, default bottom-right causal.  A = sum_j p_j |v_j|
    (what a relative error of the terms scales with); ``slack`` bounds the relative error
    that fp32 scores put into a term; P [n, Hq, m] the weights."""
    n, m = q.shape[0], k.shape[0]
    G = q.shape[1] // k.shape[1]
    q, k, v = (x.detach().double().cpu() for x in (q, k, v))
    if limit is None:
        limit = torch.arange(n) + (m - n) + 1
    seen = torch.arange(m)[None] < limit[:, None]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    s = torch.einsum("ihd,jhd->ihj", q, k) * scale
    s = torch.where(seen[:, None], s, torch.full_like(s, -math.inf))
    top = s.amax(-1, keepdim=True) if m else torch.full((n, q.shape[1], 1), -math.inf).double()
    p = torch.exp(s - torch.where(top == -math.inf, torch.zeros_like(top), top))
    p = torch.where(seen[:, None], p, torch.zeros_like(p))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    # (what is not seen has no part, also where it is not finite)
    vv = torch.where(torch.isfinite(v), v, torch.zeros_like(v))
    out = torch.einsum("ihj,jhd->ihd", p, vv)
    A = torch.einsum("ihj,jhd->ihd", p, vv.abs())
    mag = torch.einsum("ihd,jhd->ihj", q.abs(), k.abs()) * scale
    mag = torch.where(seen[:, None], mag, torch.zeros_like(mag))
    D = q.shape[2]
    # a score is a sum of D exact (16-bit types) or rounded (fp32) products in fp32, then
    # scaled by a rounded constant and subtracted from the maximum: |ds| <= (D + 6) 2^-24 mag;
    # the exponential adds 2 ulp, the sums over the keys 2^-24 each
    ds = (D + 6) * 2.0 ** -24 * (mag.amax(-1) if m else torch.zeros(n, q.shape[1]).double())
    slack = 2 * ds + 2.0 ** -21 + 2 * m * 2.0 ** -24
    return out, A, slack[..., None], p


def bound(dtype, out, A, slack):
    """|error| of one element: a rounding of every probability to the type (16-bit types: half
    an eps of each term of A), the scores' and sums' fp32 error on the terms, and the
    rounding of the result (with the smallest subnormal of the type)."""
    half = torch.finfo(dtype).eps / 2
    term = half if dtype != torch.float32 else 0.0
    # p below the type's normal numbers: fp16 probabilities (at most 1 relative to a maximum
    # that may lag by 2^8) lose at most half a subnormal step each
    tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
    return A * (term + slack) * (1 + slack) + (out.abs() + A * (term + slack)) * half + tiny


def check(got, want, dtype, what):
    out, A, slack = want[:3]
    got = got.detach().double().cpu()
    assert torch.isfinite(got).all(), f"{what}: not finite"
    room = bound(dtype, out, A, slack)
    over = ((got - out).abs() / room.clamp_min(1e-300)).max().item() if got.numel() else 0.0
    assert over <= 1.0, f"{what}: {over:.3g} times the bound"
