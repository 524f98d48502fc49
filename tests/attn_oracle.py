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


def quantise(x):
    """x [..., D] of a 16-bit type -> (codes, scale, least) in float64, [..., D / 64, 64] and
    [..., D / 64]: by counting the borders that a value is above (exact in 64 bits)."""
    dt = x.dtype
    g = x.detach().cpu().double().unflatten(-1, (-1, 64))
    least = g.amin(-1)
    scale = ((g.amax(-1) - least) / 15).float().to(dt).double()
    codes = torch.zeros_like(g)
    twice = 2 * (g - least[..., None])
    for j in range(15):
        border = (2 * j + 1) * scale[..., None]
        codes += ((twice > border) | ((twice == border) & (j % 2 == 1))).double()
    codes = torch.where(scale[..., None] > 0, codes, torch.zeros_like(codes))
    bad = ~torch.isfinite(g).all(-1)
    return codes, torch.where(bad, torch.zeros_like(scale), scale), torch.where(bad, torch.full_like(least, math.nan), least)


def values(q):
    codes, scale, least = q
    return (codes * scale[..., None] + least[..., None]).flatten(-2)


def kv4_attend(q, kq, vq, scale):
    """One sequence over quantised keys and values (quantise()'s triples of [m, Hkv, D]):
    (out, A, slack, P) as :func:`attend`, with A and the scores' magnitude as the kernel's
    sums have them: products on 1 + n / 16 times 16, scales and least values apart."""
    out, _, _, p = attend(q, values(kq), values(vq), scale)
    n, Hq, D = q.shape
    G = Hq // kq[0].shape[1]
    grow = lambda t: torch.nan_to_num(t).repeat_interleave(G, 1)
    cod, sc, le = (grow(t) for t in vq)
    A = torch.einsum("ihj,jhd->ihd", p, ((cod + 16) * sc[..., None] * 2 + le.abs()[..., None]).flatten(-2))
    cod, sc, le = (grow(t) for t in kq)
    size = ((cod + 16) * sc[..., None] * 2 + le.abs()[..., None]).flatten(-2)
    mag = torch.einsum("ihd,jhd->ihj", q.detach().cpu().double().abs(), size) * scale
    mag = torch.where(p > 0, mag, torch.zeros_like(mag))
    ds = (D + 6) * 2.0 ** -24 * (mag.amax(-1) if mag.shape[-1] else torch.zeros(n, Hq).double())
    slack = 2 * ds + 2.0 ** -21 + 2 * p.shape[-1] * 2.0 ** -24
    # (slack relative to A; the probability times the scale is what is rounded: half an eps of
    # p * s * n, which A is at least twice of)
    return out, A, slack[..., None], p
