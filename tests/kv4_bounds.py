"""Decode attention over stored codes in 64 bits, and how far the kernel's sums can be from it.

The kernel's arithmetic, of which every rounding is counted (u = 2^-24; sums inside the matrix
cores with 2 u an addition, whatever their order and rounding):

* scores, times log2(e) (c = scale log2(e), Q_g = sum of q over group g):
      x_j = sum_g 16 s_g c (sum_d q_d (1 + n_d / 16) - Q_g) + c m_g Q_g
  products exact, 65 additions a group, Q_g by 64 more, a few roundings of the factors:
      |dx_j| <= 2 u c sum_g sum_d |q_d| (16 s_g 70 (2.5 + n_d / 16) + 40 |m_g|)
* p_j = 2^(x_j - max): e_j = |dp_j| / p_j <= ln 2 (|dx_j| + 2 u (|x_j| + |x_j - max|)) + 2^-18
  (the last for the exponential and a dozen factors of new maxima and joins).  The sum of the
  weights has the same p_j in it: together they move the result by at most
      sum_j P_j e_j (|v_j| + |out|)
* p_j s_j in bf16 (half an eps: 2^-8), or as two bf16 terms where the tensors are fp16 (2^-16),
  times |n_j - 8|, as codes are taken relative to 8
* sums over the keys: C additions a chain (32 a chunk of 32 keys, a chunk a step of 128 keys and
  wave, at most 8 steps a part, then the waves and the parts) of terms of 16 s_j (1 + n_j / 16),
  their 1.5 times for the ones, middle values m_j + 8 s_j, and weights:
      2 u C (sum_j P_j (16 s_j (2.5 + n_j / 16) + |m_j + 8 s_j|) + |out|)
* the result rounded to its type
"""
from __future__ import annotations

import math

import torch

U = 2.0 ** -24


def grow(triple, G):
    """Codes [m, H, D / 64, 64] and scale, least [m, H, D / 64, 1] of every query head."""
    codes, scale, least = triple
    return [x.repeat_interleave(G, 1) for x in (codes, scale[..., None], least[..., None])]


def weights(q, kq, scale, limit=None):
    """P [n, Hq, m] and e [n, Hq, m] (module docstring) of one sequence: q [n, Hq, D], kq the
    triple of quantise() for [m, Hkv, D]; limit [n]: the keys each query sees."""
    n, Hq, D = q.shape
    m, Hkv = kq[0].shape[:2]
    codes, s, least = grow(kq, Hq // Hkv)
    q = q.detach().double().cpu()
    if limit is None:
        limit = torch.arange(n) + (m - n) + 1
    seen = (torch.arange(m)[None] < limit[:, None])[:, None]
    c = scale * math.log2(math.e)
    x = torch.einsum("ihd,jhd->ihj", q, (codes * s + least).flatten(-2)) * c
    x = torch.where(seen, x, torch.full_like(x, -math.inf))
    top = x.amax(-1, keepdim=True) if m else torch.zeros(n, Hq, 1).double()
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = torch.exp2(x - top)
    P = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    size = (16 * s * 70 * (2.5 + codes / 16) + 40 * least.abs()).flatten(-2)
    dx = 2 * U * c * torch.einsum("ihd,jhd->ihj", q.abs(), size)
    x = torch.where(seen, x, torch.zeros_like(x))
    e = math.log(2) * (dx + 2 * U * (x.abs() + (x - top).abs())) + 2.0 ** -18
    return P, torch.where(seen, e, torch.zeros_like(e)) * 1.01


def attend(q, kq, vq, scale, dtype, limit=None):
    """One sequence: (out [n, Hq, D], room of the same shape, P, e)."""
    P, e = weights(q, kq, scale, limit)
    codes, s, least = grow(vq, q.shape[1] // vq[0].shape[1])
    over = lambda w, x: torch.einsum("ihj,jhd->ihd", w, x.flatten(-2))
    v = codes * s + least
    wide = s.expand_as(codes)
    out = over(P, v)
    half = 2.0 ** -8 if dtype == torch.bfloat16 else 2.0 ** -16
    steps = -(-P.shape[-1] // 128)
    C = 32 * min(steps, 8) + 8 + steps
    room = over(P * (1 + e), wide * (codes - 8).abs()) * half
    room = room + over(P * e, v.abs()) + (P * e).sum(-1, keepdim=True) * out.abs()
    room = room + 2 * U * C * (over(P, 16 * wide * (2.5 + codes / 16) + (least + 8 * s).abs()) + out.abs())
    eps = torch.finfo(dtype).eps / 2
    room = room + (out.abs() + room) * eps + torch.finfo(dtype).smallest_normal * eps
    return out, room, P, e


def ratio(got, out, room):
    """The largest error in units of its bound; infinite where a value is not finite."""
    got = got.detach().double().cpu()
    if got.numel() == 0:
        return 0.0
    if not torch.isfinite(got).all():
        return math.inf
    return ((got - out).abs() / room).max().item()


def added(P, e, Hkv):
    """What a call adds to the keys' scores, [m, Hkv], and how far that may be off, relative
    (every weight's own error, that of its row's sum, and the sum over the rows)."""
    n, Hq, m = P.shape
    rows = n * (Hq // Hkv)
    add = P.sum(0).view(Hkv, Hq // Hkv, m).sum(1).t()
    off = e.amax() * 2.02 + (rows + 600) * 2 * U if m else 0.0
    return add, off


def marked(x, size):
    """x [m, H, D] with a dimension of its own raised by ``size`` in every step of 128 keys, so
    that a step that is lost shows."""
    x = x.clone()
    j = torch.arange(x.shape[0])
    x[j, :, (j // 128) % x.shape[2]] += size
    return x
