"""The bound that the decode attention is held to, on the CPU: the kernel's arithmetic carried
out in its roundings is within it, and what a broken kernel would return is not."""
import math

import pytest
import torch

import kv4_bounds as kb
from attn_oracle import quantise

BF16, F16 = torch.bfloat16, torch.float16


def carried_out(q, kq, vq, scale, dtype, terms=None, keys=None):
    """out with p s rounded as the kernel rounds it; ``terms``: bf16 terms of p s, ``keys``: a
    mask of the keys that are taken."""
    G = q.shape[1] // kq[0].shape[1]
    kc, ks, kl = kb.grow(kq, G)
    vc, vs, vl = kb.grow(vq, G)
    x = torch.einsum("ihd,jhd->ihj", q.double(), (kc * ks + kl).flatten(-2)) * (scale * math.log2(math.e))
    m, n = x.shape[-1], x.shape[0]
    seen = torch.arange(m)[None] < (torch.arange(n) + m - n + 1)[:, None]
    if keys is not None:
        seen = seen & keys[None]
    x = torch.where(seen[:, None], x, torch.full_like(x, -math.inf))
    p = torch.exp2(x - x.amax(-1, keepdim=True)).float()
    out = []
    for g in range(vc.shape[2]):
        y = p * vs[:, :, g, 0].t().float()[None]
        t = y.bfloat16().float()
        if (terms or (1 if dtype == BF16 else 2)) == 2:
            t = t + (y - t).bfloat16().float()
        o = torch.einsum("ihj,jhd->ihd", t.double(), vc[:, :, g] - 8)
        mid = (vl + 8 * vs)[:, :, g, 0].float().double()
        out.append(o + torch.einsum("ihj,jh->ih", p.double(), mid)[..., None])
    return (torch.cat(out, -1) / p.double().sum(-1, keepdim=True)).to(dtype)


def inputs(m, dtype, D=128, S=1, Hq=4, Hkv=2, seed=0):
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(S, Hq, D, generator=g) * 1.5).to(dtype)
    k = torch.randn(m, Hkv, D, generator=g).to(dtype)
    v = kb.marked(torch.randn(m, Hkv, D, generator=g), 6.0).to(dtype)
    return q, quantise(k), quantise(v), D ** -0.5


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m,S", [(1, 1), (33, 2), (600, 1), (4097, 1), (20000, 1)])
def test_kernels_arithmetic_is_within(dtype, m, S):
    q, kq, vq, scale = inputs(m, dtype, S=S)
    out, room, P, e = kb.attend(q, kq, vq, scale, dtype)
    assert kb.ratio(carried_out(q, kq, vq, scale, dtype), out, room) <= 1


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("m", [600, 4097, 20000])
def test_lost_keys_heads_and_results_are_not(dtype, m):
    q, kq, vq, scale = inputs(m, dtype)
    out, room, P, e = kb.attend(q, kq, vq, scale, dtype)
    good = carried_out(q, kq, vq, scale, dtype)
    assert kb.ratio(torch.zeros_like(good), out, room) > 1
    assert kb.ratio(good.flip(1), out, room) > 1
    assert kb.ratio(good * math.nan, out, room) > 1
    j = torch.arange(m)
    for step in sorted({0, 1, m // 256, m // 128 - 1}):
        assert kb.ratio(carried_out(q, kq, vq, scale, dtype, keys=j // 128 != step), out, room) > 1, step
    assert kb.ratio(carried_out(q, kq, vq, scale, dtype, keys=j < m - 512), out, room) > 1
    assert kb.ratio(carried_out(q, kq, vq, scale * 1.05, dtype), out, room) > 1


def alike(m, D=128, Hkv=2, seed=0):
    """fp16 tokens whose values are all the same and weights nearly so: the roundings of p s
    have one direction, and do not average out."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(1, 4, D, generator=g) * 0.02).half()
    k = torch.randn(1, Hkv, D, generator=g).half().expand(m, -1, -1)
    # (scales of 1 + 2^-8: half a step of bf16 from it)
    v = (((torch.randint(0, 16, (1, Hkv, D), generator=g)) - 8) * (1 + 2.0 ** -8)).half()
    v[..., ::64], v[..., 1::64] = -8 * (1 + 2.0 ** -8), 7 * (1 + 2.0 ** -8)
    return q, k.contiguous(), v.expand(m, -1, -1).contiguous(), D ** -0.5


@pytest.mark.parametrize("m", [1, 20, 300, 1500, 4097])
def test_one_bf16_term_for_fp16_is_not(m):
    q, k, v, scale = alike(m)
    kq, vq = quantise(k), quantise(v)
    out, room, P, e = kb.attend(q, kq, vq, scale, F16)
    assert kb.ratio(carried_out(q, kq, vq, scale, F16), out, room) <= 1
    assert kb.ratio(carried_out(q, kq, vq, scale, F16, terms=1), out, room) > 1


def test_weights():
    """A weight that is left out, or added twice, is past the bound of its key."""
    q, kq, vq, scale = inputs(700, BF16)
    P, e = kb.weights(q, kq, scale)
    add, off = kb.added(P, e, 2)
    assert 0 < off < 0.1 and torch.allclose(add.sum(0), torch.full((2,), 2.0).double())
    other, _ = kb.added(P.roll(1, -1), e, 2)
    assert ((other - add).abs() > add * off).any()
