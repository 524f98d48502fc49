"""Queries all of whose scores are -infinity (keys of a type's infinities): 0, as for a query
that sees no key, whichever way the call is cut; one finite score is enough for the others."""
import math

import pytest
import torch

import mqk

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("option,value", [("attn_split", 0), ("attn_split", 1), ("attn_split", 2), ("attn_split", 4),
                                          ("attn_parts", 2), ("attn_parts", 7)])
def test_only_infinite_scores(dtype, D, option, value):
    g = torch.Generator().manual_seed(D)
    n, first = 300, 170  # keys before `first` score -infinity in head 0
    q, k, v = (torch.randn(n, h, D, generator=g).to(dtype).cuda() for h in (4, 2, 2))
    q[:, :, 0] = 1.0
    clean = k.clone()
    clean[:, 0, 0] = k[:, 0, 0] = 0.0
    k[:first, 0, 0] = -math.inf
    mqk.set_option(option, value)
    try:
        out = mqk.attn_prefill(q, k, v)
        want = mqk.attn_prefill(q, clean, v)
    finally:
        mqk.set_option(option, 0)
    assert (out[:first, :2] == 0).all()
    assert torch.equal(out[:, 2:], want[:, 2:])
    # the first query that has a finite score has one key
    eps = torch.finfo(dtype).eps
    assert ((out[first, :2] - v[first, 0]).abs() <= eps * v[first, 0].abs()).all()
    assert torch.isfinite(out).all()
