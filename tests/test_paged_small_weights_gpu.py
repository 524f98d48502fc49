"""paged_attn where one key has nearly all the weight: what many others have together still counts."""
import math

import pytest
import torch

import attn_oracle
import paged_oracle

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("far", [12.0, 18.5, 20.5, 25.5, 28.5])
@pytest.mark.parametrize("form", ["chunk", "steps", "pages"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_weights_far_below_the_largest(dtype, form, far):
    """8000 keys of weight 2^-far beside the one of the first key, whose value is 0; calls with so
    many rows that no workgroup has only a part of the keys.

    A weight w, relative to the largest, is rounded to the type as 2^7 w (fp16) or w (bf16): by half
    an eps of it where that is a normal number of the type (fp16: down to w = 2^-21), by half a step
    of the subnormal ones below that (fp16: 2^-25 - 7 of the largest weight for each such key)."""
    import mqk
    n, D, B = 8000, 64, 1 if form == "chunk" else 300
    cache = paged_oracle.Cache([n], 1, D, dtype)
    k, v = (torch.zeros(n, 1, D, dtype=dtype) for _ in range(2))
    v[1:] = torch.rand(n - 1, 1, D, generator=torch.Generator().manual_seed(3)).add(0.5).to(dtype)
    k[1:, :, 0] = -far / 8  # (exact in both types)
    for rows, pages in ((k, cache.k), (v, cache.v)):
        pages[cache.table[0].long()] = rows.view(-1, 16, 1, D).cuda()
    cache.k_rows[0], cache.v_rows[0] = k, v
    scale = 2.0 * math.log(2.0)  # of q 4 at dimension 0: scores 8 k, in powers of 2
    q = torch.zeros((1024, 64, D) if form == "chunk" else (B, 2, D), dtype=dtype)
    q[..., 0] = 4.0
    some = 3 if form == "chunk" else 1  # (the last tokens; all heads and sequences are alike)
    want = attn_oracle.attend(q[-some:, :2], k, v, scale)
    room = attn_oracle.bound(dtype, *want[:3])
    if dtype == torch.float16 and far > 21:
        room = room + 2.0 ** -32 * v.double().sum(0)
    pages = None
    if form == "pages":
        pages = torch.arange(cache.cols, dtype=torch.int32, device="cuda").expand(B, 1, -1).contiguous()
    got = mqk.paged_attn(q.cuda(), cache.k, cache.v, cache.table.expand(B, -1).contiguous(), cache.lens.expand(B).contiguous(),
                         paged_oracle.offsets([1024]) if form == "chunk" else None, pages=pages, scale=scale)
    got = got[-some:, :2].double().cpu() if form == "chunk" else got.double().cpu()
    over = ((got - want[0]).abs() / room).max().item()
    assert over <= 1.0, over
