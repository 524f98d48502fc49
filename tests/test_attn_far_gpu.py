"""The prompt attention over tensors whose rows lie far apart: byte offsets past 32 bits in
q, k and v, and rows of one tile further apart than 32 bits."""
import pytest
import torch

import mqk
from attn_oracle import attend, check

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


@pytest.fixture(scope="module")
def room():
    t = torch.empty(3 << 30, dtype=BF16, device="cuda")  # 6 GiB
    yield t
    del t
    torch.cuda.empty_cache()


@pytest.mark.parametrize("stride,n", [(1 << 25, 90), (1 << 23, 380)])
@pytest.mark.parametrize("parts", [0, 3])
def test_rows_far_apart(room, stride, n, parts):
    g = torch.Generator().manual_seed(n)
    H, D = 2, 128
    q, k, v = (torch.randn(n, h, D, generator=g).to(BF16).cuda() for h in (2 * H, H, H))
    views, at = [], 0
    for t in (q, k, v):
        w = torch.as_strided(room, t.shape, (stride, D, 1), at)
        w.copy_(t)
        views.append(w)
        at += t.shape[1] * D
    assert (n - 1) * stride * 2 > 1 << 32
    mqk.set_option("attn_parts", parts)
    try:
        for split in (0, 1, 2, 4):
            mqk.set_option("attn_split", split)
            out = mqk.attn_prefill(*views)
            assert torch.equal(out, mqk.attn_prefill(q, k, v))
    finally:
        mqk.set_option("attn_split", 0)
        mqk.set_option("attn_parts", 0)
    check(out, attend(q, k, v, D ** -0.5), BF16, f"stride {stride}")
