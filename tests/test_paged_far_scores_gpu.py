"""paged_select where products leave fp32's range downwards: the choice is still that of the exact scores."""
import pytest
import torch

import paged_oracle
from test_paged_select_gpu import selection

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,box,query", [
    *((torch.bfloat16, b, t - b) for t in (115, 124, 130, 140, 148, 150, 152, 160) for b in (30, 60, 90)),
    *((torch.bfloat16, b, t - b) for t in (124, 148) for b in (10, 114)),
    *((torch.float16, b, q) for b, q in ((0, 14), (13, 13), (14, 10), (20, 20), (24, 24))),
])
def test_products_of_small_numbers(dtype, box, query):
    """Pages with many products of about 2^-(box + query) beside pages with one of 2^4 times that: a
    sum that loses the former, in part or altogether, has the latter first."""
    n, D = 300, 256
    g = torch.Generator().manual_seed(box * 200 + query)
    boxes = torch.zeros(n, D)
    boxes[::2] = torch.rand(n // 2, D, generator=g) + 0.5
    boxes[1::2, 0] = (torch.rand(n // 2, generator=g) + 0.5) * 16
    boxes = torch.ldexp(boxes.double(), torch.tensor(-box))
    both = torch.stack([boxes, boxes], 1)[:, None].to(dtype).contiguous()
    cache = paged_oracle.Cache([8], 1, D, dtype, page=8)
    cache.table = torch.randperm(n, generator=g).int()[None].cuda()
    cache.lens = torch.tensor([n * 8], dtype=torch.int32, device="cuda")
    q = torch.ldexp(torch.rand(1, 2, D, generator=g).double() + 0.5, torch.tensor(-query)).to(dtype)
    for take in (7, 100, 152, 200):
        selection(cache, both.cuda(), q, [1], take, 1, 1, cu=False)
