"""The paged operators where sizes decide: caches past 32-bit offsets, lengths that cut the
workgroups' parts anywhere, and ties of any number at the border of a selection."""
import pytest
import torch

import attn_oracle
import paged_oracle
from test_paged_attn_gpu import compare, queries
from test_paged_select_gpu import selection

pytestmark = pytest.mark.gpu


def test_offsets_past_32_bits():
    """The last pages of an 18 GB cache, and of 4.5 GB of bounds: the same bits as in a small one."""
    import mqk
    lens, new, blocks = [700, 33, 300], [1, 20, 60], 1100000
    small = paged_oracle.Cache(lens, 8, 128, page=8)
    n = small.blocks
    k, v = (torch.empty(blocks, 8, 8, 128, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    boxes = torch.empty(blocks, 8, 2, 128, dtype=torch.bfloat16, device="cuda")
    k[blocks - n:], v[blocks - n:] = small.k, small.v
    assert k.numel() * 2 > 2 ** 34 and boxes.numel() * 2 > 2 ** 32
    few = torch.zeros(n, 8, 2, 128, dtype=torch.bfloat16, device="cuda")
    table = torch.where(small.table >= 0, small.table + (blocks - n), small.table)
    boxes[blocks - n:] = 0
    q, cu = queries(sum(new), 16, 128).cuda(), paged_oracle.offsets(new)
    for a, b, t in ((small.k, few, small.table), (k, boxes, table)):
        mqk.paged_bounds(a, b, t, small.lens)
    assert torch.equal(few, boxes[blocks - n:])
    pages = [mqk.paged_select(q, b, t, small.lens, 8, 12, cu) for b, t in ((few, small.table), (boxes, table))]
    assert torch.equal(*pages)
    for kw in ({}, {"pages": pages[0]}):
        assert torch.equal(mqk.paged_attn(q, small.k, small.v, small.table, small.lens, cu, **kw),
                           mqk.paged_attn(q, k, v, table, small.lens, cu, **kw))
    attn_oracle.check(mqk.paged_attn(q, k, v, table, small.lens, cu), paged_oracle.attend(small, q.cpu(), new, 128 ** -0.5),
                      torch.bfloat16, "far")


def test_slots_past_32_bits():
    import mqk
    table = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    free = torch.tensor([2 ** 31 - 1, 2 ** 30, 5], dtype=torch.int32, device="cuda")
    lens = torch.zeros(2, dtype=torch.int32, device="cuda")
    step = mqk.paged_tables(lens, torch.tensor([17, 2], dtype=torch.int32, device="cuda"), table, free, 19)
    want = [(2 ** 31 - 1) * 16 + i for i in range(16)] + [2 ** 30 * 16] + [80, 81]
    assert step.slots.tolist() == want and step.taken.tolist() == [3]


@pytest.mark.parametrize("D,H_KV,H_Q", [(128, 8, 16), (64, 8, 8), (256, 4, 4)])
@pytest.mark.parametrize("kind", ["ragged", "short", "mixed", "one step"])
def test_parts_anywhere(kind, D, H_KV, H_Q):
    """In tables wide enough for parts: heads that begin and end inside them, many in one, none."""
    g = torch.Generator().manual_seed(5)
    some = lambda n, lo, hi: torch.randint(lo, hi, (n,), generator=g).tolist()
    lens = {"ragged": some(32, 320, 2240), "short": some(150, 1, 300), "mixed": some(40, 1, 90) + [0, 3000, 1, 128, 129],
            "one step": [100] * 70}[kind]
    compare(lens, [1] * len(lens), H_Q, H_KV, D, cols=400)
    if kind == "mixed":
        new = [(1, 0, 3, 2, 60)[i % 5] if n >= 60 else min(n, 1) for i, n in enumerate(lens)]
        compare(lens, new, H_Q, H_KV, D, cols=400)


@pytest.mark.parametrize("heads", [255, 256, 257, 320, 500, 513])
def test_workgroups_a_head(heads):
    """Narrow tables: a head a workgroup, or parts where the last round of those would be thin."""
    compare([1000 - i % 900 for i in range(heads)], [1] * heads, 2, 1, 64)


@pytest.mark.parametrize("ties", [2, 20, 63, 64, 65, 300, 511, 512, 513, 1500])
def test_ties_at_the_border(ties):
    """Of equal pages at the border the first ones are taken, however many there are."""
    g = torch.Generator().manual_seed(ties)
    n, D = 2500, 64
    boxes = torch.randn(n, 1, 2, D, generator=g).sort(2).values.bfloat16()
    q = queries(1, 4, D)
    x = boxes[:, 0].double()[:, :, None] * q[0].double()  # [n, 2, heads, D]
    best = x.amax(1).sum((1, 2)).argsort(descending=True)
    table = torch.randperm(n, generator=g)[:n - ties]
    table = torch.cat([table, best[60].repeat(ties)])[torch.randperm(n, generator=g)]
    cache = paged_oracle.Cache([8], 1, D, page=8)
    cache.table = table[None].int().cuda()
    cache.lens = torch.tensor([n * 8], dtype=torch.int32, device="cuda")
    for take in (60, 62 + ties // 2, 60 + ties, 70 + ties):
        selection(cache, boxes.cuda(), q, [1], take, 1, 1, cu=False)
