"""paged_bounds and paged_select: both are exact."""
import math

import pytest
import torch

import paged_oracle

pytestmark = pytest.mark.gpu


def made(cache, new=None, cu=True, start=7.0):
    """The cache's bounds by one call, over a tensor of ``start``."""
    import mqk
    blocks, _, H, D = cache.k.shape
    b = torch.full((blocks, H, 2, D), start, dtype=cache.dtype, device="cuda")
    if new is None:
        mqk.paged_bounds(cache.k, b, cache.table, cache.lens)
    else:
        mqk.paged_bounds(cache.k, b, cache.table, cache.lens, sum(new),
                         cu_seqlens=paged_oracle.offsets(new) if cu else None)
    return b


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,D,page", [(8, 128, 16), (1, 64, 16), (4, 256, 8), (2, 80, 24), (3, 8, 32), (40, 128, 16),
                                      (2, 128, 256)])
def test_bounds(H, D, page, dtype):
    """Whole sequences, chunks and single tokens; the other pages' bounds stay."""
    lens = [1, 15, 16, 17, 100, 0, 333, 64]
    cache = paged_oracle.Cache(lens, H, D, dtype, page)
    for new, cu in ((None, True), ([1, 3, 16, 1, 40, 0, 300, 17], True), ([1] * 8, False), ([1, 15, 16, 17, 100, 0, 333, 64], True),
                    ([0, 0, 0, 0, 0, 0, 1, 0], True)):
        got = made(cache, new, cu).float().cpu()
        want = torch.full_like(got, 7.0)
        for s, n in enumerate(lens):
            from_ = 0 if new is None else max(0, n - new[s])
            if n == 0 or (new is not None and new[s] == 0):
                continue
            for j in range(from_ // page, -(-n // page)):
                want[int(cache.table[s, j])] = paged_oracle.bounds(cache, s, j)
        assert torch.equal(got, want)


def test_bounds_step_by_step():
    """After every step's call the bounds are those of the whole sequences."""
    lens = [70, 33, 16]
    full = paged_oracle.Cache(lens, 2, 64)
    import mqk
    b = torch.zeros(full.blocks, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    at = [40, 1, 0]
    mqk.paged_bounds(full.k, b, full.table, torch.tensor(at, dtype=torch.int32, device="cuda"))
    while at != lens:
        new = [min(n - a, k) for n, a, k in zip(lens, at, (3, 1, 16))]
        at = [a + n for a, n in zip(at, new)]
        mqk.paged_bounds(full.k, b, full.table, torch.tensor(at, dtype=torch.int32, device="cuda"), sum(new),
                         cu_seqlens=paged_oracle.offsets(new))
    want = made(full, start=0.0)
    assert torch.equal(b, want)


def test_bounds_of_odd_places():
    """NaN and infinities stay; pages outside the cache and past the table are left alone; a
    negative length has none."""
    cache = paged_oracle.Cache([40, 40, 40], 2, 64)
    cache.set(0, 3, k=math.nan)
    cache.set(0, 20, k=-math.inf)
    cache.table[1, 1] = cache.blocks
    cache.table[1, 2] = -1
    cache.lens[2] = -4
    lens = [40, 40]
    got = made(cache).float().cpu()
    assert torch.isnan(got[int(cache.table[0, 0])]).all()
    assert (got[int(cache.table[0, 1]), :, 0] == -math.inf).all()
    assert torch.equal(got[int(cache.table[1, 0])], paged_oracle.bounds(cache, 1, 0))
    touched = {int(cache.table[0, j]) for j in range(3)} | {int(cache.table[1, 0])}
    for b in range(cache.blocks):
        assert b in touched or (got[b] == 7.0).all()
    cache.lens[:2] = torch.tensor([2 ** 31 - 1, 1000], dtype=torch.int32)  # (past the table)
    made(cache)
    made(cache, [10, 10, 10])


def selection(cache, boxes, q, new, take, first, recent, cu=True):
    """One call, compared with the oracle."""
    import mqk
    H, page = boxes.shape[1], cache.page
    got = mqk.paged_select(q.cuda(), boxes, cache.table, cache.lens, page, take,
                           paged_oracle.offsets(new) if cu else None, first=first, recent=recent)
    assert got.shape == (*q.shape[:-2], H, take) and got.dtype == torch.int32
    table, b, G = cache.table.cpu(), boxes.cpu(), q.shape[-2] // H
    lens = cache.lens.tolist()
    at, flat, rows = 0, q.reshape(-1, *q.shape[-2:]), got.reshape(-1, H, take).cpu()
    for s, n in enumerate(new):
        there = {j for j in range(table.shape[1]) if 0 <= table[s, j] < b.shape[0]}
        sb = b[table[s].long().clamp(0, b.shape[0] - 1)]
        for i in range(n):
            pos = max(lens[s], 0) - n + i
            for h in range(H):
                want = [-1] * take if pos < 0 else paged_oracle.select(
                    flat[at + i, h * G:(h + 1) * G], sb[:, h], pos // page, take, first, recent, there)
                assert rows[at + i, h].tolist() == want, (s, i, h)
        at += n
    assert (rows[at:] == -1).all()
    return got


def queries(*shape, dtype=torch.bfloat16, seed=1):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).mul(2).to(dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H_Q,H,D,page", [(16, 8, 128, 16), (4, 4, 64, 8), (16, 1, 256, 16), (10, 2, 80, 24), (33, 1, 128, 32),
                                          (2, 2, 8, 16)])
def test_selection(H_Q, H, D, page, dtype):
    lens = [1, 30, 700, 1100, 333]
    cache = paged_oracle.Cache(lens, H, D, dtype, page)
    boxes = made(cache)
    for take, first, recent in ((1, 0, 1), (4, 1, 1), (9, 2, 3), (20, 0, 7), (300, 1, 2)):
        selection(cache, boxes, queries(5, H_Q, D, dtype=dtype), [1] * 5, take, first, recent, cu=False)
    new = [1, 5, 0, 3, 2]
    selection(cache, boxes, queries(11 + 3, H_Q, D, dtype=dtype), new, 6, 1, 2)


@pytest.mark.parametrize("pages", [1000, 17000, 40000])
def test_long_selection(pages):
    """Past what a workgroup holds in registers at a time (16384 pages)."""
    lens = [pages * 8 - 3, 700 * 8]
    g = torch.Generator().manual_seed(2)
    boxes = torch.randn(pages + 10, 1, 2, 64, generator=g).sort(2).values.bfloat16()
    cache = paged_oracle.Cache([8], 1, 64, page=8)
    cache.table = torch.randint(0, pages + 10, (2, pages), generator=g).int().cuda()
    cache.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    for take in (2, 100, 5000, 16500):
        selection(cache, boxes.cuda(), queries(2, 2, 64), [1, 1], take, 1, 1, cu=False)


def test_equal_scores():
    """Pages with the same bounds, also across a register's worth of them: the first are taken."""
    cache = paged_oracle.Cache([8], 1, 64, page=8)
    n = 3000
    boxes = torch.zeros(4, 1, 2, 64)
    boxes[1] += 1
    boxes[2, :, 1] = 1
    boxes[3, :, 0] = -1
    boxes = boxes.bfloat16().cuda()
    g = torch.Generator().manual_seed(3)
    cache.table = torch.randint(0, 4, (3, n), generator=g).int().cuda()
    cache.table[2] = 1
    cache.lens = torch.tensor([n * 8, n * 8 - 9, n * 8], dtype=torch.int32, device="cuda")
    for take in (3, 50, 700, 1500, 2990):
        selection(cache, boxes, queries(3, 2, 64), [1] * 3, take, 1, 1, cu=False)
    q = torch.zeros(3, 2, 64, dtype=torch.bfloat16)  # (all scores 0, of either sign)
    selection(cache, boxes, q, [1] * 3, 40, 0, 1, cu=False)
    selection(cache, boxes, -q, [1] * 3, 40, 0, 1, cu=False)


def test_odd_scores():
    """NaN, infinities, scores below 0 throughout; pages that are not there."""
    lens = [1600, 1600, 320]
    cache = paged_oracle.Cache(lens, 2, 64)
    boxes = made(cache)
    boxes[int(cache.table[0, 20])] = math.nan
    boxes[int(cache.table[0, 31]), 0, 1, 5] = math.nan
    boxes[int(cache.table[0, 50]), :, 1] = math.inf
    boxes[int(cache.table[0, 51]), :, 0] = -math.inf
    cache.table[1, ::3] = -1
    cache.table[1, 1] = cache.blocks
    cache.table[1, 99] = -9  # (its own)
    cache.lens[2] = 5000     # (past the table)
    q = queries(3, 4, 64)
    for take, first, recent in ((3, 1, 1), (8, 2, 2), (60, 0, 5), (99, 5, 5)):
        selection(cache, boxes, q, [1] * 3, take, first, recent, cu=False)
    low = torch.nan_to_num(-boxes.abs(), nan=-1.0).sort(2).values  # (bounds: the least first)
    selection(cache, low, q.abs(), [1] * 3, 8, 1, 1, cu=False)


def test_nothing_there():
    cache = paged_oracle.Cache([0, 40], 2, 64)
    boxes = made(cache)
    cache.lens[0] = -3
    selection(cache, boxes, queries(2, 4, 64), [1, 1], 4, 1, 1, cu=False)
    selection(cache, boxes, queries(60, 4, 64), [9, 45], 4, 1, 1)


def test_next_to_each_other():
    """Scores that 32-bit sums would mix up: the order is that of the exact values."""
    D, n = 128, 400
    g = torch.Generator().manual_seed(4)
    base = torch.randn(D, generator=g).bfloat16().float()
    boxes = base.repeat(n, 1)
    step = torch.randint(-1, 2, (n, D), generator=g).float() * 2.0 ** -9  # one place of the least values
    boxes = (boxes * (1 + 2 * step)).bfloat16()
    both = torch.stack([boxes, boxes], 1)[:, None].contiguous()
    cache = paged_oracle.Cache([8], 1, D, page=8)
    cache.table = torch.arange(n, dtype=torch.int32)[None].cuda()
    cache.lens = torch.tensor([n * 8], dtype=torch.int32, device="cuda")
    q = (torch.randn(1, 8, D, generator=g) * 100).bfloat16()
    for take in (5, 50, 201):
        selection(cache, both.cuda(), q, [1], take, 1, 1, cu=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_small_and_large_values(dtype):
    """Bounds among the type's subnormal numbers, and values whose sums leave its range."""
    tiny = torch.finfo(dtype).smallest_normal
    cache = paged_oracle.Cache([8], 2, 64, dtype, page=8)
    n = 700
    g = torch.Generator().manual_seed(6)
    cache.table = torch.arange(n, dtype=torch.int32)[None].cuda()
    cache.lens = torch.tensor([n * 8], dtype=torch.int32, device="cuda")
    base = torch.randn(n, 2, 2, 64, generator=g).sort(2).values
    q = torch.randn(1, 8, 64, generator=g)
    big = torch.finfo(dtype).max
    for boxes, query in ((base * tiny / 8, q), (base, q * tiny / 8), (base * tiny / 8, q * tiny / 8),
                         (base * big / 8, q), (base, q * big / 8), (base * big / 8, q * big / 8)):
        for take in (2, 40, 333):
            selection(cache, boxes.to(dtype).cuda(), query.to(dtype), [1], take, 1, 1, cu=False)


@pytest.mark.parametrize("each", [2, 3, 4, 5, 9])
def test_tokens_that_share_boxes(each):
    """Tokens of a sequence four at a time: own pages that differ within them, sequences that end there."""
    lens = [300 + each, each, 517, 16 * each + 1]
    cache = paged_oracle.Cache(lens, 2, 128, page=8)
    boxes = made(cache)
    selection(cache, boxes, queries(4, each, 8, 128), [each] * 4, 7, 1, 1, cu=False)
    new = [each, 1, 2 * each, 0]
    selection(cache, boxes, queries(sum(new) + 2, 8, 128), new, 7, 0, 2)
