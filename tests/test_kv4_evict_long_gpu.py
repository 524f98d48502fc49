"""Eviction of sequences whose scores one pass over the registers does not hold (16384), with
more kept tokens than the list on chip has places (8192): equal scores on both sides of that
border, in one launch and in two."""
import pytest
import torch

import mqk
from test_kv4_evict_gpu import Full, i32, run

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype,D", [(BF16, 64), (F16, 128)])
@pytest.mark.parametrize("n", [16385, 40000])
@pytest.mark.parametrize("budget,recent", [(8191, 0), (8193, 100), (14000, 9000), (16384, 1), (255, 3)])
@pytest.mark.parametrize("levels", [0, 3])
def test_few_heads(dtype, D, n, budget, recent, levels):
    run(Full(1, -(-n // 16), 2, D, dtype, seed=n, levels=levels), [n], budget, recent)


@pytest.mark.parametrize("budget,recent,levels", [(20000, 64, 0), (39999, 500, 2), (20000, 20000, 0), (33000, 0, 4)])
def test_larger_budgets(budget, recent, levels):
    run(Full(1, 2500, 2, 64, BF16, levels=levels), [40000], budget, recent, ((0, 1200, -1), (0, 2499, -1)))


@pytest.mark.parametrize("budget,recent,levels", [(8191, 0, 0), (8193, 100, 3), (20000, 30, 3), (20000, 9000, 0)])
def test_many_heads(budget, recent, levels):
    """As many heads as take the move in the same launch, most of them of short sequences."""
    lens = [40000 - 16384 * (s == 1) if s < 2 else 100 + s for s in range(16)]
    f = Full(2, 2500, 8, 64, BF16, levels=levels)
    # (the others own no page: their tables name none, and they are within the budget)
    table = torch.cat((f.table, torch.full((14, 2500), -1, dtype=torch.int32)))
    one = f.cache.clone()
    marks = f.scores.clone()
    new, kept = mqk.kv4_evict(f.cache, f.scores, table.cuda(), i32(lens), budget, recent=recent)
    assert new.tolist() == [budget if n > budget else n for n in lens]
    # the two long ones alone take two launches: the same bytes, scores and positions
    new2, kept2 = mqk.kv4_evict(one, marks, f.table.cuda(), i32(lens[:2]), budget, recent=recent)
    assert torch.equal(kept[:2], kept2) and torch.equal(new[:2], new2)
    assert torch.equal(one.view(torch.int16), f.cache.view(torch.int16)) and torch.equal(marks, f.scores)


@pytest.mark.parametrize("border", [16384, 32768])
def test_equal_scores_across_the_border(border):
    """The last that fit are on one side of it: the first come first."""
    f = Full(1, 2500, 1, 64, BF16)
    w = torch.zeros(40000)
    w[border - 5:border + 5] = 1.0
    w[100:110] = 2.0
    t = torch.arange(40000)
    f.scores.zero_()
    f.scores[f.table[0].long()[t // 16].cuda(), 0, (t % 16).cuda()] = w.cuda()
    for take in (12, 15, 18, 20, 23):
        g = Full(1, 2500, 1, 64, BF16)
        g.scores = f.scores.clone()
        _, kept, _ = run(g, [40000], take + 2, 2)
        want = list(range(100, 110)) + list(range(border - 5, border + 5))[:take - 10]
        want = sorted(want + list(range(take - len(want)))) + [39998, 39999]
        assert kept[0, 0].tolist() == want
