"""Eviction from the 4-bit cache where it could go wrong: pages that are not there, lengths
past the table."""
import pytest
import torch

import mqk
from attn_oracle import check, kv4_attend, quantise, values

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Full:
    """Sequences that fill ``cols`` pages each (scattered, all in the cache), with scores."""

    def __init__(self, n_seqs, cols, H, D, dtype, seed=0, levels=0):
        g = torch.Generator().manual_seed(seed)
        self.n, self.cols, self.H, self.D, self.dtype = n_seqs, cols, H, D, dtype
        self.blocks = n_seqs * cols + 3
        self.table = torch.randperm(self.blocks, generator=g)[:n_seqs * cols].int().view(n_seqs, cols)
        T = n_seqs * cols * 16
        self.k, self.v = (torch.randn(T, H, D, generator=g).to(dtype).cuda() for _ in range(2))
        self.cache = mqk.kv4_cache(self.blocks, H, D, dtype=dtype)
        self.full = i32([cols * 16] * n_seqs)
        mqk.kv4_write(self.k, self.v, self.cache, self.table.cuda(), self.full)
        self.scores = torch.rand(self.blocks, H, 16, generator=g)
        if levels:  # many equal ones
            self.scores = (self.scores * levels).round() / levels
        self.scores = self.scores.cuda()

    def held(self):
        """K, V and scores [n, cols * 16, H, ..] of every position, whatever the lengths."""
        k, v = mqk.kv4_read(self.cache, self.table.cuda(), self.full, self.n * self.cols * 16)
        s = self.scores[self.table.cuda().long()].permute(0, 1, 3, 2).reshape(self.n, -1, self.H)
        return [x.view(self.n, -1, *x.shape[1:]) for x in (k, v)] + [s.clone()]


def expect(w, there, n, budget, recent):
    """Kept positions of one sequence's head by sorting: w and there of the table's positions."""
    if n <= budget:
        return list(range(n))
    p = torch.arange(len(w))
    old = p[there & (p < n - recent)]
    first = old[w[old].sort(descending=True, stable=True).indices[:budget - recent]].sort().values
    return first.tolist() + p[there & (p >= n - recent) & (p < n)].tolist()


def run(f, lens, budget, recent, missing=()):
    """Evicts and looks at everything: lengths, positions, every slot of every page."""
    holes = f.table.clone()
    for s, page, what in missing:
        holes[s, page] = what
    there = ((holes >= 0) & (holes < f.blocks)).repeat_interleave(16, 1)
    before, spare = f.held(), f.cache.clone()
    new, kept = mqk.kv4_evict(f.cache, f.scores, holes.cuda(), i32(lens), budget, recent=recent)
    after = f.held()
    for s, n in enumerate(lens):
        want = [b[s].clone() for b in before]
        w = before[2][s].cpu()
        for h in range(f.H):
            keep = expect(w[:, h], there[s], n, budget, recent)
            assert new[s] == len(keep), (s, h)
            assert kept[s, h].tolist() == keep + [-1] * (budget - len(keep)), (s, h)
            if n <= budget:
                continue
            at = torch.arange(len(keep))
            live = there[s][:len(keep)]  # (a place in a page that is not there holds nothing)
            src = torch.tensor(keep, dtype=torch.long)[live].cuda()
            for x, b in zip(want, before):
                x[at[live].cuda(), h] = b[s, src, h]
        for x, got, name in zip(want, after, ("keys", "values", "scores")):
            assert torch.equal(x, got[s]), (name, s)
    free = [b for b in range(f.blocks) if b not in set(f.table.flatten().tolist())]
    assert torch.equal(f.cache[free].view(torch.int16), spare[free].view(torch.int16))
    return new, kept, holes


GONE = ((0, 2, -1),)


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("cols,lens,budget,recent,missing", [
    (3, [48], 24, 16, GONE),                               # all of the recent tokens
    (3, [47], 24, 24, GONE), (3, [48], 24, 0, GONE),
    (4, [60], 40, 20, ((0, 2, 1 << 30),)),                 # some of them
    (7, [100], 90, 4, ((0, 1, -1), (0, 5, 1 << 30))),      # fewer there than the budget
    (3, [48, 48, 40], 30, 7, tuple((1, p, -7) for p in range(3))),  # nothing there
    (5, [80, 16, 33], 34, 3, ((0, 4, -1), (1, 0, -1), (2, 1, -1))),  # short ones are left alone
    (40, [600, 640], 500, 200, ((0, 35, -1), (1, 39, -1), (1, 38, 1 << 30), (1, 20, -2))),
    (40, [640, 300], 620, 10, tuple((0, p, -1) for p in range(25, 40))),
    (80, [1270, 1280], 1100, 1100, ((0, 79, -1), (0, 75, -1), (1, 10, -1))),
])
def test_pages_that_are_not_there(dtype, D, cols, lens, budget, recent, missing):
    run(Full(len(lens), cols, 2, D, dtype, seed=budget, levels=8 * (budget % 4 == 0)), lens, budget, recent, missing)


def test_pages_that_are_not_there_of_many_heads():
    """One launch with the move in it, past its first batch of 1024 tokens."""
    f = Full(17, 90, 8, 64, BF16, levels=50)
    lens = [1300 + 5 * s for s in range(17)]
    missing = [(s, (11 * s) % 80 + 9, -1) for s in range(0, 17, 3)] + [(16, p, -1) for p in range(40, 80)]
    run(f, lens, 1200, 64, missing)


@pytest.mark.parametrize("cols,budget,recent", [(7, 50, 8), (7, 50, 0), (7, 50, 50), (7, 130, 8), (7, 190, 150), (7, 300, 8),
                                                (60, 700, 20), (60, 990, 40), (60, 990, 985)])
@pytest.mark.parametrize("over", [3, 88])
def test_lengths_past_the_table(cols, budget, recent, over):
    """Positions past the table hold nothing, the recent ones among them."""
    run(Full(2, cols, 2, 64, BF16, seed=cols), [cols * 16 + over, cols * 16], budget, recent)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_what_was_not_there_is_not_attended_to(dtype):
    """A sequence whose recent pages are gone: decoding over it afterwards sees the kept tokens."""
    f = Full(2, 4, 2, 64, dtype)
    lens, G = [64, 50], 2
    new, kept, holes = run(f, lens, 30, 16, ((0, 3, -1), (1, 3, 1 << 30)))
    assert new.tolist() == [14, 28]
    q = torch.randn(2, 1, 2 * G, 64, generator=torch.Generator().manual_seed(1)).to(dtype).cuda()
    out = mqk.kv4_attn(q, f.cache, holes.cuda(), new)
    k, v = (x.view(2, -1, 2, 64) for x in (f.k, f.v))
    for s in range(2):
        n = int(new[s])
        src = kept[s, :, :n].long().t()[..., None].expand(-1, -1, 64)
        want = kv4_attend(q[s], quantise(k[s].gather(0, src)), quantise(v[s].gather(0, src)), 64 ** -0.5)
        check(out[s], want, dtype, f"sequence {s}")
