"""paged_attn against attention in 64 bits, at the sizes and masks where it can go wrong."""
import math

import pytest
import torch

import attn_oracle
import paged_oracle

pytestmark = pytest.mark.gpu


def queries(T, H_Q, D, dtype=torch.bfloat16, seed=1, std=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, H_Q, D, generator=g) * std).to(dtype)


def run(cache, q, new, cu=True, **kw):
    import mqk
    cu = paged_oracle.offsets(new) if cu else None
    return mqk.paged_attn(q.cuda(), cache.k, cache.v, cache.table, cache.lens, cu, **kw)


def compare(lens, new, H_Q, H_KV, D, dtype=torch.bfloat16, page=16, cu=True, seed=0, **kw):
    cache = paged_oracle.Cache(lens, H_KV, D, dtype, page, seed=seed, **kw)
    q = queries(sum(new), H_Q, D, dtype, seed + 1)
    got = run(cache, q, new, cu)
    attn_oracle.check(got, paged_oracle.attend(cache, q, new, D ** -0.5), dtype, f"{lens} {new}")
    return got


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H_Q,H_KV,D", [(16, 8, 128), (8, 8, 64), (64, 4, 128), (10, 2, 80), (6, 1, 256), (40, 8, 96),
                                        (33, 1, 128), (3, 3, 8)])
def test_steps(H_Q, H_KV, D, dtype):
    """Single tokens: one key, lengths around a tile, a page and a step, one that takes many parts."""
    compare([1, 15, 16, 17, 32, 33, 127, 128, 129, 300, 2500], [1] * 11, H_Q, H_KV, D, dtype, cu=False)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H_Q,H_KV,D", [(16, 8, 128), (8, 8, 64), (64, 4, 128), (10, 2, 80), (6, 1, 256), (33, 1, 128)])
def test_chunks_and_steps(H_Q, H_KV, D, dtype):
    """Chunks, prompts without a prefix, single tokens and sequences with nothing new in one call."""
    new = [1, 40, 0, 130, 1, 7, 64, 3, 200]
    old = [50, 0, 10, 77, 0, 500, 1000, 16, 300]
    compare([a + b for a, b in zip(new, old)], new, H_Q, H_KV, D, dtype)


@pytest.mark.parametrize("page", [8, 16, 24, 32, 64, 128, 1000])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_pages(page, D):
    compare([5, 100, 1003, 64, 640], [1, 100, 33, 2, 300], 4, 2, D, page=page)
    compare([5, 100, 1003, 64, 640], [1] * 5, 4, 2, D, page=page, cu=False)


@pytest.mark.parametrize("S", [1, 2, 3, 5, 8, 9, 17, 33])
def test_equal_tokens(S):
    """[B, S, H, D] without offsets: both launches' sides of 32 rows, 16 heads a key head."""
    lens = [S, S + 1, 129 + S, 700]
    import mqk
    cache = paged_oracle.Cache(lens, 2, 128)
    q = queries(4 * S, 8, 128)
    got = mqk.paged_attn(q.cuda().view(4, S, 8, 128), cache.k, cache.v, cache.table, cache.lens)
    assert got.shape == (4, S, 8, 128)
    attn_oracle.check(got.flatten(0, 1), paged_oracle.attend(cache, q, [S] * 4, 128 ** -0.5), torch.bfloat16, S)


@pytest.mark.parametrize("lens,new", [([9000], [1]), ([9000], [70]), ([5000, 40], [1, 1]), ([3000] * 3, [129, 1, 300]),
                                      ([2500] + [100] * 40, [600] + [1] * 40)])
def test_long(lens, new):
    """Keys in parts, over the join."""
    compare(lens, new, 8, 2, 128)
    compare(lens, new, 4, 4, 64, torch.float16)


@pytest.mark.parametrize("B", [63, 64, 65, 130, 300])
def test_many_sequences(B):
    """Around the 64 sequences that a wave looks at at a time."""
    lens = [1 + 37 * i % 200 for i in range(B)]
    compare(lens, [1] * B, 4, 2, 64, cu=False)
    new = [(1, 0, min(20, n), 1)[i % 4] for i, n in enumerate(lens)]
    compare(lens, new, 4, 2, 64)


def test_nothing_seen():
    """Padded entries of length 0, more tokens than keys, lengths below 0."""
    cache = paged_oracle.Cache([0, 3, 50, 0], 2, 128)
    for new in ([1, 1, 1, 1], [5, 8, 60, 40]):
        q = queries(sum(new), 4, 128)
        got = run(cache, q, new)
        attn_oracle.check(got, paged_oracle.attend(cache, q, new, 128 ** -0.5), torch.bfloat16, new)
        assert (got[:new[0]] == 0).all() and (got[-new[3]:] == 0).all()
        if new[1] == 8:
            assert (got[5:10] == 0).all()
    cache.lens[0] = -7
    assert (run(cache, queries(4, 4, 128), [1] * 4)[0] == 0).all()


@pytest.mark.parametrize("new", [[1, 1], [40, 1], [150, 2]])
def test_pages_that_are_not_there(new):
    """Entries outside the cache hold no keys; a length past the table has its last keys past it."""
    lens = [200, 300]
    cache = paged_oracle.Cache(lens, 2, 128)
    there = [list(range(n)) for n in lens]
    for s, j, entry in ((0, 2, -1), (0, 9, 10 ** 6), (1, 0, cache.blocks), (1, 18, -5)):
        cache.table[s, j] = entry
        there[s] = [p for p in there[s] if p // 16 != j]
    q = queries(sum(new), 4, 128)
    want = paged_oracle.attend(cache, q, new, 128 ** -0.5, there)
    attn_oracle.check(run(cache, q, new), want, torch.bfloat16, new)
    cache.table = cache.table[:, :11].contiguous()
    there = [[p for p in t if p < 11 * 16] for t in there]
    want = paged_oracle.attend(cache, q, new, 128 ** -0.5, there)
    attn_oracle.check(run(cache, q, new), want, torch.bfloat16, new)


@pytest.mark.parametrize("new,D", [([1, 20], 128), ([150, 33], 128), ([2, 3], 64), ([140, 5], 256)])
def test_values_behind_a_token(new, D):
    """Infinities and NaN among later tokens' keys and values do not reach earlier ones."""
    lens = [n + 70 for n in new]
    cache = paged_oracle.Cache(lens, 2, D)
    q = queries(sum(new), 4, D)
    want = paged_oracle.attend(cache, q, new, D ** -0.5)
    last = [n - 1 for n in lens]
    cache.set(0, last[0], k=math.nan, v=math.inf)
    cache.set(1, last[1], k=math.inf, v=math.nan)
    got = run(cache, q, new)
    keep = torch.ones(sum(new), dtype=torch.bool)
    keep[new[0] - 1] = keep[-1] = False
    attn_oracle.check(got.cpu()[keep], tuple(x[keep] for x in want), torch.bfloat16, new)
    assert torch.isnan(got[~keep.cuda()]).all()


@pytest.mark.parametrize("new", [[1, 1, 1], [3, 30, 200]])
def test_values_that_are_seen(new):
    """A value of infinity gives infinity to the tokens that see it, and to no other."""
    lens = [260, 90, 400]
    cache = paged_oracle.Cache(lens, 2, 128)
    q = queries(sum(new), 4, 128, std=0.5)
    base = paged_oracle.attend(cache, q, new, 128 ** -0.5)
    at = [m - max(1, n // 2) for m, n in zip(lens, new)]
    v = torch.zeros(2, 128, dtype=torch.bfloat16)
    v[1, 7] = math.inf
    for s, p in enumerate(at):
        cache.set(s, p, v=v)
    got = run(cache, q, new).cpu()
    row = 0
    for s, n in enumerate(new):
        for i in range(n):
            sees = lens[s] - n + i >= at[s]
            assert (got[row, 2:, 7] == math.inf).all() if sees else torch.isfinite(got[row]).all()
            if not sees:
                one = slice(row, row + 1)
                attn_oracle.check(got[one], tuple(x[one] for x in base), torch.bfloat16, (s, i))
            row += 1


@pytest.mark.parametrize("new", [[1, 1], [40, 150]])
def test_scores_of_infinity(new):
    """Keys with a score of -infinity have no part; a query with no other gives 0."""
    lens = [60, 200]
    cache = paged_oracle.Cache(lens, 1, 64)
    q = queries(sum(new), 2, 64).abs() + 0.5
    there = [list(range(n)) for n in lens]
    for s, n in enumerate(lens):
        for p in range(0, n, 3):
            cache.set(s, p, k=-math.inf)
        there[s] = [p for p in there[s] if p % 3]
    attn_oracle.check(run(cache, q, new), paged_oracle.attend(cache, q, new, 0.125, there), torch.bfloat16, new)
    for s, n in enumerate(lens):
        for p in range(n):
            cache.set(s, p, k=-math.inf)
    assert (run(cache, q, new) == 0).all()


def test_lowest_values():
    """Scores near the type's lowest value, and large ones of either sign."""
    cache = paged_oracle.Cache([100, 70], 2, 128)
    cache.k.mul_(3000.0)
    for rows in cache.k_rows:
        rows.mul_(3000.0)
    new = [1, 40]
    q = queries(41, 4, 128, std=100.0)
    attn_oracle.check(run(cache, q, new), paged_oracle.attend(cache, q, new, 128 ** -0.5), torch.bfloat16, "large")


def test_rows_behind_the_last_sequence():
    import mqk
    cache = paged_oracle.Cache([30, 90], 2, 64)
    for new in ([1, 1], [3, 50]):
        T = sum(new) + 9
        q = queries(T, 4, 64)
        cu = paged_oracle.offsets(new)
        got = mqk.paged_attn(q.cuda(), cache.k, cache.v, cache.table, cache.lens, cu)
        assert (got[sum(new):] == 0).all()
        out = torch.full_like(got, 7.0)
        assert mqk.paged_attn(q.cuda(), cache.k, cache.v, cache.table, cache.lens, cu, out=out) is out
        assert (out[sum(new):] == 7.0).all() and torch.equal(out[:sum(new)], got[:sum(new)])
    empty = mqk.paged_attn(q[:0].cuda(), cache.k, cache.v, cache.table, cache.lens, paged_oracle.offsets([0, 0]))
    assert empty.shape == (0, 4, 64)


def test_strides():
    """q as a slice of a packed projection, and as a transposed view (copied)."""
    import mqk
    cache = paged_oracle.Cache([30, 90], 2, 64)
    new = [2, 50]
    packed = queries(52, 8, 64).cuda()
    q = packed[:, 2:6]
    want = paged_oracle.attend(cache, q, new, 0.125)
    cu = paged_oracle.offsets(new)
    attn_oracle.check(mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens, cu), want, torch.bfloat16, "slice")
    t = q.transpose(0, 1).contiguous().transpose(0, 1)
    attn_oracle.check(mqk.paged_attn(t, cache.k, cache.v, cache.table, cache.lens, cu), want, torch.bfloat16, "heads first")
    t = q.transpose(1, 2).contiguous().transpose(1, 2)
    attn_oracle.check(mqk.paged_attn(t, cache.k, cache.v, cache.table, cache.lens.long(), cu.long()), want, torch.bfloat16,
                      "dims first")


def test_shared_pages():
    """Sequences with a common prefix read the same pages."""
    cache = paged_oracle.Cache([160, 170, 50], 2, 128)
    cache.table[1, :10] = cache.table[0, :10]
    cache.k_rows[1][:160], cache.v_rows[1][:160] = cache.k_rows[0], cache.v_rows[0]
    for new in ([1, 1, 1], [3, 10, 50]):
        q = queries(sum(new), 4, 128)
        attn_oracle.check(run(cache, q, new), paged_oracle.attend(cache, q, new, 128 ** -0.5), torch.bfloat16, new)


def test_same_result_again():
    """Bit for bit the same, call by call, and whether a step runs alone or beside chunks."""
    import mqk
    lens = [4000, 900, 2000]
    cache = paged_oracle.Cache(lens, 2, 128)
    q = queries(3, 8, 128).cuda()
    first = mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens)
    for _ in range(5):
        assert torch.equal(mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens), first)


@pytest.mark.parametrize("H_Q,H_KV,D,page,dtype", [(8, 2, 128, 16, torch.bfloat16), (16, 1, 64, 8, torch.float16),
                                                   (40, 1, 128, 32, torch.bfloat16), (4, 2, 256, 64, torch.bfloat16),
                                                   (6, 2, 80, 24, torch.float16)])
@pytest.mark.parametrize("take", [1, 3, 9, 70])
def test_selected_pages(H_Q, H_KV, D, page, dtype, take):
    """Lists of pages: any order, none among them, the own page in part, pages behind the token."""
    new = [1, 4, 0, 2]
    lens = [700, 90, 30, 2]
    cache = paged_oracle.Cache(lens, H_KV, D, dtype, page)
    q = queries(7, H_Q, D, dtype)
    g = torch.Generator().manual_seed(5)
    pages = torch.randint(-1, cache.cols + 2, (7, H_KV, take), generator=g).int()
    pages[0, 0, 0] = (lens[0] - 1) // page
    got = run(cache, q, new, pages=pages.cuda())
    attn_oracle.check(got, paged_oracle.attend_pages(cache, q, new, pages, D ** -0.5), dtype, take)


def test_all_pages_listed():
    """A list of all pages gives what the whole sequence gives, within the bound; parts are joined."""
    import mqk
    cache = paged_oracle.Cache([5000, 3333], 2, 128)
    q = queries(4, 8, 128)
    pages = torch.arange(cache.cols, dtype=torch.int32).expand(2, 2, 2, -1).contiguous().cuda()
    got = mqk.paged_attn(q.cuda().view(2, 2, 8, 128), cache.k, cache.v, cache.table, cache.lens, pages=pages)
    attn_oracle.check(got.flatten(0, 1), paged_oracle.attend(cache, q, [2, 2], 128 ** -0.5), torch.bfloat16, "all")


def test_lists_of_nothing():
    cache = paged_oracle.Cache([100, 0], 2, 64)
    q = queries(2, 4, 64)
    for pages in (torch.full((2, 2, 5), -1), torch.full((2, 2, 40), 6)):  # none; behind the tokens
        pages[0, 0, 3] = 7  # (past the table)
        got = run(cache, q, [1, 1], pages=pages.int().cuda())
        want = paged_oracle.attend_pages(cache, q, [1, 1], pages, 0.125)
        attn_oracle.check(got, want, torch.bfloat16, "nothing")
        assert (got[1] == 0).all()
