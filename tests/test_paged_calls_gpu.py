"""The paged operators in calls that other tests do not make: packed batches of every kind again and
again, tables much wider than their sequences, bounds of subnormal numbers beside others."""
import pytest
import torch

import attn_oracle
import paged_oracle
from test_paged_attn_gpu import queries, run
from test_paged_select_gpu import made, queries as tokens, selection

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D,dtype", [(128, torch.bfloat16), (64, torch.float16), (256, torch.bfloat16)])
def test_packed_call_again(D, dtype):
    """Steps and chunks of one call, both cut and joined: the same bits call by call, and each
    within its bound.  (Beside other sequences one may be cut elsewhere: then only the bound holds.)"""
    lens, new = [4000, 3900, 77, 2600, 5000, 0], [1, 150, 1, 300, 3, 1]
    cache = paged_oracle.Cache(lens, 2, D, dtype)
    q = queries(sum(new), 8, D, dtype)
    want = paged_oracle.attend(cache, q, new, D ** -0.5)
    first = run(cache, q, new)
    attn_oracle.check(first, want, dtype, "mixed")
    for _ in range(5):
        assert torch.equal(run(cache, q, new), first)


@pytest.mark.parametrize("B,H_Q,H_KV,cols", [(1, 16, 8, 40), (9, 32, 8, 40), (40, 8, 2, 500), (300, 8, 2, 40), (300, 40, 1, 300)])
def test_packed_steps(B, H_Q, H_KV, cols):
    """Decode steps with offsets, as ``paged_tables`` gives them: few and many sequences, narrow and
    wide tables, more heads than 32 a key head."""
    lens = [1 + 41 * i % 600 for i in range(B)]
    cache = paged_oracle.Cache(lens, H_KV, 128, cols=cols)
    q = queries(B, H_Q, 128)
    attn_oracle.check(run(cache, q, [1] * B), paged_oracle.attend(cache, q, [1] * B, 128 ** -0.5), torch.bfloat16, B)


@pytest.mark.parametrize("cu", [False, True])
@pytest.mark.parametrize("each,B", [(1, 3), (150, 4)])
def test_selection_in_a_wide_table(each, B, cu):
    """Tables much wider than any sequence, and more tokens than one round of the selection takes."""
    lens = [each, 700, 333 + each, 1100][:B]
    cache = paged_oracle.Cache(lens, 2, 64, cols=30001)
    boxes = made(cache)
    q = tokens(B * each + 2, 4, 64) if cu else tokens(B, each, 4, 64)
    selection(cache, boxes, q, [each] * B, 9, 1, 2, cu=cu)


def test_subnormal_bounds_beside_others():
    """fp16: pages whose score is a sum of subnormal numbers against pages with a single normal one.
    Were the former counted as 0, the bound of the scores' error would not cover it."""
    n, D = 900, 256
    g = torch.Generator().manual_seed(8)
    boxes = torch.zeros(n, D)
    boxes[::2] = torch.randint(1, 1024, (n // 2, D), generator=g) * 2.0 ** -24
    boxes[1::2, 0] = torch.randint(1, 64, (n // 2,), generator=g) * 2.0 ** -14
    both = torch.stack([boxes, boxes], 1)[:, None].half().contiguous()
    cache = paged_oracle.Cache([8], 1, D, torch.float16, page=8)
    cache.table = torch.randperm(n, generator=g).int()[None].cuda()
    cache.lens = torch.tensor([n * 8], dtype=torch.int32, device="cuda")
    q = torch.rand(1, 2, D, generator=g).add(0.5).half()
    for take in (7, 100, 451, 600):
        selection(cache, both.cuda(), q, [1], take, 1, 1, cu=False)


def test_captured_rounds_of_a_selection():
    """Tokens in more than one round, captured: every replay is the eager call's result."""
    import mqk
    lens, each = [700, 333, 5000], 200
    cache = paged_oracle.Cache(lens, 2, 64, cols=30001)
    boxes = made(cache)
    q = tokens(3, each, 4, 64).cuda()
    call = lambda: mqk.paged_select(q, boxes, cache.table, cache.lens, 16, 9)
    call()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = call()
    for i in range(4):
        q.copy_(tokens(3, each, 4, 64, seed=10 + i))
        cache.lens.sub_(7)
        got.zero_()
        g.replay()
        want = call()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
