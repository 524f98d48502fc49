"""The prompt attention with its keys split over workgroups: every test of it again for
several numbers of parts (more than a sequence has tiles among them), and what the split
itself can get wrong."""
import math

import pytest
import torch

import mqk
import test_attn_prefill_gpu as whole
from attn_oracle import attend, check
from test_attn_prefill_gpu import *  # noqa: F401,F403

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=[2, 5, 64], autouse=True, ids=lambda n: f"parts{n}")
def split(request):
    mqk.set_option("attn_parts", request.param)
    yield request.param
    mqk.set_option("attn_parts", 0)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 80, 128, 256])
def test_few_queries_over_many_keys(dtype, D):
    new, old = [1, 40, 0, 7], [900, 1003, 50, 0]
    lens_k = [a + b for a, b in zip(new, old)]
    q, k, v = whole.make(new, lens_k, 8, 2, D, dtype)
    out = mqk.attn_prefill(q, k, v, whole.offsets(new), cu_seqlens_k=whole.offsets(lens_k))
    a = b = 0
    for n, m in zip(new, lens_k):
        if n:
            check(out[a:a + n], attend(q[a:a + n], k[b:b + m], v[b:b + m], D ** -0.5), dtype, f"{n} over {m}")
        a, b = a + n, b + m


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_infinities_in_one_part(dtype):
    """A value that is not finite in one part's keys: seen, it reaches the result whatever
    weight its part has; unseen, it does not."""
    q, k, v = whole.make([40], [700], 4, 2, 64, dtype)
    k[300:] *= 30  # (the first part's weights become small)
    v[5, 0, 3], v[690, 1, 9], v[6, 1, 60] = math.inf, -math.inf, math.nan
    out = mqk.attn_prefill(q, k, v, whole.offsets([40]), cu_seqlens_k=whole.offsets([700]))
    # (the weights of the keys before 300 are e^-100 and less for most rows, below 2^-149, the
    # smallest fp32 number: 0 times infinity, so NaN as well as infinity is right)
    assert not torch.isfinite(out[:, :2, 3]).any() and out[:, 2:, 60].isnan().all()
    assert not torch.isfinite(out[30:, 2:, 9]).any() and torch.isfinite(out[:30, 2:, 9]).all()
    mine = torch.ones_like(out, dtype=torch.bool)
    mine[:, :2, 3] = mine[:, 2:, 60] = mine[30:, 2:, 9] = False
    assert torch.isfinite(out[mine]).all()
    k[10, 0, 0] = math.nan
    out = mqk.attn_prefill(q, k, v, whole.offsets([40]), cu_seqlens_k=whole.offsets([700]))
    assert out[:, :2].isnan().all() and torch.isfinite(out[:, 2:, :9]).all()


def test_rows_behind_the_last_sequence():
    q, k, v = whole.make([300], [300], 4, 2, 128, BF16)
    cu = whole.offsets([20, 0, 150])
    new = mqk.attn_prefill(q, k, v, cu)
    mine = torch.full_like(q, 7.0)
    mqk.attn_prefill(q, k, v, cu, out=mine)
    assert (new[170:] == 0).all() and (mine[170:] == 7).all() and torch.equal(new[:170], mine[:170])


def test_captured_with_a_workspace_of_its_own():
    """Two captured calls of one stream, replayed in turn and at once with eager calls
    between them."""
    calls = []
    for seed in (1, 2):
        q, k, v = whole.make([9, 30], [600, 900], 8, 2, 128, BF16, seed=seed)
        calls.append((q, k, v, whole.offsets([9, 30]), whole.offsets([600, 900])))
    run = lambda c: mqk.attn_prefill(*c[:4], cu_seqlens_k=c[4])
    want = [run(c) for c in calls]
    graphs, outs = [], []
    for c in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(c))
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        again = [run(c) for c in calls]
        torch.cuda.synchronize()
        for o, a, w in zip(outs, again, want):
            assert torch.equal(o, w) and torch.equal(a, w)
