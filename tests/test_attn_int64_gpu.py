"""Tables, lengths and offsets of int64 whose numbers int32 does not hold: no page, and beyond
every length, never the page or the length that their lower half names."""
import pytest
import torch

import mqk

pytestmark = pytest.mark.gpu
H, D = 2, 64


def i64(x):
    return torch.tensor(x, dtype=torch.int64, device="cuda")


@pytest.mark.parametrize("far", [1 << 32, -(1 << 32), (1 << 32) + 2, (1 << 40) + 1, (1 << 63) - 1, -(1 << 63)])
def test_pages(far):
    k, v = (torch.randn(48, H, D, device="cuda").bfloat16() for _ in range(2))
    cache = mqk.kv4_cache(4, H, D)
    scores = torch.ones(4, H, 16, device="cuda")
    mqk.kv4_write(k, v, cache, i64([[3, 0, 2]]), i64([48]))
    before = cache.clone()
    table = i64([[3, far, 2]])
    # the same as with a page that is outside the cache
    hole = torch.tensor([[3, -1, 2]], dtype=torch.int32, device="cuda")
    mqk.kv4_write(k[16:32].neg(), v[16:32], cache, table, i64([32]), scores=scores)
    assert torch.equal(cache.view(torch.int16), before.view(torch.int16)) and (scores == 1).all()
    for a, b in zip(mqk.kv4_read(cache, table, i64([48]), 48), mqk.kv4_read(cache, hole, i64([48]), 48)):
        assert torch.equal(a, b) and (a[16:32] == 0).all()
    q = torch.randn(1, 4, D, device="cuda").bfloat16()
    assert torch.equal(mqk.kv4_attn(q, cache, table, i64([48])), mqk.kv4_attn(q, cache, hole, i64([48])))
    new, kept = mqk.kv4_evict(cache, scores, table, i64([48]), 40)
    assert new.tolist() == [32] and not ((kept >= 16) & (kept < 32)).any()


def test_lengths_and_offsets():
    k, v = (torch.randn(32, H, D, device="cuda").bfloat16() for _ in range(2))
    cache = mqk.kv4_cache(2, H, D)
    table = i64([[1, 0]])
    mqk.kv4_write(k, v, cache, table, i64([32]))
    q = torch.randn(1, 4, D, device="cuda").bfloat16()
    want = mqk.kv4_attn(q, cache, table, i64([32]))
    assert torch.equal(mqk.kv4_attn(q, cache, table, i64([(1 << 32) + 3])), want)
    assert (mqk.kv4_attn(q, cache, table, i64([-(1 << 32) + 3])) == 0).all()
    x = torch.randn(20, 4, D, device="cuda").bfloat16()
    cu = [0, 5, 20]
    assert torch.equal(mqk.attn_prefill(x, x, x, i64(cu)), mqk.attn_prefill(x, x, x, i64([0, 5, (1 << 32) + 20])))
