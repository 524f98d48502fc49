"""Decode over sequences whose length goes past their table: the new tokens are the last of
that length, though the last keys have no place."""
import pytest
import torch

import kv4_bounds as kb
import mqk
from attn_oracle import quantise

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("cols", [1, 5, 70])
@pytest.mark.parametrize("S,over", [(4, 4), (5, 2), (3, 10), (20, 7), (1, 1)])
def test_lengths_past_the_table(dtype, cols, S, over):
    H, G, D, cap = 2, 4, 64, cols * 16
    g = torch.Generator().manual_seed(cols)
    lens = [cap + over, cap, max(1, cap - 9)]
    k, v = (torch.randn(3 * cap, H, D, generator=g).to(dtype).cuda() for _ in range(2))
    table = torch.randperm(3 * cols + 2, generator=g)[:3 * cols].int().view(3, cols).cuda()
    cache = mqk.kv4_cache(3 * cols + 2, H, D, dtype=dtype)
    mqk.kv4_write(k, v, cache, table, torch.tensor([cap] * 3, dtype=torch.int32, device="cuda"))
    q = torch.randn(3, S, H * G, D, generator=g).to(dtype).cuda()
    scores = torch.zeros(3 * cols + 2, H, 16, device="cuda")
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    out = mqk.kv4_attn(q, cache, table, n, scores=scores)
    assert torch.equal(out, mqk.kv4_attn(q, cache, table, n))
    for s, m in enumerate(lens):
        held = min(m, cap)
        kq, vq = (quantise(x[s * cap:s * cap + held]) for x in (k, v))
        limit = m - S + 1 + torch.arange(S)
        want, room, P, e = kb.attend(q[s], kq, vq, D ** -0.5, dtype, limit)
        assert kb.ratio(out[s], want, room) <= 1, f"sequence {s}"
        assert (out[s].cpu()[limit <= 0] == 0).all()
        add, rel = kb.added(P, e, H)
        t = torch.arange(held)
        got = scores.cpu().double()[table[s].cpu().long()[t // 16], :, t % 16]
        assert ((got - add).abs() <= add * rel + add * (S * G + 2) * kb.U).all(), f"weights of sequence {s}"


def test_one_row_more_key_by_key():
    """Lengths one and two past the table: the first token sees what a call of that token alone
    with its own length sees, to the bit."""
    H, G, D, cols = 2, 2, 128, 3
    cap = cols * 16
    g = torch.Generator().manual_seed(1)
    k, v = (torch.randn(cap, H, D, generator=g).to(BF16).cuda() for _ in range(2))
    table = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    cache = mqk.kv4_cache(3, H, D)
    one = lambda n: torch.tensor([n], dtype=torch.int32, device="cuda")
    mqk.kv4_write(k, v, cache, table, one(cap))
    q = torch.randn(1, 4, H * G, D, generator=g).to(BF16).cuda()
    for over in (0, 1, 2, 3, 4, 9):
        out = mqk.kv4_attn(q, cache, table, one(cap + over))
        for s in range(4):
            want = mqk.kv4_attn(q[:, s:s + 1], cache, table, one(cap + over - 3 + s))
            assert torch.equal(out[:, s:s + 1], want), (over, s)
