"""Results laid over the keys' scores: refused, by the C++ front and the Python path alike."""
import pytest
import torch

import mqk
from mqk import _native

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("front", [True, False])
def test_out_over_scores(monkeypatch, front):
    if not front:
        monkeypatch.setattr(_native, "_front", None)
        monkeypatch.setattr(_native, "_front_absent", True)
    cache = mqk.kv4_cache(8, 2, 64)
    table = torch.arange(8, dtype=torch.int32, device="cuda")[None]
    lens = torch.tensor([100], dtype=torch.int32, device="cuda")
    k, v = (torch.randn(100, 2, 64, device="cuda").bfloat16() for _ in range(2))
    mqk.kv4_write(k, v, cache, table, lens)
    q = torch.randn(1, 1, 4, 64, device="cuda").bfloat16()
    mqk.kv4_attn(q, cache, table, lens, scores=torch.zeros(8, 2, 16, device="cuda"))  # (the workspace: Python makes it)
    room = torch.zeros(768, device="cuda")
    scores = room[256:512].view(8, 2, 16)
    halves = room.view(torch.bfloat16)  # two of them a score: the scores' are 512 .. 1023
    for at in (264, 512, 640, 1016):
        with pytest.raises(ValueError, match="overlap"):
            mqk.kv4_attn(q, cache, table, lens, scores=scores, out=halves[at:at + 256].view(q.shape))
        assert (room == 0).all()
    want = mqk.kv4_attn(q, cache, table, lens)
    for at in (256, 1024):  # side by side is apart
        out = halves[at:at + 256].view(q.shape)
        assert mqk.kv4_attn(q, cache, table, lens, scores=scores, out=out) is not None
        assert torch.equal(out, want)
