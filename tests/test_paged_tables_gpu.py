"""paged_tables against the same step taken token by token."""
import random

import pytest
import torch

import paged_oracle

pytestmark = pytest.mark.gpu


def step(old, new, table, free, n_tokens, page=16, cursor=None):
    """One call, compared with the oracle; returns (table, step)."""
    import mqk
    dev = "cuda"
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    bt = as_int(table)
    got = mqk.paged_tables(as_int(old), as_int(new), bt, as_int(free), n_tokens, page=page,
                           cursor=None if cursor is None else as_int([cursor]))
    want = paged_oracle.tables(old, new, table, free, n_tokens, page, cursor or 0)
    assert bt.tolist() == want[0]
    for have, ref in zip(got, (*want[1:6], [want[6]])):
        assert have.tolist() == ref
    assert got.slots.dtype == torch.int64
    return bt, got


def start(old, cols, page, rng):
    """A table with the pages of ``old`` tokens, and the free ones in no order."""
    need = [min(cols, -(-max(o, 0) // page)) for o in old]
    ids = list(range(sum(need) + 2000))
    rng.shuffle(ids)
    table = [[ids.pop() for _ in range(n)] + [-1] * (cols - n) for n in need]
    return table, ids


@pytest.mark.parametrize("B", [1, 2, 63, 64, 255, 257, 1023, 1024, 1025, 3000])
@pytest.mark.parametrize("page", [1, 5, 16, 64])
def test_steps(B, page):
    rng = random.Random(B * page)
    old = [rng.randint(0, 90) for _ in range(B)]
    new = [rng.choice([0, 1, 1, 1, rng.randint(0, 70)]) for _ in range(B)]
    cols = -(-170 // page)
    table, free = start(old, cols, page, rng)
    free += list(range(10 ** 6, 10 ** 6 + sum(new)))
    step(old, new, table, free, sum(new) + rng.choice([0, 7]), page)


def test_borders():
    """Full pages, empty sequences, numbers below 0, all at page borders."""
    rng = random.Random(1)
    old = [0, 16, 15, 17, 32, 31, -5, 0, 16]
    new = [0, 0, 1, 15, 1, 2, 3, 16, -2]
    table, free = start(old, 5, 16, rng)
    step(old, new, table, free, 38)
    step(old, new, table, free, 64)


@pytest.mark.parametrize("room", [0, 1, 17, 40, 41, 100])
def test_cut(room):
    """What does not fit the call's room is cut off, lengths and pages with it."""
    rng = random.Random(2)
    old = [10, 0, 30, 5]
    new = [20, 21, 0, 40]
    table, free = start(old, 6, 16, rng)
    step(old, new, table, free, room)


def test_short_list():
    """Pages past the end of the free list are -1 and `taken` says so."""
    old, new = [10, 0, 30], [20, 40, 40]
    table, free = start(old, 6, 16, random.Random(3))
    _, got = step(old, new, table, free[:4], 100)
    assert got.taken.item() > 4
    step(old, new, table, [], 100)
    step(old, new, table, free[:4], 100, cursor=2)
    step(old, new, table, free[:4], 100, cursor=9)


def test_narrow_table():
    """Positions past the table have no slot and take no page."""
    old, new = [10, 0, 60, 40], [100, 33, 40, 1]
    table, free = start(old, 3, 16, random.Random(4))
    step(old, new, table, free, 174)


def test_one_step_after_another():
    """The cursor and the lengths carried on, on the device, through a run of steps."""
    import mqk
    rng = random.Random(5)
    B, cols, page = 40, 30, 16
    table, free = [[-1] * cols for _ in range(B)], list(range(2000))
    rng.shuffle(free)
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    bt, lens, list_, cursor = as_int(table), as_int([0] * B), as_int(free), as_int([0])
    old, at = [0] * B, 0
    for i in range(12):
        new = [rng.randint(0, 50) if i == 0 else 1 if i % 3 else rng.randint(0, 30) for _ in range(B)]
        got = mqk.paged_tables(lens, as_int(new), bt, list_, sum(new) + 3, page=page, cursor=cursor)
        table, old, cu, seq, pos, slots, at = paged_oracle.tables(old, new, table, free, sum(new) + 3, page, at)
        lens, cursor = got.seq_lens, got.taken
        assert bt.tolist() == table and lens.tolist() == old and cursor.item() == at
        assert got.slots.tolist() == slots and got.kv_pos.tolist() == pos and got.kv_seq.tolist() == seq
        assert got.cu_seqlens.tolist() == cu
    held = [b for row in table for b in row if b >= 0]
    assert len(set(held)) == len(held) == at


def test_large_numbers():
    """Lengths near the end of int32, blocks whose slots pass 32 bits."""
    import mqk
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    bt = torch.full((2, 4), -1, dtype=torch.int32, device="cuda")
    got = mqk.paged_tables(as_int([2 ** 31 - 3, 0]), as_int([10, 20]), bt, as_int([2 ** 30, 2 ** 31 - 1]), 30, page=16)
    assert got.seq_lens.tolist() == [2 ** 31 - 1, 20] and got.cu_seqlens.tolist() == [0, 2, 22]
    assert got.slots.tolist()[:3] == [-1, -1, 2 ** 34] and got.slots[21].item() == (2 ** 31 - 1) * 16 + 3
    got = mqk.paged_tables(torch.tensor([5, 6], device="cuda"), torch.tensor([2 ** 40, 1], device="cuda"), bt,
                           as_int([7, 8]), 8, page=16)  # (int64 lengths)
    assert got.seq_lens.tolist() == [13, 6] and got.taken.item() == 0


def test_front_takes_a_step():
    """The front writes a step's keys where the slots say, and those of rows behind the last token
    nowhere."""
    import mqk
    from conftest import Case
    c = Case(1, 40, 512, 4, 2, seed=3, rows=128)
    dev = torch.device("cuda")
    old, new = [5, 0, 30], [1, 20, 15]
    as_int = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    bt = as_int([[3, -1, -1], [-1] * 3, [1, 4, -1]])
    s = mqk.paged_tables(as_int(old), as_int(new), bt, as_int([0, 7, 2, 5]), 40)
    k_cache = torch.zeros(8, 16, 2, 128, dtype=torch.bfloat16, device=dev)
    v_cache = torch.zeros_like(k_cache)
    args = [t for t in c.args(dev)[:8]]
    x = args[0].view(40, 512)
    q, k, v = mqk.fused_qkv_rope_varlen(x, *args[1:8], s.cu_seqlens, seq_pos0=as_int(old), k_cache=k_cache,
                                        v_cache=v_cache, block_table=bt, kv_seq=s.kv_seq, kv_pos=s.kv_pos)
    slots = s.slots[:36].long()
    assert torch.equal(k_cache.view(-1, 2, 128)[slots], k[:36]) and torch.equal(v_cache.view(-1, 2, 128)[slots], v[:36])
    rest = torch.ones(128, dtype=torch.bool, device=dev)
    rest[slots] = False
    assert (k_cache.view(-1, 2, 128)[rest] == 0).all()
