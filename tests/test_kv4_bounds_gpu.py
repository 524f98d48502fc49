"""Decode attention against the bound that counts its roundings one by one (kv4_bounds.py;
test_kv4_bounds.py has what that bound turns down): lengths over every cut into parts, both
types, rows past one block of 16, the second term of fp16, every key's weight, and a serving
run on the stored values themselves."""
import pytest
import torch

import kv4_bounds as kb
import mqk
from attn_oracle import quantise
from test_kv4_bounds import alike

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


class Store:
    """Sequences in scattered pages of a cache that starts as NaN, in tables of ``cols`` columns."""

    def __init__(self, lens, k, v, cols=None):
        H, D = k.shape[1:]
        need = [-(-n // 16) for n in lens]
        self.lens, self.k, self.v, self.H, self.D, self.dtype = lens, k, v, H, D, k.dtype
        self.blocks = sum(need) + 2
        ids = torch.randperm(self.blocks, generator=torch.Generator().manual_seed(len(lens))).int()
        table = torch.full((len(lens), cols or max(1, max(need))), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            table[i, :n] = ids[at:at + n]
            at += n
        self.table = table.cuda()
        self.cache = mqk.kv4_cache(self.blocks, H, D, dtype=k.dtype)
        self.cache.view(torch.int16).fill_(-1)
        mqk.kv4_write(k.cuda(), v.cuda(), self.cache, self.table, i32(lens), offsets(lens))

    def attend(self, q, what="", scores=False):
        """Decodes and checks every sequence, and with ``scores`` every key's weight."""
        marks = torch.rand(self.blocks, self.H, 16, device="cuda") if scores else None
        before = marks.clone() if scores else None
        q = q.cuda()
        out = mqk.kv4_attn(q, self.cache, self.table, i32(self.lens), scores=marks)
        at = 0
        for b, n in enumerate(self.lens):
            kq, vq = quantise(self.k[at:at + n]), quantise(self.v[at:at + n])
            want, room, P, e = kb.attend(q[b], kq, vq, self.D ** -0.5, self.dtype)
            off = kb.ratio(out[b], want, room)
            assert off <= 1, f"{what} sequence {b} of {n} keys: {off:.3g} times the bound"
            if scores:
                add, rel = kb.added(P, e, self.H)
                t = torch.arange(n)
                page = self.table[b].cpu().long()[t // 16]
                got, base = (x.cpu().double()[page, :, t % 16] for x in (marks, before))
                room = add * rel + (base + add) * (q.shape[1] * q.shape[2] + 2) * kb.U
                assert ((got - base - add).abs() <= room).all(), f"{what} weights of sequence {b}"
                before[page.cuda(), :, t.cuda() % 16] = marks[page.cuda(), :, t.cuda() % 16]
            at += n
        if scores:  # nobody else's entries
            assert torch.equal(marks, before)
        return out


def store(lens, H, D, dtype, cols=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    T = sum(lens)
    k = torch.randn(T, H, D, generator=g) * (0.5 + torch.rand(D, generator=g))
    v, at = torch.randn(T, H, D, generator=g), 0
    for n in lens:
        v[at:at + n] = kb.marked(v[at:at + n], 6.0)
        at += n
    return Store(lens, k.to(dtype), v.to(dtype), cols)


def queries(B, S, Hq, D, dtype, std=1.5, seed=1):
    return (torch.randn(B, S, Hq, D, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [1, 5])
@pytest.mark.parametrize("lens", [[1, 17, 128], [700, 129, 0, 33], [20000, 3, 4097, 0, 600], [1025], [2600, 2300]])
def test_lengths(dtype, D, S, lens):
    store(lens, 2, D, dtype, seed=len(lens)).attend(queries(len(lens), S, 8, D, dtype), scores=True)


@pytest.mark.parametrize("Hq,Hkv,S", [(64, 4, 1), (64, 2, 2), (8, 1, 17), (40, 8, 1)])
def test_head_layouts(Hq, Hkv, S):
    store([900, 2100, 31], Hkv, 128, BF16).attend(queries(3, S, Hq, 128, BF16), scores=True)


@pytest.mark.parametrize("m", [1, 20, 300, 1500, 4097, 20000])
def test_second_term_of_fp16(m):
    q, k, v, _ = alike(m)
    Store([m], k, v).attend(q[None])


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("B,H,cols", [(2, 2, 5000), (2, 2, 20000), (9, 1, 3000), (40, 4, 500), (1, 1, 16384), (1, 1, 16385)])
def test_weights_in_wide_tables(dtype, B, H, cols):
    """Tables as wide as the longest sequence a server allows: longer runs of pages a wave."""
    lens = [(1900 * (i + 1) + 37 * i) % 2600 for i in range(B)]
    lens[0] = min(cols * 16, 4100)
    assert max(lens) <= cols * 16
    store(lens, H, 64, dtype, cols=cols).attend(queries(B, 2, 2 * H, 64, dtype), scores=True)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_serving_run(dtype):
    """Prompts, decode steps that keep count of the weights, an eviction, and more steps: the
    reference holds the same stored codes, gathered as the eviction says."""
    g = torch.Generator().manual_seed(3)
    Hq, H, D, budget, recent = 8, 2, 128, 700, 40
    lens = [1200, 90, 701]
    need = [(n + 20 + 15) // 16 for n in lens]
    table = torch.full((3, max(need)), -1, dtype=torch.int32)
    ids, at = torch.randperm(sum(need), generator=g).int(), 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    table = table.cuda()
    cache = mqk.kv4_cache(sum(need), H, D, dtype=dtype)
    marks = torch.zeros(sum(need), H, 16, device="cuda")
    new = lambda n: [torch.randn(n, H, D, generator=g).to(dtype) for _ in range(2)]
    k, v = new(sum(lens))
    mqk.kv4_write(k.cuda(), v.cuda(), cache, table, i32(lens), offsets(lens), scores=marks)
    held = [list(x) for x in zip(k.split(lens), v.split(lens))]  # the tokens of each sequence
    for step in range(8):
        if step == 4:
            n, kept = mqk.kv4_evict(cache, marks, table, i32(lens), budget, recent=recent)
            lens = [min(x, budget) for x in lens]
            assert n.tolist() == lens
            for b, m in enumerate(lens):
                src = kept[b, :, :m].cpu().long().t()[..., None].expand(-1, -1, D)
                held[b] = [x.gather(0, src) for x in held[b]]
        lens = [n + 1 for n in lens]
        k, v = new(3)
        mqk.kv4_write(k.cuda(), v.cuda(), cache, table, i32(lens), scores=marks)
        held = [[torch.cat((x, y[b:b + 1])) for x, y in zip(held[b], (k, v))] for b in range(3)]
        q = queries(3, 1, Hq, D, dtype, std=2.0, seed=step)
        out = mqk.kv4_attn(q.cuda(), cache, table, i32(lens), scores=marks)
        for b in range(3):
            want, room, _, _ = kb.attend(q[b], *(quantise(x) for x in held[b]), D ** -0.5, dtype)
            off = kb.ratio(out[b], want, room)
            assert off <= 1, f"step {step}, sequence {b}: {off:.3g} times the bound"
