"""The 4-bit paged cache: writing, reading, attending, evicting, against plain 64-bit forms.

A stored value is exact to the bit: codes, scales and least values follow from the
definition, and reading rounds once.  The attention's bound counts the rounding of the
probabilities (times a scale) and of the result to the type, and the fp32 sums."""
import math
import threading

import pytest
import torch

import mqk
from attn_oracle import attend, check, kv4_attend, quantise, values

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


class Store:
    """Sequences in a cache whose bytes all start as 0xFF (scales and least values NaN)."""

    def __init__(self, lens, Hkv, D, dtype, seed=0, spare=2, cols=None, write=True):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.Hkv, self.D, self.dtype = list(lens), Hkv, D, dtype
        need = [-(-n // 16) for n in lens]
        self.cols = cols or max(1, max(need))
        self.blocks = sum(need) + spare
        ids = torch.randperm(self.blocks, generator=g)
        self.table = torch.full((len(lens), self.cols), -1, dtype=torch.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[i, :n] = ids[at:at + n].int()
            at += n
        self.table = self.table.cuda()
        self.cache = mqk.kv4_cache(self.blocks, Hkv, D, dtype=dtype)
        self.cache.view(torch.int16).fill_(-1)
        T = sum(lens)
        self.k = (torch.randn(T, Hkv, D, generator=g) * (0.5 + torch.rand(D, generator=g))).to(dtype).cuda()
        self.v = torch.randn(T, Hkv, D, generator=g).to(dtype).cuda()
        if write:
            mqk.kv4_write(self.k, self.v, self.cache, self.table, i32(self.lens), offsets(lens))

    def read(self, lens=None):
        lens = self.lens if lens is None else lens
        return mqk.kv4_read(self.cache, self.table, i32(lens), sum(lens), offsets(lens))


def same(a, b):
    """Equal, NaN where NaN."""
    return ((a == b) | (a.isnan() & b.isnan())).all()


def stored(x):
    return values(quantise(x)).float().to(x.dtype)


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Hkv", [1, 3, 8])
@pytest.mark.parametrize("lens", [[1], [16, 17], [5, 0, 40, 1, 100]])
def test_write_read(dtype, D, Hkv, lens):
    st = Store(lens, Hkv, D, dtype)
    k, v = st.read()
    assert k.dtype == dtype and k.shape == st.k.shape
    assert torch.equal(k.cpu(), stored(st.k)) and torch.equal(v.cpu(), stored(st.v))
    # token by token, equally many a sequence, from strided tensors: the same bytes
    one = mqk.kv4_cache(st.blocks, Hkv, D, dtype=dtype)
    one.view(torch.int16).fill_(-1)
    both = torch.stack((st.k, st.v), 1)
    at = offsets(lens).tolist()
    for p in range(max(lens)):
        rows = [s for s, n in enumerate(lens) if p < n]
        t = torch.tensor([at[s] + p for s in rows]).cuda()
        x = both[t]
        mqk.kv4_write(x[:, 0], x[:, 1], one, st.table[rows], i32([p + 1] * len(rows)))
    assert torch.equal(one.view(torch.int16), st.cache.view(torch.int16))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
def test_values_on_the_borders(dtype, D):
    """Constant groups, values half way between two codes, groups of far apart sizes, the
    type's largest and smallest numbers, zeros of both signs."""
    g = torch.Generator().manual_seed(4)
    top = torch.finfo(dtype).max
    rows = [torch.zeros(D), torch.full((D,), 3.25), torch.arange(D) % 31 * 0.5, torch.arange(D) % 16 * 1.0,
            -(torch.arange(D) % 30) * 0.25 + 2, torch.randint(-15, 16, (D,), generator=g) * 0.5,
            torch.randn(D, generator=g) * 1e-4, torch.randn(D, generator=g) * torch.finfo(dtype).tiny,
            torch.randn(D, generator=g).sign() * top, torch.where(torch.arange(D) % 7 == 0, top, 1.0),
            -torch.zeros(D), torch.cat([torch.randn(D - 1, generator=g) * 1e-3, torch.tensor([100.0])])]
    rows += [torch.randint(-120, 121, (D,), generator=g) * 2.0 ** -e for e in range(8)]
    x = torch.stack(rows)[:, None].to(dtype).cuda()
    n = x.shape[0]
    cache = mqk.kv4_cache(4, 1, D, dtype=dtype)
    table = torch.arange(4, dtype=torch.int32, device="cuda")[None]
    mqk.kv4_write(x, x.flip(0), cache, table, i32([n]))
    k, v = mqk.kv4_read(cache, table, i32([n]), n)
    assert torch.equal(k.cpu(), stored(x)) and torch.equal(v.cpu(), stored(x.flip(0)))


def test_group_that_is_not_finite():
    for bad in (math.inf, -math.inf, math.nan):
        for dtype in (BF16, F16):
            x = torch.randn(20, 2, 128).to(dtype).cuda()
            x[3, 1, 70] = bad
            cache = mqk.kv4_cache(2, 2, 128, dtype=dtype)
            table = i32([[1, 0]])
            mqk.kv4_write(x, x, cache, table, i32([20]))
            k, v = mqk.kv4_read(cache, table, i32([20]), 20)
            for y in (k, v):
                assert y[3, 1, 64:].isnan().all()
                y[3, 1, 64:] = 0
                want = stored(x).cuda()
                want[3, 1, 64:] = 0
                assert torch.equal(y, want)


def test_what_has_no_place_is_not_written():
    """Positions below 0 or past the table, pages that are not there, tokens behind the last
    sequence: skipped, nothing else is touched, and they read back as 0."""
    Hkv, D = 2, 64
    cache = mqk.kv4_cache(4, Hkv, D)
    cache.view(torch.int16).fill_(0x1234)
    scores = torch.full((4, Hkv, 16), 5.0, device="cuda")
    before = cache.clone()
    k = torch.randn(6, Hkv, D).bfloat16().cuda()
    table = i32([[-1, 9], [4, 1 << 30], [2, -7]])
    for lens in ([0, 0, 0], [1, 17, 33], [-5, 1 << 30, 40]):
        mqk.kv4_write(k[:3], k[:3], cache, table, i32(lens), scores=scores)
        assert (mqk.kv4_read(cache, table, i32(lens), 3)[0] == 0).all()
    mqk.kv4_write(k, k, cache, table, i32([4, 4, 4]), offsets([0, 0, 0]), scores=scores)
    assert torch.equal(cache.view(torch.int16), before.view(torch.int16)) and (scores == 5).all()
    # more new tokens than the sequence has: the first ones fall away
    mqk.kv4_write(k, k, cache, table, i32([0, 0, 4]), offsets([0, 0, 6]), scores=scores)
    got = mqk.kv4_read(cache, table, i32([0, 0, 4]), 4, offsets([0, 0, 4]))[0]
    assert torch.equal(got.cpu(), stored(k[2:]))
    assert (scores[2, :, :4] == 0).all() and (scores[2, :, 4:] == 5).all() and (scores[[0, 1, 3]] == 5).all()
    rest = cache.clone()
    rest[2] = before[2]
    assert torch.equal(rest.view(torch.int16), before.view(torch.int16))
    for cu in ([0, 3, 1, 6], [-4, 2, 9, 1 << 30], [6, 4, 2, 0]):  # offsets out of order
        mqk.kv4_write(k, k, cache, table, i32([4, 4, 4]), i32(cu))
        mqk.kv4_read(cache, table, i32([4, 4, 4]), 6, i32(cu))
    assert torch.equal(cache[[0, 1, 3]].view(torch.int16), before[[0, 1, 3]].view(torch.int16))


def queries(B, S, Hq, D, dtype, seed=1, std=1.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, S, Hq, D, generator=g) * std).to(dtype).cuda()


def verify(st, q, out, scale=None, lens=None, scores=None, before=None):
    """Every sequence against the definition on the stored codes; the scores likewise."""
    S, scale = q.shape[1], st.D ** -0.5 if scale is None else scale
    at = 0
    for b, n in enumerate(st.lens):
        m = n if lens is None else lens[b]
        kq, vq = quantise(st.k[at:at + m]), quantise(st.v[at:at + m])
        want = kv4_attend(q[b], kq, vq, scale)
        check(out[b], want, st.dtype, f"sequence {b} ({m} keys)")
        if scores is not None:
            t = torch.arange(m)
            page = st.table[b].cpu().long()[t // 16]
            got = scores.cpu().double()[page, :, t % 16] - 0
            add = want[3].sum(0).view(st.Hkv, q.shape[2] // st.Hkv, m).sum(1).t()
            base = before.cpu().double()[page, :, t % 16]
            rows = S * q.shape[2] // st.Hkv
            room = add * want[2].max() + (base.abs() + add) * (rows + 2) * 2.0 ** -24 + 1e-30
            assert ((got - base - add).abs() <= room).all(), f"scores of sequence {b}"
        at += n


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("S", [1, 2, 5])
@pytest.mark.parametrize("lens", [[1], [7, 16, 17], [300, 31, 32, 33, 129], [1000, 2, 600]])
def test_attention(dtype, D, S, lens):
    st = Store(lens, 2, D, dtype, seed=len(lens))
    q = queries(len(lens), S, 8, D, dtype)
    out = mqk.kv4_attn(q, st.cache, st.table, i32(lens))
    assert out.shape == q.shape and out.dtype == dtype
    verify(st, q, out)
    for b, n in enumerate(lens):  # tokens before the sequence's start see nothing
        assert (out[b, :max(0, S - n)] == 0).all()


@pytest.mark.parametrize("Hq,Hkv,S", [(1, 1, 1), (3, 3, 2), (16, 8, 1), (40, 8, 1), (32, 4, 3), (64, 4, 1), (64, 2, 1),
                                      (8, 1, 17), (6, 2, 40)])
def test_attention_head_layouts(Hq, Hkv, S):
    lens = [90, 40, 700]
    st = Store(lens, Hkv, 128, BF16)
    q = queries(3, S, Hq, 128, BF16)
    scores = torch.rand(st.blocks, Hkv, 16, device="cuda")
    before = scores.clone()
    out = mqk.kv4_attn(q, st.cache, st.table, i32(lens), scores=scores)
    verify(st, q, out, scores=scores, before=before)
    assert torch.equal(out, mqk.kv4_attn(q, st.cache, st.table, i32(lens)))
    if S == 1:
        assert torch.equal(out[:, 0], mqk.kv4_attn(q[:, 0], st.cache, st.table, i32(lens)))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
def test_scores(dtype, D):
    lens = [1, 513, 200, 0, 1100]
    st = Store(lens, 2, D, dtype, seed=8)
    scores = torch.rand(st.blocks, 2, 16, device="cuda")
    before = scores.clone()
    q = queries(5, 2, 6, D, dtype)
    out = mqk.kv4_attn(q, st.cache, st.table, i32(lens), scores=scores)
    verify(st, q, out, scores=scores, before=before)
    # entries of nobody's keys, and of slots past a length, stay
    mine = torch.zeros_like(scores, dtype=torch.bool)
    for b, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        mine[st.table[b].long()[t // 16], :, t % 16] = True
    assert torch.equal(scores[~mine], before[~mine])


def test_long_and_ragged():
    """Sequences of very different lengths, cut into many splits."""
    lens = [20000, 3, 4097, 0, 600]
    st = Store(lens, 2, 128, BF16, seed=3)
    q = queries(5, 1, 8, 128, BF16)
    scores = torch.zeros(st.blocks, 2, 16, device="cuda")
    before = scores.clone()
    verify(st, q, mqk.kv4_attn(q, st.cache, st.table, i32(lens), scores=scores), scores=scores, before=before)


def test_many_sequences():
    lens = [(37 * i) % 90 for i in range(300)]
    st = Store(lens, 1, 64, BF16, seed=3, cols=70)
    q = queries(300, 1, 2, 64, BF16)
    verify(st, q, mqk.kv4_attn(q, st.cache, st.table, i32(lens)))


def test_shorter_than_written():
    """Keys past seq_lens do not count; a padded entry with length 0 gives 0; lengths beyond
    the table end with it."""
    lens = [100, 64, 30]
    st = Store(lens, 2, 64, BF16)
    q = queries(3, 1, 4, 64, BF16)
    for now in ([51, 64, 0], [1, 17, 29]):
        out = mqk.kv4_attn(q, st.cache, st.table, i32(now))
        verify(st, q, out, lens=now)
    out = mqk.kv4_attn(q[:1], st.cache, st.table[:1, :6].contiguous(), i32([1 << 30]))
    st.lens, st.k, st.v = [96], st.k[:96], st.v[:96]
    verify(st, q[:1], out)
    assert (mqk.kv4_attn(q[:1], st.cache, st.table[:1], i32([-3])) == 0).all()


def test_pages_that_are_not_there():
    """Pages outside the cache hold no keys; a table of nothing else gives 0."""
    st = Store([200], 2, 128, BF16)
    q = queries(1, 1, 8, 128, BF16)
    table = st.table.clone()
    table[0, 3], table[0, 8] = -5, st.blocks
    scores = torch.zeros(st.blocks, 2, 16, device="cuda")
    out = mqk.kv4_attn(q, st.cache, table, i32([200]), scores=scores)
    keep = [t for t in range(200) if t // 16 not in (3, 8)]
    kq, vq = quantise(st.k[keep]), quantise(st.v[keep])
    check(out[0], kv4_attend(q[0], kq, vq, 128 ** -0.5), BF16, "without two pages")
    assert abs(scores.sum().item() - 8) < 1e-4
    assert (mqk.kv4_attn(q, st.cache, torch.full_like(table, 1 << 30), i32([200])) == 0).all()


def test_not_finite_keys_and_values():
    """A group of NaN in a key reaches its head's rows, one in a value its 64 dimensions;
    behind a token's limit neither reaches it."""
    lens = [70]
    st = Store(lens, 2, 128, BF16, write=False)
    q = queries(1, 3, 8, 128, BF16)
    st.v[68, 1, 70] = math.inf
    mqk.kv4_write(st.k, st.v, st.cache, st.table, i32(lens))
    out = mqk.kv4_attn(q, st.cache, st.table, i32(lens))
    assert torch.isfinite(out[0, 0]).all() and torch.isfinite(out[0, :, :4]).all()
    assert out[0, 1:, 4:, 64:].isnan().all() and torch.isfinite(out[0, :, :, :64]).all()
    st.v[68, 1, 70] = 0
    st.k[69, 0, 3] = math.nan
    mqk.kv4_write(st.k, st.v, st.cache, st.table, i32(lens))
    out = mqk.kv4_attn(q, st.cache, st.table, i32(lens))
    assert torch.isfinite(out[0, :2]).all() and torch.isfinite(out[0, 2, 4:]).all() and out[0, 2, :4].isnan().all()


@pytest.mark.parametrize("n", [33, 1025])
def test_nan_key_alone(n):
    """A key of NaN that a wave, or a part of the sequence, has for itself is not lost."""
    st = Store([n], 2, 128, BF16, write=False)
    st.k[n - 1, 0, 3] = math.nan
    mqk.kv4_write(st.k, st.v, st.cache, st.table, i32([n]))
    out = mqk.kv4_attn(queries(1, 1, 8, 128, BF16), st.cache, st.table, i32([n]))
    assert out[0, 0, :4].isnan().all() and torch.isfinite(out[0, 0, 4:]).all()


def test_scale_and_large_scores():
    lens = [150]
    st = Store(lens, 2, 64, BF16)
    q = queries(1, 1, 4, 64, BF16)
    for scale in (1.0, 1e-3, 1e-30):
        verify(st, q, mqk.kv4_attn(q, st.cache, st.table, i32(lens), scale=scale), scale=scale)
    # scores of 1e6 and more: one key holds all the weight
    big = (q * 1e6).to(BF16)
    out = mqk.kv4_attn(big, st.cache, st.table, i32(lens))
    k, v = values(quantise(st.k)), values(quantise(st.v))
    best = torch.einsum("hd,jhd->hj", big[0, 0].cpu().double(), k.repeat_interleave(2, 1)).argmax(-1)
    want = torch.stack([v[best[h], h // 2] for h in range(4)])
    assert ((out[0, 0].cpu().double() - want).abs() <= 2.0 ** -6 * v.abs().max()).all()


def test_far_pages():
    """A cache past 4 GiB: pages whose byte offsets need more than 32 bits."""
    blocks, Hkv, D = 250_000, 8, 128
    cache = torch.empty(blocks, Hkv, 9 * D, dtype=BF16, device="cuda")
    ids = [blocks - 1, 0, blocks - 2, 233_100, 116_600, blocks - 3]
    table = i32([ids])
    st = Store([90], Hkv, D, BF16)
    st.table, st.cache, st.blocks = table, cache, blocks
    mqk.kv4_write(st.k, st.v, cache, table, i32([90]))
    k, v = st.read()
    assert torch.equal(k.cpu(), stored(st.k)) and torch.equal(v.cpu(), stored(st.v))
    q = queries(1, 1, 16, D, BF16)
    scores = torch.zeros(blocks, Hkv, 16, device="cuda")
    before = torch.zeros(blocks, Hkv, 16)
    verify(st, q, mqk.kv4_attn(q, cache, table, i32([90]), scores=scores), scores=scores, before=before)
    lens, kept = mqk.kv4_evict(cache, scores, table, i32([90]), 40, recent=4)
    k2, _ = st.read([40])
    for h in range(Hkv):
        assert torch.equal(k2[:, h], k[kept[0, h].long(), h])


def test_out_and_strided_queries():
    lens = [40, 90]
    st = Store(lens, 2, 64, BF16)
    q = queries(2, 3, 4, 64, BF16)
    want = mqk.kv4_attn(q, st.cache, st.table, i32(lens))
    wide = torch.zeros(2, 3, 9, 64, dtype=BF16, device="cuda")
    wide[:, :, :4] = q
    mine = torch.empty_like(q)
    assert mqk.kv4_attn(wide[:, :, :4], st.cache, st.table, i32(lens), out=mine) is mine
    assert torch.equal(mine, want)
    assert torch.equal(want, mqk.kv4_attn(q, st.cache, st.table.long(), torch.tensor(lens).cuda()))


def expect_evict(scores, st, budget, recent):
    """New lengths and kept positions by sorting, in Python."""
    out = []
    for b, n in enumerate(st.lens):
        t = torch.arange(n)
        w = scores.cpu()[st.table[b].cpu().long()[t // 16], :, t % 16]
        for h in range(st.Hkv):
            if n <= budget:
                out.append(list(range(n)))
                continue
            key = [math.inf if math.isnan(x) else x for x in w[:n - recent, h].tolist()]
            nan = [math.isnan(x) for x in w[:n - recent, h].tolist()]
            first = sorted(range(n - recent), key=lambda i: (not nan[i], -key[i], i))[:budget - recent]
            out.append(sorted(first) + list(range(n - recent, n)))
    return out


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64), (BF16, 64), (F16, 128)])
@pytest.mark.parametrize("lens,budget,recent", [
    ([50], 16, 0), ([50], 17, 17), ([100, 20, 64, 0, 1], 33, 5), ([1500], 700, 64), ([16, 17, 48], 16, 3),
    ([3000, 1025], 1024, 0), ([40, 40], 1, 0), ([40], 1, 1), ([30], 64, 8)])
def test_evict(dtype, D, lens, budget, recent):
    st = Store(lens, 3, D, dtype, seed=budget)
    g = torch.Generator(device="cuda").manual_seed(7)
    scores = torch.rand(st.blocks, 3, 16, generator=g, device="cuda").pow(4)
    if budget % 2:  # many equal ones
        scores = (scores * 4).round() / 4
    before, cache = scores.clone(), st.cache.clone()
    k0, v0 = st.read()
    want = expect_evict(scores, st, budget, recent)
    new, kept = mqk.kv4_evict(st.cache, scores, st.table, i32(lens), budget, recent=recent)
    now = [min(n, budget) for n in lens]
    assert new.dtype == torch.int32 and new.tolist() == now
    assert kept.shape == (len(lens), 3, budget) and kept.dtype == torch.int32
    for i, w in enumerate(want):
        assert kept.view(-1, budget)[i].tolist() == w + [-1] * (budget - len(w))
    k1, v1 = st.read(now)
    a = b = 0
    for s, (n, m) in enumerate(zip(lens, now)):
        t = torch.arange(n, device="cuda")
        pages, slots = st.table[s].long()[t // 16], t % 16
        for h in range(3):
            src = kept[s, h, :m].long()
            assert torch.equal(k1[b:b + m, h], k0[a + src, h]) and torch.equal(v1[b:b + m, h], v0[a + src, h])
            w0 = before[pages, h, slots]
            assert torch.equal(scores[pages[:m], h, slots[:m]], w0[src])
        # what lies behind stays
        assert torch.equal(scores[pages[m:], :, slots[m:]], before[pages[m:], :, slots[m:]])
        if n > m:
            tail = mqk.kv4_read(st.cache, st.table[s:s + 1], i32([n]), n - m)[0]
            assert torch.equal(tail, k0[a + m:a + n])
        a, b = a + n, b + m
    free = sorted(set(range(st.blocks)) - set(st.table.flatten().tolist()))
    assert torch.equal(st.cache[free].view(torch.int16), cache[free].view(torch.int16))


def test_evict_odd_scores():
    """Zeros of both signs are equal, infinities and NaN are ordered, negative ones come last."""
    st = Store([64], 1, 64, BF16)
    row = torch.tensor([0.0, -0.0, -1.0, math.inf, 1.0, math.nan, -math.inf, 1e-45, -0.0, 0.0, math.nan, 2.0] * 6)[:64]
    for budget, recent in ((5, 0), (12, 2), (20, 3), (40, 0), (60, 1), (63, 63)):
        scores = torch.zeros(st.blocks, 1, 16, device="cuda")
        t = torch.arange(64, device="cuda")
        scores[st.table[0].long()[t // 16], 0, t % 16] = row.cuda()
        want = expect_evict(scores, st, budget, recent)
        kept = mqk.kv4_evict(st.cache.clone(), scores, st.table, i32([64]), budget, recent=recent)[1]
        assert kept[0, 0].tolist() == want[0]


def test_evict_pages_that_are_not_there():
    """Tokens of pages outside the cache rank last; nothing out of bounds is touched."""
    st = Store([100], 2, 64, BF16)
    table = st.table.clone()
    table[0, 1], table[0, 5] = -1, 1 << 30
    scores = torch.rand(st.blocks, 2, 16, device="cuda") + 1
    new, kept = mqk.kv4_evict(st.cache, scores, table, i32([100]), 30)
    assert new.tolist() == [30]
    lost = (kept // 16 == 1) | (kept // 16 == 5)
    assert not lost.any() and (kept >= 0).all()
    mqk.kv4_evict(st.cache, scores, table, i32([1 << 30]), 30)
    mqk.kv4_evict(st.cache, scores, table, i32([-4]), 30)
    torch.cuda.synchronize()


def test_serving_run():
    """Prompts through the front, the prompt attention and the cache, decode steps that keep
    count of the weights, eviction, and decoding on: each step against the definition on what
    the cache holds."""
    g = torch.Generator().manual_seed(0)
    hidden, Hq, Hkv, D = 512, 8, 2, 128
    w = [(torch.randn(h * D, hidden, generator=g) * 0.05).bfloat16().cuda() for h in (Hq, Hkv, Hkv)]
    one = torch.ones(D, dtype=BF16, device="cuda")
    cos, sin = (t.bfloat16().cuda() for t in mqk.rope_tables(D, 256))
    prompts = [50, 33, 90]
    x = torch.randn(sum(prompts), hidden, generator=g).bfloat16().cuda()
    cu = offsets(prompts)
    q, k, v = mqk.fused_qkv_rope_varlen(x, *w, one, one, cos, sin, cu)
    out = mqk.attn_prefill(q, k, v, cu)
    a = 0
    for n in prompts:
        check(out[a:a + n], attend(q[a:a + n], k[a:a + n], v[a:a + n], D ** -0.5), BF16, "prompt")
        a += n
    blocks, cols = 30, 10
    cache = mqk.kv4_cache(blocks, Hkv, D)
    scores = torch.zeros(blocks, Hkv, 16, device="cuda")
    table = torch.randperm(blocks, generator=g).int().view(3, cols).cuda()
    lens = i32(prompts)
    mqk.kv4_write(k, v, cache, table, lens, cu, scores=scores)
    got = mqk.kv4_read(cache, table, lens, sum(prompts), cu)
    assert torch.equal(got[0].cpu(), stored(k)) and torch.equal(got[1].cpu(), stored(v))
    place = list(prompts)  # positions of the next tokens, which eviction does not change
    for step in range(8):
        if step == 4:
            lens, kept = mqk.kv4_evict(cache, scores, table, lens, 40, recent=8)
            assert lens.tolist() == [40, 37, 40]
        x = torch.randn(3, 1, hidden, generator=g).bfloat16().cuda()
        q, k, v = mqk.fused_qkv_rope(x, *w, one, one, cos, sin, i32(place))
        lens = lens + 1
        place = [p + 1 for p in place]
        mqk.kv4_write(k, v, cache, table, lens, scores=scores)
        out = mqk.kv4_attn(q, cache, table, lens, scores=scores)
        held = lens.tolist()
        # (read back exactly: the oracle quantises them again to the same codes only where the
        # stored values' own range is unchanged, so it takes the values as they are)
        kk, vv = mqk.kv4_read(cache, table, lens, sum(held), offsets(held))
        a = 0
        for b, n in enumerate(held):
            o, A, slack, p = attend(q[b], kk[a:a + n], vv[a:a + n], D ** -0.5)
            # kk and vv are rounded to bf16 once more: half an eps of each key's part of a
            # score (to first order its largest part, over D terms) and of each value
            kmag = (q[b].double().abs().cpu()[:, :, None] * kk[a:a + n].double().abs().cpu()
                    .repeat_interleave(Hq // Hkv, 1).permute(1, 0, 2)[None]).sum(-1).amax(-1) * D ** -0.5
            check(out[b], (o, A + vv[a:a + n].abs().max().double().cpu() * 3, slack + 2.0 ** -8 + 2.0 ** -7 * kmag[..., None]),
                  BF16, f"step {step}")
            a += n
    total = sum(scores[table[b].long()].sum().item() for b in range(3))
    assert total > 0 and torch.isfinite(scores).all()


def test_prompt_that_continues_over_the_cache():
    """The values of a cached prefix, and a prompt's next tokens attending over them."""
    lens = [70, 40]
    st = Store(lens, 2, 128, BF16)
    k, v = st.read()
    new = [9, 30]
    q = queries(1, sum(new), 8, 128, BF16)[0]
    out = mqk.attn_prefill(q, k, v, offsets(new), cu_seqlens_k=offsets(lens))
    a = b = 0
    for n, m in zip(new, lens):
        check(out[a:a + n], attend(q[a:a + n], k[b:b + m], v[b:b + m], 128 ** -0.5), BF16, "continued")
        a, b = a + n, b + m


def test_same_bits_again_and_on_other_streams():
    lens = [3000, 700, 1]
    st = Store(lens, 4, 128, BF16)
    q = queries(3, 1, 16, 128, BF16)
    want = mqk.kv4_attn(q, st.cache, st.table, i32(lens))
    n = i32(lens)
    for _ in range(5):
        assert torch.equal(want, mqk.kv4_attn(q, st.cache, st.table, n))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [mqk.kv4_attn(q, st.cache, st.table, n) for _ in range(3)]
    here = [mqk.kv4_attn(q, st.cache, st.table, n) for _ in range(3)]
    side.synchronize()
    torch.cuda.synchronize()
    assert all(torch.equal(want, x) for x in got + here)


def test_two_graphs():
    """Two captured decode steps share no workspace; replayed in turn and at once, with eager
    calls between, each gives its own results.  Lengths are read at replay."""
    stores = [Store([2500, 40], 2, 128, BF16, seed=s) for s in (1, 2)]
    qs = [queries(2, 1, 8, 128, BF16, seed=s) for s in (1, 2)]
    lens = [i32([2500, 40]) for _ in stores]
    graphs, outs, marks = [], [], []
    for st, q, n in zip(stores, qs, lens):
        mark = torch.zeros(st.blocks, 2, 16, device="cuda")
        mqk.kv4_attn(q, st.cache, st.table, n)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mqk.kv4_attn(q, st.cache, st.table, n, scores=mark)
        graphs.append(graph), outs.append(out), marks.append(mark)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for now in ([2500, 40], [1111, 1], [2499, 0]):
        for n in lens:
            n.copy_(i32(now))
        want = [mqk.kv4_attn(q, st.cache, st.table, n) for st, q, n in zip(stores, qs, lens)]
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for out, w in zip(outs, want):
            assert torch.equal(out, w)
    # three steps of 8 rows of weight 1 for the first sequence, two for the second
    for mark in marks:
        assert abs(mark.sum().item() - (3 + 2) * 8) < 1e-3


def test_threads_on_one_stream():
    """Calls of several launches from several threads that share the stream's workspace."""
    stores = [Store([1500 + 100 * i], 2, 128, BF16, seed=i) for i in range(4)]
    qs = [queries(1, 1, 8, 128, BF16, seed=i) for i in range(4)]
    lens = [i32(st.lens) for st in stores]
    want = [mqk.kv4_attn(q, st.cache, st.table, n) for st, q, n in zip(stores, qs, lens)]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        for _ in range(150):
            if not torch.equal(mqk.kv4_attn(qs[i], stores[i].cache, stores[i].table, lens[i]), want[i]):
                bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad


def test_refusals():
    st = Store([20], 2, 64, BF16)
    n = i32([20])
    q = queries(1, 1, 4, 64, BF16)
    s = torch.zeros(st.blocks, 2, 16, device="cuda")
    c, t, k = st.cache, st.table, st.k
    cases = [
        (ValueError, lambda: mqk.kv4_cache(4, 2, 96)),
        (TypeError, lambda: mqk.kv4_cache(4, 2, 64, dtype=torch.float32)),
        (ValueError, lambda: mqk.kv4_cache(0, 2, 64)),
        (TypeError, lambda: mqk.kv4_write(k.half(), k, c, t, n)),
        (ValueError, lambda: mqk.kv4_write(k[:, :1], k[:, :1], c, t, n)),
        (ValueError, lambda: mqk.kv4_write(k, k[:5], c, t, n)),
        (ValueError, lambda: mqk.kv4_write(k, k, c.cpu(), t, n)),
        (ValueError, lambda: mqk.kv4_write(k, k, c[:, :, :100], t, n)),
        (ValueError, lambda: mqk.kv4_write(k, k, c[:, 1:], t, n)),
        (TypeError, lambda: mqk.kv4_write(k, k, c.view(torch.int16), t, n)),
        (ValueError, lambda: mqk.kv4_write(k, k, c, t[0], n)),
        (TypeError, lambda: mqk.kv4_write(k, k, c, t.float(), n)),
        (ValueError, lambda: mqk.kv4_write(k, k, c, t, i32([20, 20]))),
        (ValueError, lambda: mqk.kv4_write(k, k, c, t, n, offsets([10, 10]))),
        (ValueError, lambda: mqk.kv4_write(k[:3], k[:3], c, t.expand(2, -1), i32([3, 3]))),
        (TypeError, lambda: mqk.kv4_write(k, k, c, t, n, scores=s.half())),
        (ValueError, lambda: mqk.kv4_write(k, k, c, t, n, scores=s[:, :1])),
        (ValueError, lambda: mqk.kv4_read(c, t, n, -1)),
        (ValueError, lambda: mqk.kv4_attn(q[..., :32], c, t, n)),
        (ValueError, lambda: mqk.kv4_attn(q[:, :, :3], c, t, n)),
        (TypeError, lambda: mqk.kv4_attn(q.half(), c, t, n)),
        (ValueError, lambda: mqk.kv4_attn(q.expand(2, -1, -1, -1), c, t, n)),
        (ValueError, lambda: mqk.kv4_attn(q[0, 0], c, t, n)),
        (ValueError, lambda: mqk.kv4_attn(q, c, t, n, scale=-1.0)),
        (ValueError, lambda: mqk.kv4_attn(q, c, t, n.cpu())),
        (ValueError, lambda: mqk.kv4_attn(q, c, t, n, out=q[:, :, :2])),
        (ValueError, lambda: mqk.kv4_evict(c, s, t, n, 0)),
        (ValueError, lambda: mqk.kv4_evict(c, s, t, n, 8, recent=9)),
        (ValueError, lambda: mqk.kv4_evict(c, s, t, n, 8, recent=-1)),
        (TypeError, lambda: mqk.kv4_evict(c, None, t, n, 8)),
    ]
    for i, (exc, fn) in enumerate(cases):
        with pytest.raises(exc):
            fn()
            pytest.fail(f"case {i} was taken")


def test_nothing_to_do():
    c = mqk.kv4_cache(2, 2, 64)
    none = torch.empty(0, 3, dtype=torch.int32, device="cuda")
    e = torch.empty(0, 2, 64, dtype=BF16, device="cuda")
    n = i32([])
    mqk.kv4_write(e, e, c, none, n)
    assert mqk.kv4_read(c, none, n, 0)[0].shape == (0, 2, 64)
    assert mqk.kv4_attn(e[:, None], c, none, n).shape == (0, 1, 2, 64)
    s = torch.zeros(2, 2, 16, device="cuda")
    assert mqk.kv4_evict(c, s, none, n, 4)[1].shape == (0, 2, 4)
