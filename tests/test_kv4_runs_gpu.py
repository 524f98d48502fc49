"""The 4-bit cache's long runs of tokens (written and read a page at a time), its calls
through the C++ front and captured, and outputs laid over inputs."""
import math

import pytest
import torch

import mqk
from attn_oracle import check, kv4_attend, quantise, values

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def offsets(lens):
    return torch.tensor([0] + list(lens)).cumsum(0).to(torch.int32).cuda()


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def stored(x):
    return values(quantise(x)).float().to(x.dtype)


def bits(t):
    return t.contiguous().view(torch.int16)


def pages_of(lens, seed=0, spare=3):
    """A table of scattered pages with -1 past a sequence's last one, and the pages it takes."""
    need = [-(-n // 16) for n in lens]
    ids = torch.randperm(sum(need) + spare, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(lens), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(need):
        table[i, :n] = ids[at:at + n]
        at += n
    return table.cuda(), sum(need) + spare


def tokens(T, H, D, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(T, H, D, generator=g).to(dtype).cuda() for _ in range(2)]


def fresh(blocks, H, D, dtype):
    c = mqk.kv4_cache(blocks, H, D, dtype=dtype)
    bits(c).fill_(-1)
    return c


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("H,lens", [(8, [600]), (8, [1, 511, 40, 0, 250, 16, 33]), (3, [1500]), (1, [4100, 3]),
                                    (8, [4200]), (8, [1, 2511, 40, 0, 1250, 16, 433]), (3, [11000, 17]), (1, [33000])])
def test_runs(dtype, D, H, lens):
    """Whole prompts: the bytes of the definition, those of the same tokens in small calls,
    and the values back; strided sources give the same."""
    T = sum(lens)
    table, blocks = pages_of(lens)
    k, v = tokens(T, H, D, dtype)
    one, few, packed = (fresh(blocks, H, D, dtype) for _ in range(3))
    mqk.kv4_write(k, v, one, table, i32(lens), offsets(lens))
    gk, gv = mqk.kv4_read(one, table, i32(lens), T, offsets(lens))
    assert torch.equal(gk.cpu(), stored(k)) and torch.equal(gv.cpu(), stored(v))
    at = 0
    part = 100 if T < 2000 else 997  # tokens of a small call
    for s, n in enumerate(lens):
        for a in range(0, n, part):
            b = min(n, a + part)
            mqk.kv4_write(k[at + a:at + b], v[at + a:at + b], few, table[s:s + 1], i32([b]))
            rk, rv = mqk.kv4_read(one, table[s:s + 1], i32([b]), b - a)
            assert torch.equal(rk, gk[at + a:at + b]) and torch.equal(rv, gv[at + a:at + b])
        at += n
    assert torch.equal(bits(one), bits(few))
    wide = torch.zeros(T, 2 * H + 1, D, dtype=dtype, device="cuda")
    wide[:, :H], wide[:, H:2 * H] = k, v
    mqk.kv4_write(wide[:, :H], wide[:, H:2 * H], packed, table, i32(lens), offsets(lens))
    assert torch.equal(bits(one), bits(packed))


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("have", [[0, 0, 0], [16, 5, 31], [1, 15, 17], [700, 3, 2]])
@pytest.mark.parametrize("new", [[333, 410, 95], [1333, 1410, 1495]])
def test_runs_that_continue(dtype, D, have, new):
    """New tokens behind ones that are there, from the middle of a page to the middle of one:
    nothing else in the pages changes, new tokens' scores are cleared, others' stay."""
    H = 8
    lens = [a + b for a, b in zip(have, new)]
    table, blocks = pages_of(lens, seed=1)
    k, v = tokens(sum(new), H, D, dtype, seed=2)
    cache = fresh(blocks, H, D, dtype)
    k0, v0 = tokens(max(1, sum(have)), H, D, dtype, seed=3)
    if sum(have):
        mqk.kv4_write(k0[:sum(have)], v0[:sum(have)], cache, table, i32(have), offsets(have))
    other = cache.clone()
    marks = torch.rand(blocks, H, 16, device="cuda") + 1
    before = marks.clone()
    mqk.kv4_write(k, v, cache, table, i32(lens), offsets(new), scores=marks)
    at = 0
    for s, n in enumerate(new):
        for a in range(0, n, n // 7):
            b = min(n, a + n // 7)
            mqk.kv4_write(k[at + a:at + b], v[at + a:at + b], other, table[s:s + 1], i32([have[s] + b]))
        t = torch.arange(have[s], lens[s], device="cuda")
        before[table[s].long()[t // 16], :, t % 16] = 0
        at += n
    assert torch.equal(bits(cache), bits(other))
    assert torch.equal(marks, before)
    rk, rv = mqk.kv4_read(cache, table, i32(lens), sum(new), offsets(new))
    assert torch.equal(rk.cpu(), stored(k)) and torch.equal(rv.cpu(), stored(v))


@pytest.mark.parametrize("S", [150, 1100])
def test_runs_of_equal_length(S):
    """[B, S, H, D] without offsets."""
    B, H, D = 4, 8, 128
    table, blocks = pages_of([S + 9] * B)
    k, v = tokens(B * S, H, D, BF16)
    a, b = fresh(blocks, H, D, BF16), fresh(blocks, H, D, BF16)
    mqk.kv4_write(k.view(B, S, H, D), v.view(B, S, H, D), a, table, i32([S + 9] * B))
    mqk.kv4_write(k, v, b, table, i32([S + 9] * B), offsets([S] * B))
    assert torch.equal(bits(a), bits(b))
    rk, rv = mqk.kv4_read(a, table, i32([S + 9] * B), B * S)
    assert torch.equal(rk.cpu(), stored(k)) and torch.equal(rv.cpu(), stored(v))


@pytest.mark.parametrize("times", [1, 7])
def test_runs_without_a_place(times):
    """Pages that are not there, tokens behind the last sequence and before a sequence's
    start, positions past the table: not written, read as 0; offsets out of order stay in
    bounds."""
    H, D, T, n0, n1, cap = 8, 64, 700 * times, 300 * times, 330 * times, 320 * times
    k, v = tokens(T, H, D, BF16)
    table, blocks = pages_of([cap, cap], seed=5)
    cache = fresh(blocks, H, D, BF16)
    marks = torch.full((blocks, H, 16), 7.0, device="cuda")
    holes = table.clone()
    holes[0, 3], holes[1, 0], holes[1, -1] = -1, blocks, 1 << 30
    # the first sequence's last n0 - 10 tokens have a place, the second has more than the table
    cu, lens = i32([0, n0, n0 + n1]), i32([n0 - 10, n1])
    mqk.kv4_write(k, v, cache, holes, lens, cu, scores=marks)
    rk, rv = mqk.kv4_read(cache, holes, lens, T, cu)
    want = [stored(k).cuda(), stored(v).cuda()]
    gone = torch.zeros(T, dtype=torch.bool)
    gone[:10] = gone[10 + 48:10 + 64] = True
    gone[n0:n0 + 16] = gone[n0 + cap - 16:] = True
    for got, w in zip((rk, rv), want):
        w[gone] = 0
        assert torch.equal(got, w)
    mine = torch.zeros(blocks, H, 16, dtype=torch.bool, device="cuda")
    for s, (first, n) in enumerate(((10, n0 - 10), (n0, cap))):
        for p in range(n):
            if not gone[first + p]:
                mine[table[s, p // 16], :, p % 16] = True
    assert (marks[mine] == 0).all() and (marks[~mine] == 7).all()
    keep = [i for i in range(blocks) if not mine[i].any()]
    assert (bits(cache)[keep] == -1).all()
    for odd in ([0, 500, 100], [-9, 1 << 30, 3], [T, 0, 350], [650, 690, T]):
        mqk.kv4_write(k, v, cache, holes, lens, i32(odd))
        mqk.kv4_read(cache, holes, lens, T, i32(odd))
    for n in ([-4, 1 << 30], [0, 0], [-(1 << 31), (1 << 31) - 1]):
        mqk.kv4_write(k, v, cache, holes, i32(n), cu)
        mqk.kv4_read(cache, holes, i32(n), T, cu)
    torch.cuda.synchronize()
    assert (bits(cache)[[i for i in range(blocks) if i not in table.flatten().tolist()]] == -1).all()


@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("T", [600, 4300])
def test_runs_with_groups_that_are_not_finite(dtype, T):
    H, D = 8, 128
    k, v = tokens(T, H, D, dtype)
    k[3, 1, 70], k[500, 7, 0], v[17, 0, 127], v[599, 2, 64] = math.inf, math.nan, -math.inf, math.nan
    table, blocks = pages_of([T])
    cache = fresh(blocks, H, D, dtype)
    mqk.kv4_write(k, v, cache, table, i32([T]))
    rk, rv = mqk.kv4_read(cache, table, i32([T]), T)
    for x, got in ((k, rk), (v, rv)):
        bad = ~torch.isfinite(x).unflatten(-1, (-1, 64)).all(-1, keepdim=True).expand(-1, -1, -1, 64).flatten(-2).cpu()
        got = got.cpu()
        assert got[bad].isnan().all() and torch.equal(got[~bad], stored(x)[~bad])


@pytest.mark.parametrize("dtype,D", [(BF16, 128), (F16, 64)])
@pytest.mark.parametrize("n_seqs", [1, 3, 17])
@pytest.mark.parametrize("budget,recent", [(255, 0), (300, 40), (1030, 7)])
def test_evict_few_and_many_heads(dtype, D, n_seqs, budget, recent):
    """The kept tokens' values and scores stand at the front in their order, whether the move
    is a launch of its own or not; nothing else changes, and missing pages stay missing."""
    H, lens = 8, [1100 + 37 * s for s in range(n_seqs)]
    lens[-1] = 2200
    table, blocks = pages_of(lens, seed=n_seqs)
    k, v = tokens(sum(lens), H, D, dtype)
    cache = fresh(blocks, H, D, dtype)
    marks = torch.rand(blocks, H, 16, device="cuda")
    mqk.kv4_write(k, v, cache, table, i32(lens), offsets(lens))
    k0, v0 = mqk.kv4_read(cache, table, i32(lens), sum(lens), offsets(lens))
    before, old = marks.clone(), cache.clone()
    holes = table.clone()
    holes[-1, 100], holes[-1, 3] = -1, blocks
    new, kept = mqk.kv4_evict(cache, marks, holes, i32(lens), budget, recent=recent)
    assert new.tolist() == [budget] * n_seqs
    a = 0
    for s, n in enumerate(lens):
        t = torch.arange(n, device="cuda")
        w = before[table[s].long()[t // 16], :, t % 16].t()  # [H, n]
        if s == n_seqs - 1:
            w[:, 100 * 16:101 * 16] = w[:, 48:64] = -1.0  # (the last to be kept)
        w[:, n - recent:] = 2.0
        first = w.sort(dim=1, descending=True, stable=True).indices[:, :budget].sort(dim=1).values
        assert torch.equal(kept[s].long(), first)
        at = torch.arange(budget, device="cuda")
        gk, gv = mqk.kv4_read(cache, table[s:s + 1], i32([budget]), budget)
        here = torch.ones(budget, dtype=torch.bool, device="cuda")
        if s == n_seqs - 1:
            here[48:64] = False  # (written to nowhere)
        for h in range(H):
            src = kept[s, h].long()
            assert torch.equal(gk[here, h], k0[a + src[here], h]) and torch.equal(gv[here, h], v0[a + src[here], h])
            got = marks[table[s].long()[at // 16], h, at % 16]
            assert torch.equal(got[here], before[table[s].long()[src // 16], h, src % 16][here])
        a += n
    # pages past the kept tokens, those without an owner and the missing ones are as they were
    used = torch.zeros(blocks, dtype=torch.bool)
    for s in range(n_seqs):
        used[[p for i, p in enumerate(holes[s, :-(-budget // 16)].tolist()) if 0 <= p < blocks]] = True
    assert torch.equal(bits(cache)[~used], bits(old)[~used]) and torch.equal(marks[~used], before[~used])


@pytest.mark.parametrize("n_seqs", [1, 64, 65, 200, 256, 257])
@pytest.mark.parametrize("most", [40, 900])
def test_attention_of_many_sequences(n_seqs, most):
    """The cut of the row of steps for every way of summing the lengths, tables wider than the
    sequences, with steps enough for parts of two and of more."""
    g = torch.Generator().manual_seed(n_seqs)
    lens = torch.randint(0, most, (n_seqs,), generator=g).tolist()
    lens[0], lens[-1] = 0 if n_seqs > 1 else most, 2000
    table, blocks = pages_of(lens, seed=2)
    H, D = 1, 64
    k, v = tokens(sum(lens), H, D, BF16)
    cache = fresh(blocks, H, D, BF16)
    mqk.kv4_write(k, v, cache, table, i32(lens), offsets(lens))
    q = torch.randn(n_seqs, 1, 3, D, generator=g).to(BF16).cuda()
    marks = torch.zeros(blocks, H, 16, device="cuda")
    out = mqk.kv4_attn(q, cache, table, i32(lens), scores=marks)
    at = 0
    for s, n in enumerate(lens):
        check(out[s], kv4_attend(q[s], quantise(k[at:at + n]), quantise(v[at:at + n]), D ** -0.5), BF16, f"sequence {s}")
        at += n
    # every sequence with a key gives the weights of its three rows
    held = sum(n > 0 for n in lens)
    assert abs(marks.double().sum().item() - 3 * held) < 1e-4 * held


def serving(H=2, Hq=8, D=128, n=(700, 90)):
    lens = list(n)
    table, blocks = pages_of([x + 40 for x in lens])
    k, v = tokens(sum(lens), H, D, BF16)
    cache = mqk.kv4_cache(blocks, H, D)
    marks = torch.zeros(blocks, H, 16, device="cuda")
    mqk.kv4_write(k, v, cache, table, i32(lens), offsets(lens), scores=marks)
    q = torch.randn(len(lens), 1, Hq, D, device="cuda").to(BF16)
    return table, cache, marks, q, i32(lens)


def test_ordinary_calls_are_taken():
    """The extension answers them itself, and as the Python path does."""
    from mqk import _native
    ext = _native.front()
    table, cache, marks, q, lens = serving()
    k, v = tokens(2, 2, 128, BF16, seed=9)
    want = mqk.kv4_attn(q, cache, table, lens)  # (the workspace)
    x = torch.randn(64, 6, 128, device="cuda").to(BF16)
    cu = offsets([40, 24])
    full = mqk.attn_prefill(x[:, :4], x[:, 4:5], x[:, 5:], cu)
    got = ext.attn_prefill(x[:, :4], x[:, 4:5], x[:, 5:], cu, None, None, None)
    assert torch.equal(got, full)
    for dtype in (F16, torch.float32):
        y = x.to(dtype)
        assert type(ext.attn_prefill(y[:, :4], y[:, 4:5], y[:, 5:], cu, cu, 0.5, torch.empty(64, 4, 128, dtype=dtype, device="cuda"))) is torch.Tensor
    assert type(ext.attn_prefill(x[None], x[None, :, :2], x[None, :, 2:4], None, None, None, None)) is torch.Tensor
    assert torch.equal(ext.kv4_attn(q, cache, table, lens, None, None, None), want)
    assert torch.equal(ext.kv4_attn(q[:, 0], cache, table, lens, 128 ** -0.5, marks, torch.empty_like(q[:, 0])), want[:, 0])
    assert ext.kv4_write(k, v, cache, table, lens + 1, None, marks) is True
    rk, rv = ext.kv4_read(cache, table, lens + 1, 2, None)
    assert torch.equal(rk.cpu(), stored(k)) and torch.equal(rv.cpu(), stored(v))
    new, kept = ext.kv4_evict(cache, marks, table, lens, 64, 8)
    assert new.tolist() == [64, 64] and kept.shape == (2, 2, 64)
    # and what is not ordinary is left to Python
    assert ext.kv4_attn(q.cpu(), cache, table, lens, None, None, None) is None
    assert ext.kv4_attn(q, cache, table, lens, None, None, q) is None
    assert ext.kv4_attn(q, cache, table.long(), lens, None, None, None) is None
    assert ext.attn_prefill(x[:, :4], x[:, 4:5], x[:, 5:], cu, None, None, x.view(-1)[:64 * 4 * 128].view(64, 4, 128)) is None


def test_without_the_front(monkeypatch):
    """The same results from the Python path alone."""
    from mqk import _native
    runs = []
    for alone in (False, True):
        if alone:
            monkeypatch.setattr(_native, "_front", None)
            monkeypatch.setattr(_native, "_front_absent", True)
            assert _native.front() is None
        torch.manual_seed(0)
        table, cache, marks, q, lens = serving()
        out = [mqk.kv4_attn(q, cache, table, lens, scores=marks), mqk.kv4_attn(q[:, 0], cache, table, lens, scale=0.2)]
        new, kept = mqk.kv4_evict(cache, marks, table, lens, 64, recent=8)
        out += [new, kept, *mqk.kv4_read(cache, table, new, 128), mqk.attn_prefill(q, q[:, :, :2], q[:, :, 2:4])]
        runs.append(out + [marks])
    for a, b in zip(*runs):
        assert torch.equal(a, b)


def test_captured_steps():
    """A captured serving step (write, attend and count, evict) replayed over changing inputs
    does what the eager calls do, with eager work on the same stream in between."""
    table, cache, marks, q, lens = serving()
    mine = [t.clone() for t in (cache, marks)]
    k, v = tokens(2, 2, 128, BF16, seed=4)

    def step(cache, marks, n):
        mqk.kv4_write(k, v, cache, table, n, scores=marks)
        out = mqk.kv4_attn(q, cache, table, n, scores=marks)
        return (out, *mqk.kv4_evict(cache, marks, table, n, 500, recent=20))

    now = lens + 1
    warm = [t.clone() for t in (cache, marks)]
    step(*warm, now)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(cache, marks, now)
    for i in range(4):
        k.copy_(torch.randn(k.shape, device="cuda"))
        v.copy_(torch.randn(k.shape, device="cuda"))
        q.copy_(torch.randn(q.shape, device="cuda"))
        want = step(*mine, now)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b), f"replay {i}"
        assert torch.equal(bits(cache), bits(mine[0])) and torch.equal(marks, mine[1])
        now.copy_(want[1] + 1)
    assert now.tolist() == [501, 95]


def test_captured_prompts():
    """Offsets are read at replay."""
    x = torch.randn(300, 6, 128, device="cuda").to(BF16)
    cu = offsets([100, 120, 80])
    call = lambda: mqk.attn_prefill(x[:, :4], x[:, 4:5], x[:, 5:], cu)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = call()
    for lens in ([100, 120, 80], [1, 298, 1], [0, 0, 300], [10, 20, 30]):
        cu.copy_(offsets(lens))
        x.copy_(torch.randn(x.shape, device="cuda"))
        want = call()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want), lens


def test_outputs_over_inputs_are_refused():
    table, cache, marks, q, lens = serving()
    with pytest.raises(ValueError, match="overlap"):
        mqk.kv4_attn(q, cache, table, lens, out=q)
    flat = cache.view(-1)[64:64 + q.numel()].view(q.shape)
    with pytest.raises(ValueError, match="overlap"):
        mqk.kv4_attn(q, cache, table, lens, out=flat)
    x = torch.randn(40, 4, 64, device="cuda").to(BF16)
    y = torch.randn(40, 4, 64, device="cuda").to(BF16)
    for out in (x, y):
        with pytest.raises(ValueError, match="overlap"):
            mqk.attn_prefill(x, y, y.clone(), out=out)
        with pytest.raises(ValueError, match="overlap"):
            mqk.attn_prefill(x, y.clone(), y, out=out)
    # side by side in one tensor is apart
    both = torch.empty(2, 40, 4, 64, dtype=BF16, device="cuda")
    both[0] = x
    assert torch.equal(mqk.attn_prefill(both[0], y, y, out=both[1]), mqk.attn_prefill(x, y, y))
