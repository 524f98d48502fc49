"""The paged operators together, as serving uses them, captured and replayed, on several streams,
and their refusals with tensors on the GPU."""
import threading

import pytest
import torch

import attn_oracle
import paged_oracle
from test_paged_attn_gpu import queries, run

pytestmark = pytest.mark.gpu

HIDDEN, H_Q, H_KV, D = 512, 8, 2, 128


class Model:
    """One layer's front with its paged cache, free pages and lengths."""

    def __init__(self, B, cols, seed=0):
        from conftest import Case
        c = Case(1, 1, HIDDEN, H_Q, H_KV, seed=seed, rows=cols * 16)
        self.weights = c.args(torch.device("cuda"))[1:8]
        blocks = B * cols + 5
        z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")
        self.k, self.v = z(blocks, 16, H_KV, D), z(blocks, 16, H_KV, D)
        self.bounds = z(blocks, H_KV, 2, D)
        self.table = torch.full((B, cols), -1, dtype=torch.int32, device="cuda")
        g = torch.Generator().manual_seed(seed)
        self.free = torch.randperm(blocks, generator=g).int().cuda()
        self.lens, self.cursor = z(B, dtype=torch.int32), z(1, dtype=torch.int32)

    def step(self, x, new, take=None):
        """x [n_tokens, HIDDEN] of ``new`` tokens a sequence; the lengths and the cursor go on."""
        import mqk
        s = mqk.paged_tables(self.lens, new, self.table, self.free, x.shape[0], cursor=self.cursor)
        q, _, _ = mqk.fused_qkv_rope_varlen(x, *self.weights, s.cu_seqlens, seq_pos0=self.lens, k_cache=self.k,
                                            v_cache=self.v, block_table=self.table, kv_seq=s.kv_seq, kv_pos=s.kv_pos,
                                            return_kv=False)
        mqk.paged_bounds(self.k, self.bounds, self.table, s.seq_lens, x.shape[0], cu_seqlens=s.cu_seqlens)
        pages = None
        if take is not None:
            pages = mqk.paged_select(q, self.bounds, self.table, s.seq_lens, 16, take, s.cu_seqlens)
        out = mqk.paged_attn(q, self.k, self.v, self.table, s.seq_lens, s.cu_seqlens, pages=pages)
        self.lens.copy_(s.seq_lens)
        self.cursor.copy_(s.taken)
        return q, out, pages

    def rows(self):
        """A paged_oracle cache with what the pages hold now."""
        c = paged_oracle.Cache.__new__(paged_oracle.Cache)
        c.lens_list, c.page, c.dtype, c.cols = self.lens.tolist(), 16, torch.bfloat16, self.table.shape[1]
        table = self.table.cpu().long()
        k, v = self.k.cpu(), self.v.cpu()
        c.k_rows, c.v_rows = [], []
        for s, n in enumerate(c.lens_list):
            ids = table[s, :-(-n // 16)]
            assert (ids >= 0).all()
            c.k_rows.append(k[ids].flatten(0, 1)[:n])
            c.v_rows.append(v[ids].flatten(0, 1)[:n])
        return c


def tokens(n, seed):
    return torch.randn(n, HIDDEN, generator=torch.Generator().manual_seed(seed)).bfloat16().cuda()


def numbers(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("take", [None, 4])
def test_serving(take):
    """Prompts, then decode steps with a prompt that goes on, padded rows behind the last token."""
    m = Model(5, 24)
    steps = [([70, 0, 33, 16, 1], 0), ([1, 200, 1, 1, 1], 7), ([1, 1, 100, 1, 1], 0), ([1, 1, 1, 0, 1], 3), ([3, 3, 3, 3, 3], 0)]
    for i, (new, pad) in enumerate(steps):
        n = sum(new)
        q, out, pages = m.step(tokens(n + pad, i), numbers(new), take)
        c = m.rows()
        want = paged_oracle.attend(c, q[:n].cpu(), new, D ** -0.5) if pages is None else \
            paged_oracle.attend_pages(c, q[:n].cpu(), new, pages[:n].cpu(), D ** -0.5)
        attn_oracle.check(out[:n], want, torch.bfloat16, (i, new))
        assert (out[n:] == 0).all()
        if pages is not None:
            assert (pages[n:] == -1).all()
            boxes = m.bounds.float().cpu()
            for s, length in enumerate(c.lens_list):
                for j in range(-(-length // 16)):
                    assert torch.equal(boxes[int(m.table[s, j])], paged_oracle.bounds(c, s, j))
    held = m.table[m.table >= 0]
    assert held.unique().numel() == held.numel() == m.cursor.item()


@pytest.mark.parametrize("take", [None, 6])
@pytest.mark.parametrize("each", [1, 40])
def test_captured_step(take, each):
    """A whole step as a graph: its replays follow the lengths and tables on the device."""
    B = 6
    a, b = Model(B, 40), Model(B, 40)
    for m in (a, b):  # (eager calls first: the front's workspace)
        m.step(tokens(90, 0), numbers([40, 1, 9, 0, 24, 16]), take)
        m.step(tokens(B * each, 1), numbers([each] * B), take)
    x, new = tokens(B * each, 2), numbers([each] * B)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        a.step(x, new, take)
        b.step(x, new, take)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=s):
        q, out, pages = a.step(x, new, take)
    for i in range(4):
        new.copy_(numbers([each if (i + j) % 3 else max(1, each // 2) for j in range(B)]))
        x.copy_(tokens(B * each, 10 + i))
        g.replay()
        q1, want, pages1 = b.step(x, new, take)
        torch.cuda.synchronize()
        n = int(new.sum())
        assert torch.equal(a.lens, b.lens) and torch.equal(a.table, b.table) and torch.equal(a.cursor, b.cursor)
        assert torch.equal(a.k, b.k) and torch.equal(a.bounds, b.bounds)
        assert torch.equal(q[:n], q1[:n]) and torch.equal(out, want)
        if take is not None:
            assert torch.equal(pages, pages1)


def test_two_graphs():
    """Two graphs replayed in turn and on two streams at once share nothing."""
    import mqk
    made = []
    for seed in range(2):
        cache = paged_oracle.Cache([4000, 300, 70], 2, 128, seed=seed)
        q = queries(3 + 160, 8, 128, seed=seed).cuda()
        boxes = torch.zeros(cache.blocks, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
        mqk.paged_bounds(cache.k, boxes, cache.table, cache.lens)
        cu = paged_oracle.offsets([100, 60, 3])

        def calls():
            pages = mqk.paged_select(q, boxes, cache.table, cache.lens, 16, 9, cu)
            return (mqk.paged_attn(q[:3], cache.k, cache.v, cache.table, cache.lens), pages,
                    mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens, cu),
                    mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens, cu, pages=pages))
        want = [t.clone() for t in calls()]
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = calls()
        made.append((g, got, want, cache, q, boxes, cu))
    streams = [torch.cuda.Stream() for _ in made]
    for i in range(6):
        for _, got, *_ in made:
            for t in got:
                t.zero_()
        torch.cuda.synchronize()
        for s, (g, *_) in zip(streams, made):
            with torch.cuda.stream(s if i % 2 else torch.cuda.current_stream()):
                g.replay()
        torch.cuda.synchronize()
        for _, got, want, *_ in made:
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_streams_and_threads():
    """Calls from several host threads, each on a stream of its own."""
    import mqk
    cases = []
    for seed in range(4):
        cache = paged_oracle.Cache([2000 + 100 * seed, 50], 2, 64, seed=seed)
        q = queries(2, 8, 64, seed=seed).cuda()
        cases.append((cache, q, mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens)))
    torch.cuda.synchronize()
    wrong = []

    def work(cache, q, want):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(30):
                got = mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens)
                s.synchronize()
                if not torch.equal(got, want):
                    wrong.append(1)
    threads = [threading.Thread(target=work, args=c) for c in cases]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


@pytest.mark.parametrize("kind", ["int64", "unaligned", "strided"])
def test_forms_of_the_same_numbers(kind):
    """Lengths, tables, offsets and lists of int64, at odd addresses, or strided: the same results."""
    import mqk
    cache = paged_oracle.Cache([300, 90, 17], 2, 128)
    new = [3, 40, 1]
    q = queries(44, 8, 128).cuda()
    cu, free = paged_oracle.offsets(new), numbers([9, 8, 7, 6, 5, 4, 3, 2])
    boxes = torch.zeros(cache.blocks, 2, 2, 128, dtype=torch.bfloat16, device="cuda")

    def form(t):
        if kind == "int64":
            return t.long()
        if kind == "unaligned":
            x = torch.zeros(t.numel() + 1, dtype=t.dtype, device="cuda")
            x[1:] = t.flatten()
            return x[1:].view(t.shape)
        return torch.stack([t, t], -1)[..., 0]

    def calls(f):
        mqk.paged_bounds(cache.k, boxes, f(cache.table), f(cache.lens), 44, cu_seqlens=f(cu))
        pages = mqk.paged_select(q, boxes, f(cache.table), f(cache.lens), 16, 3, f(cu))
        bt = cache.table.clone() if kind == "int64" else f(cache.table).contiguous() if kind == "strided" else f(cache.table)
        step = mqk.paged_tables(f(cache.lens), f(numbers(new)), bt, f(free), 50, cursor=f(numbers([1])))
        return [boxes.clone(), pages, mqk.paged_attn(q, cache.k, cache.v, f(cache.table), f(cache.lens), f(cu)),
                mqk.paged_attn(q, cache.k, cache.v, f(cache.table), f(cache.lens), f(cu), pages=f(pages)), bt, *step]
    for got, want in zip(calls(form), calls(lambda t: t)):
        assert torch.equal(got, want)


def test_offsets_out_of_order():
    """Unspecified rows, but nothing beyond what the call may write, and the next call is right."""
    import mqk
    cache = paged_oracle.Cache([300, 90, 17, 1000], 2, 128)
    q = queries(60, 8, 128).cuda()
    boxes = torch.zeros(cache.blocks + 2, 2, 2, 128, dtype=torch.bfloat16, device="cuda")
    good = paged_oracle.offsets([3, 40, 1, 16])
    for cu in ([0, 50, 10, 60, 20], [60, 0, 60, 0, 60], [-5, 100, -100, 2 ** 31 - 1, 60], [40, 30, 20, 10, 0], [0, 0, 0, 0, 99],
               [7, 8, 9, 10, 11]):
        cu = numbers(cu)
        whole = torch.full((62, 8, 128), 7.0, dtype=torch.bfloat16, device="cuda")
        mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens, cu, out=whole[1:61])
        assert (whole[0] == 7).all() and (whole[61] == 7).all()
        mqk.paged_bounds(cache.k, boxes[1:-1], cache.table, cache.lens, 60, cu_seqlens=cu)
        assert (boxes[0] == 0).all() and (boxes[-1] == 0).all()
        pages = mqk.paged_select(q, boxes[1:-1], cache.table, cache.lens, 16, 5, cu)
        assert ((pages >= -1) & (pages < cache.cols)).all()
        mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens, cu, pages=pages)
    got = mqk.paged_attn(q, cache.k, cache.v, cache.table, cache.lens, good)
    attn_oracle.check(got, paged_oracle.attend(cache, q, [3, 40, 1, 16], 128 ** -0.5), torch.bfloat16, "after")


def test_refusals():
    import mqk
    cache = paged_oracle.Cache([30, 90], 2, 64)
    q = queries(2, 4, 64).cuda()
    k, v, table, lens = cache.k, cache.v, cache.table, cache.lens
    boxes = torch.zeros(cache.blocks, 2, 2, 64, dtype=torch.bfloat16, device="cuda")
    attn = lambda **kw: mqk.paged_attn(**{**dict(q=q, k_cache=k, v_cache=v, block_table=table, seq_lens=lens), **kw})
    select = lambda **kw: mqk.paged_select(**{**dict(q=q, bounds=boxes, block_table=table, seq_lens=lens, page=16, n_pages=3), **kw})
    for kw, error, text in (
            (dict(q=q.half()), TypeError, "q must be"), (dict(q=q.cpu()), ValueError, "q must be on"),
            (dict(q=q[..., :32]), ValueError, "head_dim"), (dict(q=q[:, :3]), ValueError, "multiple of H_KV"),
            (dict(q=queries(3, 4, 64).cuda()), ValueError, "cu_seqlens"), (dict(q=q[:1]), ValueError, "cu_seqlens"),
            (dict(v_cache=v[:3]), ValueError, "v_cache"), (dict(v_cache=v.half()), ValueError, "v_cache"),
            (dict(k_cache=k[..., :32], v_cache=v[..., :32]), ValueError, "contiguous"),
            (dict(k_cache=k[:, :12].contiguous(), v_cache=v[:, :12].contiguous()), ValueError, "multiple of 8"),
            (dict(block_table=table[0]), ValueError, "block_table"), (dict(block_table=table.float()), TypeError, "block_table"),
            (dict(block_table=table.cpu()), ValueError, "block_table"), (dict(seq_lens=lens[:1]), ValueError, "seq_lens"),
            (dict(cu_seqlens=lens), ValueError, "cu_seqlens"), (dict(scale=0.0), ValueError, "scale"),
            (dict(scale=float("inf")), ValueError, "scale"), (dict(out=q), ValueError, "overlap"),
            (dict(out=q[:1]), ValueError, "out"), (dict(out=q.float()), TypeError, "out"),
            (dict(pages=table), ValueError, "pages"), (dict(pages=torch.zeros(2, 4, 3, dtype=torch.int32, device="cuda")), ValueError, "pages"),
            (dict(pages=torch.zeros(2, 2, 3, device="cuda")), TypeError, "pages"), (dict(pages=3), TypeError, "pages")):
        with pytest.raises(error, match=text):
            attn(**kw)
    with pytest.raises(ValueError, match="overlap"):
        attn(out=k.view(-1)[:q.numel()].view(q.shape))
    for kw, error, text in (
            (dict(n_pages=1), ValueError, "n_pages"), (dict(recent=0), ValueError, "recent"), (dict(first=-1), ValueError, "first"),
            (dict(page=12), ValueError, "multiple of 8"), (dict(page=0), ValueError, "multiple of 8"),
            (dict(bounds=boxes[:, :, 0]), ValueError, "bounds"), (dict(bounds=boxes.float()), TypeError, "bounds"),
            (dict(q=q.half()), TypeError, "q must be"), (dict(cu_seqlens=lens), ValueError, "cu_seqlens")):
        with pytest.raises(error, match=text):
            select(**kw)
    bounds = lambda **kw: mqk.paged_bounds(**{**dict(k_cache=k, bounds=boxes, block_table=table, seq_lens=lens, n_tokens=2), **kw})
    for kw, error, text in (
            (dict(bounds=boxes.half()), TypeError, "bounds"), (dict(bounds=boxes[1:]), ValueError, "bounds"),
            (dict(n_tokens=3), ValueError, "cu_seqlens"), (dict(n_tokens=-1), ValueError, "n_tokens"),
            (dict(n_tokens=None, cu_seqlens=paged_oracle.offsets([1, 1])), ValueError, "n_tokens")):
        with pytest.raises(error, match=text):
            bounds(**kw)
    lens2 = lens.clone()
    tables = lambda **kw: mqk.paged_tables(**{**dict(seq_lens=lens, new_lens=lens2, block_table=table.clone(), free_pages=lens2,
                                                   n_tokens=9), **kw})
    for kw, error, text in (
            (dict(block_table=table.long()), TypeError, "int32"), (dict(block_table=table[:, ::2]), ValueError, "block_table"),
            (dict(seq_lens=lens[:1]), ValueError, "seq_lens"), (dict(new_lens=lens2.float()), TypeError, "new_lens"),
            (dict(free_pages=table), ValueError, "free_pages"), (dict(cursor=lens), ValueError, "cursor"),
            (dict(n_tokens=-1), ValueError, "n_tokens"), (dict(page=0), ValueError, "page")):
        with pytest.raises(error, match=text):
            tables(**kw)
    with pytest.raises(ValueError, match="overlap"):
        tables(block_table=table, free_pages=table.view(-1)[:2])
    many = torch.zeros(16385, 1, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="overlap"):  # (one column is contiguous: the table itself)
        mqk.paged_tables(many[:, 0].contiguous(), many[:, 0].contiguous(), many, lens2, 1)
    with pytest.raises(mqk.MqkNativeError):
        mqk.paged_tables(many[:, 0].clone(), many[:, 0].clone(), many, lens2, 1)
