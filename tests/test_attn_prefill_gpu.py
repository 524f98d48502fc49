"""mqk.attn_prefill against a plain 64-bit form: types, head layouts, ragged and empty
sequences, strides, masked places that hold what is not finite, and other streams.

The 16-bit kernels round the probabilities to the type, and fp16 ones below 2^-14 of the
maximum to its subnormal step: with m keys that adds at most m 2^-25 max|v| (and 2^8 less
of it relative to the sum, whose largest term is at least 1)."""
import math

import pytest
import torch

import mqk
from attn_oracle import attend, check

pytestmark = pytest.mark.gpu
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(params=[0, 1, 2, 4], autouse=True, ids=lambda n: f"split{n}")
def split(request):
    """Every test on each number of wave groups that share a head's keys."""
    mqk.set_option("attn_split", request.param)
    yield request.param
    mqk.set_option("attn_split", 0)


def make(lens_q, lens_k, Hq, Hkv, D, dtype, seed=0, std=1.5):
    g = torch.Generator().manual_seed(seed)
    r = lambda n, h, s: (torch.randn(n, h, D, generator=g) * s).to(dtype).cuda()
    return r(sum(lens_q), Hq, std), r(sum(lens_k), Hkv, 1.0), r(sum(lens_k), Hkv, 1.0)


def offsets(lens):
    return torch.tensor([0] + lens).cumsum(0).to(torch.int32).cuda()


def verify(out, q, k, v, lens_q, lens_k, dtype, scale=None):
    a = b = 0
    scale = q.shape[2] ** -0.5 if scale is None else scale
    for i, (n, m) in enumerate(zip(lens_q, lens_k)):
        want = attend(q[a:a + n], k[b:b + m], v[b:b + m], scale)
        o, A, slack, p = want
        if dtype == F16:
            # (half a subnormal step a term; check() takes 2^-11 of A)
            A = A + (m * 2.0 ** -25 * v[b:b + m].abs().max().double().item() if m else 0.0) * 2.0 ** 11
        check(out[a:a + n], (o, A, slack), dtype, f"sequence {i} ({n} of {m})")
        a, b = a + n, b + m


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("lens", [[1], [5], [64], [127], [128], [129], [300], [1, 33, 0, 200, 64, 31]])
def test_lengths(dtype, D, lens):
    q, k, v = make(lens, lens, 4, 2, D, dtype)
    out = mqk.attn_prefill(q, k, v, offsets(lens))
    assert out.shape == q.shape and out.dtype == dtype
    verify(out, q, k, v, lens, lens, dtype)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("D", [8, 16, 40, 72, 80, 96, 120, 136, 256])
def test_head_sizes(dtype, D):
    lens = [70, 150]
    q, k, v = make(lens, lens, 6, 2, D, dtype, seed=D)
    verify(mqk.attn_prefill(q, k, v, offsets(lens)), q, k, v, lens, lens, dtype)


@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (3, 1), (8, 8), (16, 8), (40, 8), (32, 4), (64, 4)])
def test_head_layouts(Hq, Hkv):
    lens = [100, 61]
    q, k, v = make(lens, lens, Hq, Hkv, 128, BF16)
    verify(mqk.attn_prefill(q, k, v, offsets(lens)), q, k, v, lens, lens, BF16)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("lens_q,lens_k", [([1], [500]), ([64, 3], [64, 700]), ([130, 1, 20], [1000, 1, 20]),
                                           ([200], [70]), ([5, 9], [0, 9]), ([150, 150], [149, 400])])
def test_other_keys_than_queries(dtype, lens_q, lens_k):
    """Continued prompts, and sequences with fewer keys than queries: the first queries see
    none and get 0."""
    q, k, v = make(lens_q, lens_k, 4, 2, 128, dtype, seed=3)
    out = mqk.attn_prefill(q, k, v, offsets(lens_q), cu_seqlens_k=offsets(lens_k))
    verify(out, q, k, v, lens_q, lens_k, dtype)
    a = 0
    for n, m in zip(lens_q, lens_k):
        assert (out[a:a + max(0, n - m)] == 0).all()
        a += n


def test_long_prompt():
    """Many key tiles: the running maximum moves, the early keys hold large scores."""
    lens = [2500]
    q, k, v = make(lens, lens, 2, 1, 128, BF16, seed=5)
    k[100] *= 6
    verify(mqk.attn_prefill(q, k, v, offsets(lens)), q, k, v, lens, lens, BF16)


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rising_scores(dtype):
    """Scores that rise with the key, by more than 2^8 a tile: every tile rescales."""
    n, D = 400, 64
    q, k, v = make([n], [n], 2, 2, D, dtype, seed=7, std=0.1)
    q[..., 0], k[..., 0] = 8.0, (torch.arange(n, device="cuda")[:, None] * 0.25).to(dtype)
    verify(mqk.attn_prefill(q, k, v, offsets([n])), q, k, v, [n], [n], dtype)


def test_dense_batch_and_strides():
    B, S, Hq, Hkv, D = 3, 77, 8, 2, 128
    g = torch.Generator().manual_seed(1)
    packed = torch.randn(B, S, Hq + 2 * Hkv, D, generator=g).bfloat16().cuda()
    q, k, v = packed.split([Hq, Hkv, Hkv], 2)
    out = mqk.attn_prefill(q, k, v)
    assert out.shape == (B, S, Hq, D) and out.is_contiguous()
    flat = [x.reshape(B * S, -1, D) for x in (q, k, v)]
    verify(out.view(B * S, Hq, D), *flat, [S] * B, [S] * B, BF16)
    # the same call on copies, on heads-first storage, and at an odd offset: the same bits
    assert torch.equal(out, mqk.attn_prefill(*(x.contiguous() for x in (q, k, v))))
    heads = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (q, k, v)]
    assert torch.equal(out, mqk.attn_prefill(*heads))
    odd = torch.empty(q.numel() + 1, dtype=BF16, device="cuda")[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(out, mqk.attn_prefill(odd, k, v))
    wide = torch.zeros(B, S, Hq, 2 * D, dtype=BF16, device="cuda")
    wide[..., ::2] = q
    assert torch.equal(out, mqk.attn_prefill(wide[..., ::2], k, v))
    one = k[:, :, :1].expand(B, S, Hkv, D)  # one stored head for all
    assert torch.equal(mqk.attn_prefill(q, one, v), mqk.attn_prefill(q, one.contiguous(), v))
    # k and v with more tokens than q: the last S of them are q's
    verify(mqk.attn_prefill(q[:, 40:], k, v).reshape(-1, Hq, D), q[:, 40:].reshape(-1, Hq, D), *flat[1:],
           [S - 40] * B, [S] * B, BF16)


def test_rows_behind_the_last_sequence():
    lens = [50, 100]
    q, k, v = make([50, 100, 300], [50, 100, 300], 4, 2, 64, BF16)
    q[150:] = math.nan
    out = mqk.attn_prefill(q, k, v, offsets(lens))
    verify(out[:150], q, k, v, lens, lens, BF16)
    assert (out[150:] == 0).all()
    mine = torch.full_like(q, 7.0)
    assert mqk.attn_prefill(q, k, v, offsets(lens), out=mine) is mine
    assert torch.equal(mine[:150], out[:150]) and (mine[150:] == 7).all()


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_not_finite_where_masked(dtype, bad):
    """A key or value that a query does not see does not reach it, whatever it holds; one
    that it sees does."""
    lens = [200, 90]
    q, k, v = make(lens, lens, 4, 2, 128, dtype, seed=2)
    cu = offsets(lens)
    clean = mqk.attn_prefill(q, k, v, cu)
    for at in (0, 63, 64, 150, 199):
        kk, vv = k.clone(), v.clone()
        vv[at, 1, 5] = bad
        out = mqk.attn_prefill(q, k, vv, cu)
        assert torch.equal(out[:at], clean[:at]) and torch.equal(out[200:], clean[200:])
        assert torch.equal(out[:200, :2], clean[:200, :2])
        seen = out[at:200, 2:, 5].float()
        assert not torch.isfinite(seen).any()
        if not math.isnan(bad):  # (a weight that underflows to 0 gives NaN)
            assert ((seen == bad) | seen.isnan()).all() and (seen == bad).any()
        keep = torch.arange(128) != 5
        assert torch.equal(out[:, :, keep], clean[:, :, keep])
        kk[at, 0, 3] = math.nan
        out = mqk.attn_prefill(q, kk, v, cu)
        assert torch.equal(out[:at], clean[:at]) and torch.equal(out[200:], clean[200:])
        assert out[at:200, :2].isnan().all() and torch.equal(out[:200, 2:], clean[:200, 2:])


def test_lowest_scores():
    """Scores at the type's lowest values (what an additive mask would leave) are scores."""
    n = 80
    q, k, v = make([n], [n], 2, 1, 64, BF16)
    q[:, :, 1:], k[:, :, 1:] = 0, 0
    q[:, :, 0] = 1e18
    k[:, :, 0] = -1e19
    k[7, :, 0] = 1e19
    out = mqk.attn_prefill(q, k, v, offsets([n]))
    want = torch.stack([v[:i + 1].double().mean(0) if i < 7 else v[7].double() for i in range(n)])
    err = (out.double() - want.repeat_interleave(2, 1)).abs()
    assert (err <= 2.0 ** -7 * v.abs().max()).all()


def test_scale():
    lens = [130]
    q, k, v = make(lens, lens, 4, 4, 64, BF16)
    for scale in (1.0, 0.01, 1e-30):
        verify(mqk.attn_prefill(q, k, v, offsets(lens), scale=scale), q, k, v, lens, lens, BF16, scale)


def test_many_sequences():
    """More sequences than one search round of 64 takes, empty ones among them."""
    lens = [(7 * i) % 13 for i in range(150)]
    q, k, v = make(lens, lens, 2, 1, 64, BF16, seed=9)
    verify(mqk.attn_prefill(q, k, v, offsets(lens)), q, k, v, lens, lens, BF16)


def test_offsets_out_of_order():
    """Offsets that do not rise, or leave the tensor, read and write inside it."""
    q, k, v = make([300], [300], 2, 1, 64, BF16)
    guard = torch.full((900, 2, 64), 3.0, dtype=BF16, device="cuda")
    for cu in ([0, 200, 100, 300], [-5, 50, 1 << 30, 7], [300, 200, 100, 0], [0, 0, 0, 0]):
        out = guard[300:600]
        mqk.attn_prefill(q, k, v, torch.tensor(cu, dtype=torch.int32).cuda(), out=out)
        mqk.attn_prefill(q, k, v, offsets([100, 100, 100]), cu_seqlens_k=torch.tensor(cu, dtype=torch.int32).cuda())
    torch.cuda.synchronize()
    assert (guard[:300] == 3).all() and (guard[600:] == 3).all()


def test_other_stream_and_graph():
    lens = [150, 40]
    q, k, v = make(lens, lens, 8, 4, 128, BF16)
    cu = offsets(lens)
    want = mqk.attn_prefill(q, k, v, cu)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = mqk.attn_prefill(q, k, v, cu)
    side.synchronize()
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = mqk.attn_prefill(q, k, v, cu)
    for seed in (11, 12, 13):
        q2, k2, v2 = make(lens, lens, 8, 4, 128, BF16, seed=seed)
        q.copy_(q2), k.copy_(k2), v.copy_(v2)
        cu.copy_(offsets([90, 100]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, mqk.attn_prefill(q2, k2, v2, offsets([90, 100])))


def test_empty():
    e = torch.empty(0, 4, 64, dtype=BF16, device="cuda")
    assert mqk.attn_prefill(e, e, e).shape == (0, 4, 64)
    q = torch.randn(5, 4, 64, device="cuda").bfloat16()
    out = mqk.attn_prefill(q, e, e, offsets([5]), cu_seqlens_k=offsets([0]))
    assert (out == 0).all()


def test_refusals():
    q = torch.zeros(6, 4, 64, dtype=BF16, device="cuda")
    k = torch.zeros(6, 2, 64, dtype=BF16, device="cuda")
    cu = offsets([6])
    cases = [
        (TypeError, lambda: mqk.attn_prefill(q, k.half(), k, cu)),
        (TypeError, lambda: mqk.attn_prefill(q.double(), k.double(), k.double(), cu)),
        (TypeError, lambda: mqk.attn_prefill(q, k, k, cu.float())),
        (ValueError, lambda: mqk.attn_prefill(q, k.cpu(), k, cu)),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu.cpu())),
        (ValueError, lambda: mqk.attn_prefill(q, k[:5], k[:5], cu)),
        (ValueError, lambda: mqk.attn_prefill(q, k, k[:5], cu)),
        (ValueError, lambda: mqk.attn_prefill(q[:, :3], k, k, cu)),
        (ValueError, lambda: mqk.attn_prefill(q[..., :60], k[..., :60], k[..., :60], cu)),
        (ValueError, lambda: mqk.attn_prefill(q, k[..., :32], k[..., :32], cu)),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu, scale=0.0)),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu, scale=-1.0)),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu, scale=math.nan)),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu[:1])),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu_seqlens_k=cu)),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu, cu_seqlens_k=offsets([3, 3]))),
        (ValueError, lambda: mqk.attn_prefill(q, k, k, cu, out=q[:5])),
        (TypeError, lambda: mqk.attn_prefill(q, k, k, cu, out=q.half())),
        (ValueError, lambda: mqk.attn_prefill(q[None], k, k, cu)),
    ]
    for i, (exc, fn) in enumerate(cases):
        with pytest.raises(exc):
            fn()
            pytest.fail(f"case {i} was taken")
