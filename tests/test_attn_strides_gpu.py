"""Tokens and heads stored in descending order: negative strides at the C entry points (torch
has no such tensors).  The same bits as of the tensors in order."""
import ctypes

import pytest
import torch

import mqk
from mqk import _native

pytestmark = pytest.mark.gpu
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def backwards(t, tokens=True, heads=True):
    """t [T, H, D] in reversed storage, and its descriptor."""
    dims = [d for d, on in enumerate((tokens, heads)) if on]
    x = t.flip(dims).contiguous()
    T, H, D = x.shape
    at = (T - 1) * H * D * tokens + (H - 1) * D * heads
    return x, _native.AttnTensor(x.data_ptr() + at * x.element_size(), -H * D if tokens else H * D, -D if heads else D)


def prefill(descs, like, dtype, T, Tk, Hq, Hkv, D):
    lib = _native.library()
    stream = _native.stream_handle(like.device)
    out = torch.empty_like(like)
    ws = _native.workspace(like.device, stream, int(lib.mqk_attn_prefill_workspace_size(dtype, T, Tk, 1, 0, Hq, Hkv, D)))
    status = lib.mqk_attn_prefill(*(ctypes.byref(d) for d in descs), dtype, None, None, T, Tk, 1, Hq, Hkv, D, D ** -0.5,
                                  1, out.data_ptr(), _native.ptr(ws), 0 if ws is None else ws.numel(), stream)
    _native.check(status, "mqk_attn_prefill")
    return out


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("D", [64, 80, 128, 256])
@pytest.mark.parametrize("n,m", [(300, 300), (70, 700)])
def test_prefill(dtype, D, n, m):
    g = torch.Generator().manual_seed(D)
    Hq, Hkv = 4, 2
    q, k, v = (torch.randn(t, h, D, generator=g).to(dtype).cuda() for t, h in ((n, Hq), (m, Hkv), (m, Hkv)))
    for option, value in (("attn_split", 0), ("attn_split", 1), ("attn_split", 2), ("attn_split", 4), ("attn_parts", 3)):
        mqk.set_option(option, value)
        try:
            want = mqk.attn_prefill(q, k, v)
            for tokens, heads in ((True, True), (True, False), (False, True)):
                held = [backwards(t, tokens, heads) for t in (q, k, v)]
                got = prefill([d for _, d in held], q, DTYPES[dtype], n, m, Hq, Hkv, D)
                assert torch.equal(got, want), (option, value, tokens, heads)
        finally:
            mqk.set_option(option, 0)


@pytest.mark.parametrize("T", [20, 9000])
def test_write(T):
    H, D = 2, 128
    g = torch.Generator().manual_seed(T)
    k, v = (torch.randn(T, H, D, generator=g).bfloat16().cuda() for _ in range(2))
    pages = -(-T // 16)
    table = torch.randperm(pages, generator=g).int().cuda()[None]
    lens = torch.tensor([T], dtype=torch.int32, device="cuda")
    want, got = mqk.kv4_cache(pages, H, D), mqk.kv4_cache(pages, H, D)
    mqk.kv4_write(k, v, want, table, lens)
    held = [backwards(t) for t in (k, v)]
    desc = _native.Kv4Cache(got.data_ptr(), table.data_ptr(), pages, pages, 1, 0, H, D)
    status = _native.library().mqk_kv4_write(*(ctypes.byref(d) for _, d in held), ctypes.byref(desc), lens.data_ptr(), None, T,
                                             None, _native.stream_handle(k.device))
    _native.check(status, "mqk_kv4_write")
    assert torch.equal(got.view(torch.int16), want.view(torch.int16))
