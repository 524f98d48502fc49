"""The attention operators' checks that need no GPU: what the C entry points refuse before
anything is launched, what the Python ones refuse, and the option knob."""
from __future__ import annotations

import ctypes

import pytest
import torch

import mqk

FAKE = 1 << 20  # 16-byte aligned, never touched: every case ends before a launch
NULL, SHAPE, UNSUPPORTED, MISALIGNED, WORKSPACE, OPTION = -1, -2, -3, -4, -5, -7


@pytest.fixture(scope="module")
def lib():
    from mqk import _native
    if not _native.LIB_PATH.exists():
        pytest.skip("libmqk.so not built")
    return _native.library()


def tensor(data=FAKE, token=1024, head=128):
    from mqk import _native
    return _native.AttnTensor(data, token, head)


def ref(x):
    return None if x is None else ctypes.byref(x)


def cache(**kw):
    from mqk import _native
    a = dict(cache=FAKE, table=FAKE, num_blocks=8, bt_cols=4, n_seqs=2, dtype=0, Hkv=2, D=128)
    a.update(kw)
    return _native.Kv4Cache(*a.values())


def prefill(lib, **kw):
    a = dict(q=tensor(), k=tensor(), v=tensor(), dtype=0, cu_q=FAKE, cu_k=None, T=8, Tk=8, n_seqs=2, Hq=8, Hkv=2, D=128,
             scale=0.1, fill=1, out=FAKE, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    for n in "qkv":
        a[n] = ref(a[n])
    return lib.mqk_attn_prefill(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(q=None), NULL), (dict(out=None), NULL), (dict(k=tensor(None)), NULL), (dict(q=tensor(None)), NULL),
    (dict(dtype=3), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED),
    (dict(D=0), UNSUPPORTED), (dict(D=60), UNSUPPORTED), (dict(D=264), UNSUPPORTED),
    (dict(T=-1), SHAPE), (dict(T=1 << 31, Tk=1 << 31), SHAPE), (dict(Tk=-1, cu_k=FAKE), SHAPE),
    (dict(Hq=0), SHAPE), (dict(Hq=7), SHAPE), (dict(Hkv=0), SHAPE), (dict(Hkv=-2), SHAPE),
    (dict(n_seqs=0), SHAPE), (dict(n_seqs=(1 << 20) + 1), SHAPE),
    (dict(scale=0.0), SHAPE), (dict(scale=float("nan")), SHAPE), (dict(scale=-1.0), SHAPE), (dict(scale=float("inf")), SHAPE),
    (dict(Tk=9), SHAPE), (dict(cu_q=None, n_seqs=3), SHAPE), (dict(cu_q=None, Tk=9), SHAPE),
    (dict(q=tensor(FAKE + 2)), MISALIGNED), (dict(out=FAKE + 8), MISALIGNED), (dict(k=tensor(token=1020)), MISALIGNED),
    (dict(v=tensor(head=4)), MISALIGNED),
    (dict(q=tensor(token=1026), dtype=2), MISALIGNED),
])
def test_prefill_refusals(lib, change, code):
    assert prefill(lib, **change) == code, change


def test_prefill_of_nothing(lib):
    assert prefill(lib, T=0, Tk=0) == 0


def test_prefill_workspace(lib):
    """Few queries over many keys need one, a long prompt none; too small a one is refused."""
    size = lambda T, Tk, dtype=0, D=128: lib.mqk_attn_prefill_workspace_size(dtype, T, Tk, 1, 1, 8, 2, D)
    assert size(8192, 8192) == 0 and size(0, 100) == 0 and size(16, 9000, dtype=5) == 0 and size(16, 9000, D=60) == 0
    need = size(16, 9000)
    assert need > 16 * 8 * 2 * (128 + 2) * 4
    a = dict(T=16, Tk=9000, n_seqs=1, cu_k=FAKE)
    assert prefill(lib, **a) == WORKSPACE and prefill(lib, **a, ws=FAKE, ws_bytes=need - 1) == WORKSPACE
    assert prefill(lib, **a, ws=FAKE + 8, ws_bytes=need) == MISALIGNED
    try:
        assert lib.mqk_set_option(b"attn_parts", 1) == 0 and size(16, 9000) == 0
        assert lib.mqk_set_option(b"attn_parts", 3) == 0
        assert size(100, 100) >= 100 * 8 * 3 * (128 + 2) * 4
        for bad in (-1, 65):
            assert lib.mqk_set_option(b"attn_parts", bad) == OPTION
        assert lib.mqk_get_option(b"attn_parts") == 3
    finally:
        lib.mqk_set_option(b"attn_parts", 0)


def write(lib, c, k=None, v=None, lens=FAKE, cu=FAKE, T=8):
    return lib.mqk_kv4_write(ref(k or tensor()), ref(v or tensor()), ref(c), lens, cu, T, None, None)


def read(lib, c, k=FAKE, v=FAKE, lens=FAKE, cu=FAKE, T=8):
    return lib.mqk_kv4_read(ref(c), lens, cu, T, k, v, None)


def attn(lib, c, q=FAKE, lens=FAKE, S=1, Hq=8, scale=0.1, out=FAKE, ws=None, nbytes=0):
    return lib.mqk_kv4_attn(q, ref(c), lens, S, Hq, scale, None, out, ws, nbytes, None)


def evict(lib, c, scores=FAKE, lens=FAKE, budget=16, recent=4, new=FAKE, kept=FAKE):
    return lib.mqk_kv4_evict(ref(c), scores, lens, budget, recent, new, kept, None)


@pytest.mark.parametrize("call", [write, read, attn, evict])
@pytest.mark.parametrize("change,code", [
    (None, NULL), (dict(cache=None), NULL), (dict(table=None), NULL), (dict(cache=FAKE + 4), MISALIGNED),
    (dict(dtype=2), UNSUPPORTED), (dict(D=96), UNSUPPORTED), (dict(D=256), UNSUPPORTED),
    (dict(Hkv=0), SHAPE), (dict(num_blocks=0), SHAPE), (dict(num_blocks=1 << 31), SHAPE), (dict(bt_cols=0), SHAPE),
    (dict(bt_cols=1 << 27), SHAPE), (dict(n_seqs=-1), SHAPE), (dict(n_seqs=(1 << 20) + 1), SHAPE),
])
def test_cache_refusals(lib, call, change, code):
    assert call(lib, None if change is None else cache(**change)) == code


def test_kv4_refusals(lib):
    c = cache()
    assert lib.mqk_kv4_write(None, ref(tensor()), ref(c), FAKE, FAKE, 8, None, None) == NULL
    assert write(lib, c, k=tensor(None)) == NULL and write(lib, c, lens=None) == NULL
    assert write(lib, c, T=-1) == SHAPE and write(lib, c, cu=None, T=3) == SHAPE
    assert write(lib, c, v=tensor(FAKE + 8)) == MISALIGNED and write(lib, c, k=tensor(head=12)) == MISALIGNED
    assert write(lib, cache(n_seqs=0)) == SHAPE and write(lib, cache(n_seqs=0), T=0) == 0
    assert write(lib, cache(Hkv=4096), T=1 << 30) == SHAPE
    assert read(lib, c, k=None) == NULL and read(lib, c, v=FAKE + 2) == MISALIGNED and read(lib, c, T=0) == 0
    assert read(lib, c, lens=None) == NULL and read(lib, c, T=1 << 31) == SHAPE
    assert attn(lib, c, q=None) == NULL and attn(lib, c, out=None) == NULL and attn(lib, c, lens=None) == NULL
    assert attn(lib, c, S=0) == SHAPE and attn(lib, c, Hq=7) == SHAPE and attn(lib, c, Hq=0) == SHAPE
    assert attn(lib, c, S=1 << 20) == SHAPE and attn(lib, c, scale=0.0) == SHAPE
    assert attn(lib, c, scale=float("inf")) == SHAPE and attn(lib, c, q=FAKE + 2) == MISALIGNED
    assert attn(lib, cache(n_seqs=0)) == 0
    wide = cache(bt_cols=4096)
    need = lib.mqk_kv4_attn_workspace_size(ref(wide), 1, 8, 0)
    assert need > 0 and attn(lib, wide) == WORKSPACE and attn(lib, wide, ws=FAKE, nbytes=need - 1) == WORKSPACE
    assert attn(lib, wide, ws=FAKE + 8, nbytes=need) == MISALIGNED
    assert lib.mqk_kv4_attn_workspace_size(ref(wide), 1, 8, 1) > need
    assert lib.mqk_kv4_attn_workspace_size(ref(cache(D=96)), 1, 8, 0) == 0
    assert evict(lib, c, budget=0) == SHAPE and evict(lib, c, recent=17) == SHAPE and evict(lib, c, recent=-1) == SHAPE
    assert evict(lib, c, scores=None) == NULL and evict(lib, c, kept=None) == NULL and evict(lib, c, new=None) == NULL
    assert evict(lib, cache(n_seqs=0)) == 0


def test_split_option(lib):
    start = lib.mqk_get_option(b"attn_split")
    assert start == 0
    try:
        for good in (1, 2, 4, 0):
            assert lib.mqk_set_option(b"attn_split", good) == 0 and lib.mqk_get_option(b"attn_split") == good
        for bad in (-1, 3, 8):
            assert lib.mqk_set_option(b"attn_split", bad) == OPTION
    finally:
        lib.mqk_set_option(b"attn_split", start)


def test_python_refusals():
    """What is not on a GPU is refused, never worked out some other way."""
    x = torch.zeros(4, 2, 64).bfloat16()
    with pytest.raises(ValueError):
        mqk.attn_prefill(x, x, x)
    for shape in ((4, 2, 96), (0, 2, 64), (4, 0, 64)):
        with pytest.raises(ValueError):
            mqk.kv4_cache(*shape, device="cpu")
    with pytest.raises(TypeError):
        mqk.kv4_cache(4, 2, 64, dtype=torch.float32, device="cpu")
    c = mqk.kv4_cache(4, 2, 64, device="cpu")
    assert c.shape == (4, 2, 576) and c.dtype == torch.bfloat16
    t, n = torch.zeros(1, 2, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    s = torch.zeros(4, 2, 16)
    for call in (lambda: mqk.kv4_write(x[:1], x[:1], c, t, n), lambda: mqk.kv4_read(c, t, n, 1),
                 lambda: mqk.kv4_attn(x[:1], c, t, n), lambda: mqk.kv4_evict(c, s, t, n, 1)):
        with pytest.raises(ValueError, match="GPU"):
            call()
