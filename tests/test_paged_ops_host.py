"""The paged operators' checks that need no GPU: what the C entry points refuse before anything
is launched, and what the Python ones refuse."""
from __future__ import annotations

import ctypes

import pytest
import torch

import mqk

FAKE = 1 << 20  # 16-byte aligned, never touched: every case ends before a launch
FAR = 1 << 30   # (another place)
NULL, SHAPE, UNSUPPORTED, MISALIGNED, WORKSPACE = -1, -2, -3, -4, -5
HUGE = 1 << 40

# (a call that is not refused would launch on these addresses)
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="addresses that no GPU may be given")


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
    a = dict(k=FAKE, v=FAKE, table=FAKE, num_blocks=8, bt_cols=4, n_seqs=2, dtype=0, page=16, Hkv=2, D=128)
    a.update(kw)
    return _native.PagedCache(*a.values())


CACHES = [
    (dict(dtype=2), UNSUPPORTED), (dict(dtype=-1), UNSUPPORTED), (dict(D=0), UNSUPPORTED), (dict(D=60), UNSUPPORTED),
    (dict(D=264), UNSUPPORTED), (dict(page=0), UNSUPPORTED), (dict(page=12), UNSUPPORTED), (dict(page=-8), UNSUPPORTED),
    (dict(page=(1 << 20) + 8), UNSUPPORTED), (dict(Hkv=0), SHAPE), (dict(Hkv=4097), SHAPE), (dict(num_blocks=0), SHAPE),
    (dict(num_blocks=1 << 27), SHAPE), (dict(num_blocks=1 << 62), SHAPE), (dict(bt_cols=0), SHAPE),
    (dict(bt_cols=1 << 27), SHAPE), (dict(n_seqs=-1), SHAPE), (dict(n_seqs=(1 << 20) + 1), SHAPE),
]


def attn(lib, **kw):
    a = dict(q=tensor(), cache=cache(), lens=FAKE, cu=None, T=8, Hq=8, scale=0.1, pages=None, n_pages=0, fill=1, out=FAKE,
             ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    a["q"], a["cache"] = ref(a["q"]), ref(a["cache"])
    return lib.mqk_paged_attn(*a.values())


@pytest.mark.parametrize("change,code", [
    *((dict(cache=cache(**c)), code) for c, code in CACHES),
    (dict(q=None), NULL), (dict(cache=None), NULL), (dict(q=tensor(None)), NULL), (dict(cache=cache(k=None)), NULL),
    (dict(cache=cache(v=None)), NULL), (dict(cache=cache(table=None)), NULL), (dict(lens=None), NULL), (dict(out=None), NULL),
    (dict(T=-1), SHAPE), (dict(T=1 << 31), SHAPE), (dict(T=9), SHAPE), (dict(T=9, cache=cache(n_seqs=0)), SHAPE),
    (dict(T=1 << 28, Hq=8), SHAPE), (dict(Hq=0), SHAPE), (dict(Hq=7), SHAPE), (dict(Hq=1 << 17), SHAPE),
    (dict(scale=0.0), SHAPE), (dict(scale=-1.0), SHAPE), (dict(scale=float("nan")), SHAPE), (dict(scale=float("inf")), SHAPE),
    (dict(scale=3e38), SHAPE), (dict(pages=FAKE), SHAPE), (dict(n_pages=3), SHAPE), (dict(n_pages=-1), SHAPE),
    (dict(pages=FAKE, n_pages=1 << 28), SHAPE),
    (dict(q=tensor(FAKE + 2)), MISALIGNED), (dict(q=tensor(token=1020)), MISALIGNED), (dict(q=tensor(head=4)), MISALIGNED),
    (dict(out=FAKE + 8), MISALIGNED), (dict(cache=cache(k=FAKE + 8)), MISALIGNED), (dict(cache=cache(v=FAKE + 2)), MISALIGNED),
    (dict(cache=cache(bt_cols=1000)), WORKSPACE), (dict(ws=FAKE, ws_bytes=100, cache=cache(bt_cols=1000)), WORKSPACE),
    (dict(ws=FAKE + 8, ws_bytes=HUGE, cache=cache(bt_cols=1000)), MISALIGNED),
    (dict(cu=FAKE, T=100), WORKSPACE), (dict(T=100), WORKSPACE),
    (dict(pages=FAKE, n_pages=1 << 18, T=2, cache=cache(bt_cols=1 << 20, n_seqs=1)), WORKSPACE),
])
def test_attn_refusals(lib, change, code):
    assert attn(lib, **change) == code
    assert lib.mqk_last_error_detail()


def test_steps_fit_32_bits(lib):
    c = dict(bt_cols=(1 << 27) - 4096, num_blocks=8, page=16, n_seqs=1)
    assert attn(lib, T=1, Hq=128, cache=cache(Hkv=64, **c)) == WORKSPACE
    assert attn(lib, T=1, Hq=128, cache=cache(Hkv=128, **c)) == SHAPE


def test_no_tokens(lib):
    assert attn(lib, T=0, q=tensor(None), lens=None, out=None) == 0
    assert attn(lib, T=0, cache=cache(n_seqs=0, k=None, v=None, table=None), q=tensor(None)) == 0
    assert lib.mqk_paged_bounds(ref(cache(k=None)), None, None, 0, None, None) == 0
    assert select(lib, T=0, q=tensor(None), bounds=None, lens=None, pages=None) == 0


def test_workspace_sizes(lib):
    size = lambda c, T, Hq, cu, n: lib.mqk_paged_attn_workspace_size(ref(c), T, Hq, cu, n)
    assert size(cache(), 0, 8, 0, 0) == 0 and size(cache(page=12), 2, 8, 0, 0) == 0 and size(None, 2, 8, 0, 0) == 0
    assert size(cache(), 9, 8, 0, 0) == 0 and size(cache(), 9, 8, 1, 0) > 0
    assert size(cache(), 2, 8, 0, 1) == 0  # (a page of each token: no parts)
    assert size(cache(), 2, 8, 0, 512) > 0
    sel = lambda c, T: lib.mqk_paged_select_workspace_size(ref(c), T)
    assert sel(cache(), 0) == 0 and sel(cache(D=4), 1) == 0 and sel(cache(), 3) >= 3 * 2 * 4 * 8


def tables(lib, **kw):
    a = dict(lens=FAKE, new=FAKE + 64, n_seqs=2, table=FAR, cols=4, free=FAKE + 128, n_free=8, cursor=None, page=16, n_tokens=4,
             out_lens=FAR + 256, cu=FAR + 512, seq=FAR + 768, pos=FAR + 1024, slots=FAR + 2048, taken=FAR + 4096, stream=None)
    a.update(kw)
    return lib.mqk_paged_tables(*a.values())


@pytest.mark.parametrize("change,code", [
    (dict(n_seqs=0), SHAPE), (dict(n_seqs=-1), SHAPE), (dict(n_seqs=16385), SHAPE), (dict(cols=0), SHAPE),
    (dict(cols=1 << 31), SHAPE), (dict(page=0), SHAPE), (dict(page=(1 << 20) + 1), SHAPE), (dict(n_free=-1), SHAPE),
    (dict(n_free=1 << 31), SHAPE), (dict(n_tokens=-1), SHAPE), (dict(n_tokens=1 << 31), SHAPE),
    *((dict([(n, None)]), NULL) for n in ("lens", "new", "table", "free", "out_lens", "cu", "seq", "pos", "slots", "taken")),
    (dict(out_lens=FAKE), SHAPE), (dict(cu=FAKE + 64), SHAPE), (dict(taken=FAKE + 128 + 28), SHAPE),
    (dict(table=FAKE + 60), SHAPE), (dict(cursor=FAR + 4096), SHAPE), (dict(pos=FAR + 768 + 12), SHAPE),
    (dict(seq=FAR + 28), SHAPE),
])
def test_tables_refusals(lib, change, code):
    assert tables(lib, **change) == code
    assert lib.mqk_last_error_detail()


@pytest.mark.parametrize("change,code", [
    *((dict(cache=cache(**c)), code) for c, code in CACHES),
    (dict(cache=None), NULL), (dict(cache=cache(k=None)), NULL), (dict(cache=cache(table=None)), NULL), (dict(lens=None), NULL),
    (dict(bounds=None), NULL), (dict(T=-2), SHAPE), (dict(T=3), SHAPE), (dict(T=-1, cu=FAKE), SHAPE),
    (dict(T=4, cache=cache(n_seqs=0)), SHAPE), (dict(cache=cache(k=FAKE + 8)), MISALIGNED), (dict(bounds=FAKE + 4), MISALIGNED),
    (dict(T=-1, cache=cache(n_seqs=1 << 20, bt_cols=1 << 20)), SHAPE),
])
def test_bounds_refusals(lib, change, code):
    a = dict(cache=cache(), lens=FAKE, cu=None, T=2, bounds=FAKE, stream=None)
    a.update(change)
    a["cache"] = ref(a["cache"])
    assert lib.mqk_paged_bounds(*a.values()) == code
    assert lib.mqk_last_error_detail()


def select(lib, **kw):
    a = dict(q=tensor(), bounds=FAKE, cache=cache(k=None, v=None), lens=FAKE, cu=None, T=2, Hq=8, n_pages=4, first=1, recent=1,
             pages=FAKE, ws=None, ws_bytes=0, stream=None)
    a.update(kw)
    a["q"], a["cache"] = ref(a["q"]), ref(a["cache"])
    return lib.mqk_paged_select(*a.values())


@pytest.mark.parametrize("change,code", [
    *((dict(cache=cache(**c)), code) for c, code in CACHES),
    (dict(q=None), NULL), (dict(q=tensor(None)), NULL), (dict(cache=None), NULL), (dict(cache=cache(table=None)), NULL),
    (dict(lens=None), NULL), (dict(bounds=None), NULL), (dict(pages=None), NULL),
    (dict(T=-1), SHAPE), (dict(T=3), SHAPE), (dict(Hq=7), SHAPE), (dict(n_pages=0), SHAPE), (dict(n_pages=1 << 25), SHAPE),
    (dict(first=-1), SHAPE), (dict(recent=0), SHAPE), (dict(first=4), SHAPE), (dict(first=2, recent=3), SHAPE),
    (dict(first=2 ** 31 - 1, recent=2 ** 31 - 1), SHAPE), (dict(T=1 << 24), SHAPE),
    (dict(q=tensor(FAKE + 8)), MISALIGNED), (dict(q=tensor(head=60)), MISALIGNED), (dict(bounds=FAKE + 8), MISALIGNED),
    (dict(), WORKSPACE), (dict(ws=FAKE, ws_bytes=64), WORKSPACE), (dict(ws=FAKE + 8, ws_bytes=HUGE), MISALIGNED),
])
def test_select_refusals(lib, change, code):
    assert select(lib, **change) == code
    assert lib.mqk_last_error_detail()


def test_python_refusals():
    """Host tensors, wrong types and shapes."""
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)
    q = torch.zeros(2, 4, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        mqk.paged_attn(q, k, k, table, lens)
    with pytest.raises(TypeError, match="v_cache"):
        mqk.paged_attn(q, k, None, table, lens)
    with pytest.raises(TypeError, match="k_cache"):
        mqk.paged_attn(q, None, k, table, lens)
    with pytest.raises(TypeError, match="bf16 or fp16"):
        mqk.paged_attn(q, k.float(), k.float(), table, lens)
    with pytest.raises(ValueError, match="GPU"):
        mqk.paged_bounds(k, k, table, lens)
    with pytest.raises(ValueError, match="GPU"):
        mqk.paged_select(q, k, table, lens, 16, 4)
    with pytest.raises(TypeError, match="bounds"):
        mqk.paged_select(q, None, table, lens, 16, 4)
    with pytest.raises(ValueError, match="GPU"):
        mqk.paged_tables(lens, lens, table, lens, 2)
    with pytest.raises(TypeError, match="block_table"):
        mqk.paged_tables(lens, lens, None, lens, 2)
