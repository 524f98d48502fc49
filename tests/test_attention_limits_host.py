"""Calls of the attention operators' C entry points that cannot be answered, refused before
anything is launched (no GPU needed: no address is read)."""
from __future__ import annotations

import ctypes

import pytest

SHAPE = -2
MB = 1 << 20


@pytest.fixture(scope="module")
def lib():
    from mqk import _native
    if not _native.LIB_PATH.exists():
        pytest.skip("libmqk.so not built")
    return _native.library()


# Where a call's buffers lie: each a MiB from the next, 8 sequences of 32 pages in 64 blocks.
AT = dict(cache=1 * MB, table=2 * MB, scores=3 * MB, lens=4 * MB, new=5 * MB, kept=6 * MB)
N, COLS, BLOCKS, HKV, D, BUDGET = 8, 32, 64, 2, 128, 100
SIZES = dict(cache=BLOCKS * HKV * 18 * D, table=N * COLS * 4, scores=BLOCKS * HKV * 16 * 4, lens=N * 4)


def evict(lib, **at):
    from mqk import _native
    a = dict(AT, **at)
    c = _native.Kv4Cache(a["cache"], a["table"], BLOCKS, COLS, N, 0, HKV, D)
    return lib.mqk_kv4_evict(ctypes.byref(c), a["scores"], a["lens"], BUDGET, 4, a["new"], a["kept"], None)


@pytest.mark.parametrize("read", sorted(SIZES))
@pytest.mark.parametrize("out,size", [("new", N * 4), ("kept", N * HKV * BUDGET * 4)])
def test_evict_writes_over_nothing_it_reads(lib, read, out, size):
    """New lengths in the place of the lengths, and every other overlap: workgroups would read
    what others have written."""
    first, last = AT[read], AT[read] + SIZES[read] - 4
    for at in (first, last, first - size + 4):
        assert evict(lib, **{out: at}) == SHAPE, (read, out, at)
    assert b"overlap" in lib.mqk_last_error_detail()


def test_evict_outputs_apart(lib):
    assert evict(lib, new=AT["kept"] + 8) == SHAPE and evict(lib, new=AT["kept"] - N * 4 + 4) == SHAPE


@pytest.mark.parametrize("scale,decode,prompt", [(1e30, 0, 0), (1.2e37, 0, 0), (1.6e37, SHAPE, 0), (2e38, SHAPE, 0),
                                                 (2.4e38, SHAPE, SHAPE), (2.9e38, SHAPE, SHAPE)])
def test_largest_scales(lib, scale, decode, prompt):
    """The scale is taken times log2(e), by kv4_attn also times the 16 of its operands: one that
    leaves fp32's range is refused.  (With nothing to do the checks are all there is.)"""
    from mqk import _native
    c = _native.Kv4Cache(AT["cache"], AT["table"], BLOCKS, COLS, 0, 0, HKV, D)
    assert lib.mqk_kv4_attn(MB, ctypes.byref(c), AT["lens"], 1, 8, scale, None, MB, None, 0, None) == decode
    t = ctypes.byref(_native.AttnTensor(MB, 1024, 128))
    assert lib.mqk_attn_prefill(t, t, t, 0, None, None, 0, 0, 1, 8, 2, D, scale, 1, MB, None, 0, None) == prompt


def attend(lib, n_seqs, S, Hq, Hkv, cols, scores):
    from mqk import _native
    c = _native.Kv4Cache(MB, MB, BLOCKS, cols, n_seqs, 0, Hkv, D)
    need = lib.mqk_kv4_attn_workspace_size(ctypes.byref(c), S, Hq, int(scores))
    return lib.mqk_kv4_attn(MB, ctypes.byref(c), MB, S, Hq, 0.1, MB if scores else None, MB, MB, need, None)


@pytest.mark.parametrize("n_seqs,S,Hq,Hkv,cols,scores", [
    (1 << 19, 1, 32, 8, 4096, False),      # the join's workgroups
    (1 << 10, 64, 256, 8, 4096, False),
    (1 << 20, 1, 16, 16, 8, False),        # one launch, too many heads
    (1 << 16, 1, 8, 8, 1 << 14, True),     # the weights'
])
def test_more_threads_than_a_launch_has(lib, n_seqs, S, Hq, Hkv, cols, scores):
    """A launch has less than 2^32 threads: a call one of whose launches would have more is
    refused before the first of them has run."""
    assert attend(lib, n_seqs, S, Hq, Hkv, cols, scores) == SHAPE


def test_more_heads_than_a_launch_evicts(lib):
    from mqk import _native
    c = _native.Kv4Cache(1 << 50, 1 << 51, 1, 1, 1 << 20, 0, 4, D)
    assert lib.mqk_kv4_evict(ctypes.byref(c), 1 << 52, 1 << 53, 1, 0, 1 << 54, 1 << 55, None) == SHAPE


def test_prompt_parts_of_too_many_rows(lib):
    """Parts are joined by a second launch with lanes for every row."""
    from mqk import _native
    t = ctypes.byref(_native.AttnTensor(MB, 128, 128))
    T, Hq = 1 << 20, 128
    try:
        assert lib.mqk_set_option(b"attn_parts", 2) == 0
        need = lib.mqk_attn_prefill_workspace_size(0, T, T, 1, 0, Hq, 1, 128)
        assert lib.mqk_attn_prefill(t, t, t, 0, None, None, T, T, 1, Hq, 1, 128, 0.1, 1, MB, MB, need, None) == SHAPE
    finally:
        lib.mqk_set_option(b"attn_parts", 0)
