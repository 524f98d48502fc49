"""The operators around the paged cache that the projection front writes.

A cache is two tensors ``[num_blocks, page, H_KV, D]`` (bf16 as the front writes them, or
fp16), addressed by a block table: position p of sequence s is in slot ``p % page`` of block
``block_table[s, p // page]``.  A serving step:

    step = mqk.paged_tables(seq_lens, new_lens, block_table, free_pages, n_tokens)
    q, *_ = mqk.fused_qkv_rope_varlen(..., step.cu_seqlens, seq_pos0=seq_lens, k_cache=k_cache,
                                      v_cache=v_cache, block_table=block_table, kv_seq=step.kv_seq,
                                      kv_pos=step.kv_pos, return_kv=False)
    out = mqk.paged_attn(q, k_cache, v_cache, block_table, step.seq_lens, step.cu_seqlens)

:func:`paged_attn` takes chunks of prompts, single tokens, or both in one call (the
reference's paged_attn_prefill over cached keys and paged_attn_decode).  For contexts that are
too long to be read whole, :func:`paged_bounds` keeps the least and the largest key of every
page, :func:`paged_select` chooses pages for each token by the largest score that these bounds
allow, and ``paged_attn(..., pages=)`` reads only those.
"""
from __future__ import annotations

import ctypes
from typing import NamedTuple, Optional

import torch

from . import _native
from .attention import _DTYPES, _desc, _heads, _int32, _out, _scale, _scratch, _span


class PagedStep(NamedTuple):
    """What :func:`paged_tables` returns (all on the GPU, int32 but for the slots)."""
    seq_lens: torch.Tensor    # [n_seqs] the lengths with the step's tokens
    cu_seqlens: torch.Tensor  # [n_seqs + 1] offsets of the sequences' tokens among the step's
    kv_seq: torch.Tensor      # [n_tokens] each token's sequence,
    kv_pos: torch.Tensor      # its position there,
    slots: torch.Tensor       # and block * page + slot (int64); -1 behind the last sequence
    taken: torch.Tensor       # [1] the cursor behind the pages taken


def paged_tables(
    seq_lens: torch.Tensor,
    new_lens: torch.Tensor,
    block_table: torch.Tensor,
    free_pages: torch.Tensor,
    n_tokens: int,
    *,
    page: int = 16,
    cursor: Optional[torch.Tensor] = None,
) -> PagedStep:
    """A step's block tables and slots, made on the GPU from its requests' lengths.

    Sequence s has ``seq_lens[s]`` tokens in the cache and gets ``new_lens[s]`` more (1 for a
    decode step, a chunk of a prompt, 0 for none).  Pages it needs and does not have are taken
    from ``free_pages`` in the order of the sequences, beginning at ``cursor`` (int32 ``[1]``,
    default 0), and written into ``block_table [n_seqs, cols]`` (int32), in place.  Where the
    list ends the entries are -1, and their tokens' slots: ``taken`` is then past its length
    (nothing here waits for the device, so no error is raised).  Passed as the next step's
    ``cursor``, ``taken`` carries on with the list.

    ``n_tokens``: how many new tokens the call has room for; what does not fit is cut off, and
    the lengths returned are without it.  Rows behind the last token are -1, which the front
    takes for no place in the cache.  n_seqs is at most 16384.
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.paged_tables(seq_lens, new_lens, block_table, free_pages, n_tokens, page, cursor)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_paged_tables")
            return PagedStep(*done)
    if not isinstance(block_table, torch.Tensor):
        raise TypeError("block_table must be a torch.Tensor")
    device = block_table.device
    if not block_table.is_cuda:
        raise ValueError(f"block_table must be on a GPU device, got {device}")
    if block_table.dtype != torch.int32:
        raise TypeError(f"block_table must be int32 (it is written in place), got {block_table.dtype}")
    if block_table.dim() != 2 or block_table.shape[0] < 1 or block_table.shape[1] < 1 or not block_table.is_contiguous():
        raise ValueError(f"block_table must be contiguous and [n_seqs, pages], got {tuple(block_table.shape)}")
    n_seqs, cols = block_table.shape
    old = _int32(seq_lens, "seq_lens", device, n_seqs)
    new = _int32(new_lens, "new_lens", device, n_seqs)
    free = _int32(free_pages, "free_pages", device)
    if free.dim() != 1:
        raise ValueError(f"free_pages must be 1-D, got {tuple(free_pages.shape)}")
    cursor = None if cursor is None else _int32(cursor, "cursor", device, 1)
    n_tokens, page = int(n_tokens), int(page)
    if n_tokens < 0 or page < 1:
        raise ValueError(f"n_tokens {n_tokens} must not be negative, page {page} positive")
    first, end = _span(block_table)
    for t in (old, new, free, cursor):
        if t is not None and _span(t)[0] < end and first < _span(t)[1]:
            raise ValueError("block_table must not overlap what the call reads")

    def ints(n, dtype=torch.int32):
        return torch.empty(n, dtype=dtype, device=device)

    step = PagedStep(ints(n_seqs), ints(n_seqs + 1), ints(n_tokens), ints(n_tokens), ints(n_tokens, torch.int64), ints(1))
    status = _native.call(
        device, _native.library().mqk_paged_tables, old.data_ptr(), new.data_ptr(), n_seqs, block_table.data_ptr(), cols,
        free.data_ptr(), free.numel(), _native.ptr(cursor), page, n_tokens, *(t.data_ptr() for t in step[:5]),
        step.taken.data_ptr(), _native.stream_handle(device))
    _native.check(status, "mqk_paged_tables")
    return step


def _cache(k_cache, v_cache, block_table, seq_lens):
    """Checked descriptor of a paged cache and a call's sequences, and what it points to
    (``v_cache`` None where values are not read)."""
    for t, name in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if t is None and name == "v_cache":
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError(f"{name} must be a torch.Tensor")
        if t.dtype not in (torch.bfloat16, torch.float16):
            raise TypeError(f"{name} must be bf16 or fp16, got {t.dtype}")
        if not t.is_cuda:
            raise ValueError(f"{name} must be on a GPU device, got {t.device}")
        if t.dim() != 4 or min(t.shape) < 1:
            raise ValueError(f"{name} must be [num_blocks, page, H_KV, D], got {tuple(t.shape)}")
        if not t.is_contiguous() or t.data_ptr() % 16 != 0:
            raise ValueError(f"{name} must be contiguous and 16-byte aligned (it is used in place)")
    if v_cache is not None and (v_cache.shape != k_cache.shape or v_cache.dtype != k_cache.dtype
                                or v_cache.device != k_cache.device):
        raise ValueError(f"v_cache must be like k_cache: {tuple(k_cache.shape)} {k_cache.dtype} on {k_cache.device}, "
                         f"got {tuple(v_cache.shape)} {v_cache.dtype} on {v_cache.device}")
    blocks, page, H_KV, D = k_cache.shape
    return _sequences(k_cache.data_ptr(), _native.ptr(v_cache), block_table, seq_lens, k_cache.device, k_cache.dtype, blocks,
                      page, H_KV, D)


def _sequences(k, v, block_table, seq_lens, device, dtype, blocks: int, page: int, H_KV: int, D: int):
    if D % 8 != 0 or D > 256:
        raise ValueError(f"head_dim {D} must be a multiple of 8 up to 256")
    if page < 1 or page % 8 != 0:
        raise ValueError(f"a page of {page} tokens: a multiple of 8")
    table = _int32(block_table, "block_table", device)
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"block_table must be [n_seqs, pages], got {tuple(block_table.shape)}")
    lens = _int32(seq_lens, "seq_lens", device, table.shape[0])
    desc = _native.PagedCache(k, v, table.data_ptr(), blocks, table.shape[1], table.shape[0], _DTYPES[dtype], page, H_KV, D)
    return desc, table, lens


def _queries(q, device, dtype, n_seqs: int, H_KV: int, D: int, cu_seqlens):
    """q as tokens [T, H_Q, D] and the offsets of its sequences."""
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    q3 = _heads(q, "q", device, dtype)
    T, H_Q = q3.shape[:2]
    if q3.shape[2] != D:
        raise ValueError(f"q {tuple(q.shape)} does not match a cache of head_dim {D}")
    if H_Q < 1 or H_Q % H_KV != 0:
        raise ValueError(f"H_Q={H_Q} must be a positive multiple of H_KV={H_KV}")
    if cu_seqlens is not None:
        return q3, _int32(cu_seqlens, "cu_seqlens", device, n_seqs + 1)
    if q.dim() == 4 and q.shape[0] != n_seqs:
        raise ValueError(f"q has {q.shape[0]} sequences, block_table {n_seqs}")
    if T and (n_seqs == 0 or T % n_seqs != 0):
        raise ValueError(f"{T} tokens of {n_seqs} sequences: cu_seqlens is needed")
    return q3, None


def paged_attn(
    q: torch.Tensor,
    k_cache: torch.Tensor,
    v_cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    *,
    pages: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Attention of new tokens over a paged cache, their own keys and values in it already.

    ``q [T, H_Q, D]`` packed with ``cu_seqlens [n_seqs + 1]`` int32 (chunks and single tokens
    in one call), or ``[B, S, H_Q, D]`` / ``[B, H_Q, D]`` with equally many tokens a sequence;
    of the caches' type (bf16, fp16), ``D`` a multiple of 8 up to 256.  ``k_cache`` /
    ``v_cache [num_blocks, page, H_KV, D]`` with pages of a multiple of 8 tokens.

    The n tokens of a sequence are the last of its ``seq_lens[s]``; number i sees the first
    ``seq_lens[s] - n + i + 1`` keys (those that the table has and whose pages lie in the
    cache).  A token that sees none (a padded batch entry with ``seq_lens`` 0), or only
    scores of -infinity, gives 0.  Unused slots of pages may hold anything.  Sequences may
    share pages.

    ``pages`` (int32 ``[..tokens of q.., H_KV, n]``, see :func:`paged_select`): the pages of
    its sequence that a token sees, per key / value head, of its own page the keys up to
    itself.  -1 is none; a page listed twice counts twice.

    ``scale``: of the scores, default ``D ** -0.5``.  ``out``: where the result goes (no part of
    what is read); rows behind the last sequence are left as they are in it (in a new one they
    are 0).  Returns a tensor shaped like ``q``.  The result has no gradient.
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.paged_attn(q, k_cache, v_cache, block_table, seq_lens, cu_seqlens, pages, scale, out)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_paged_attn")
            return done
    if v_cache is None:
        raise TypeError("v_cache must be a torch.Tensor")
    desc, table, lens = _cache(k_cache, v_cache, block_table, seq_lens)
    device, dtype = k_cache.device, k_cache.dtype
    q3, cu = _queries(q, device, dtype, desc.n_seqs, desc.Hkv, desc.D, cu_seqlens)
    T, H_Q, D = q3.shape
    scale = _scale(scale, D)
    n_pages = 0
    if pages is not None:
        if not isinstance(pages, torch.Tensor):
            raise TypeError("pages must be a torch.Tensor")
        if pages.dim() < 2 or tuple(pages.shape[:-1]) != (*q.shape[:-2], desc.Hkv) or pages.shape[-1] < 1:
            raise ValueError(f"pages must be {(*q.shape[:-2], desc.Hkv)} and a number of pages, got {tuple(pages.shape)}")
        pages = _int32(pages, "pages", device)
        n_pages = pages.shape[-1]
    fill = out is None
    out = _out(out, [t for t in (q3, k_cache, v_cache, table, lens, cu, pages) if t is not None], q.shape, dtype, device)
    if q.numel() == 0:
        return out
    lib, stream = _native.library(), _native.stream_handle(device)
    ws = _scratch(device, stream, _native.call(device, lib.mqk_paged_attn_workspace_size, ctypes.byref(desc), T, H_Q,
                                               int(cu is not None), n_pages))
    status = _native.call(
        device, lib.mqk_paged_attn, ctypes.byref(_desc(q3)), ctypes.byref(desc), lens.data_ptr(), _native.ptr(cu), T, H_Q,
        scale, _native.ptr(pages), n_pages, int(fill), out.data_ptr(), _native.ptr(ws), 0 if ws is None else ws.numel(),
        stream)
    _native.check(status, "mqk_paged_attn")
    return out


def _bounds(bounds, like, device, dtype, blocks, H_KV, D) -> torch.Tensor:
    shape = (blocks, H_KV, 2, D)
    if not isinstance(bounds, torch.Tensor):
        raise TypeError("bounds must be a torch.Tensor")
    if bounds.dtype != dtype or bounds.device != device:
        raise TypeError(f"bounds must be {dtype} on {device} as {like} is, got {bounds.dtype} on {bounds.device}")
    if tuple(bounds.shape) != shape or not bounds.is_contiguous() or bounds.data_ptr() % 16 != 0:
        raise ValueError(f"bounds must be contiguous, 16-byte aligned and {shape}, got {tuple(bounds.shape)}")
    return bounds


def paged_bounds(
    k_cache: torch.Tensor,
    bounds: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    n_tokens: Optional[int] = None,
    *,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> None:
    """The least and the largest key of pages, per head and dimension, in place.

    ``bounds [num_blocks, H_KV, 2, D]`` of the cache's type (``k_cache.new_zeros(...)``).  Those
    of the pages that the last ``n_tokens`` tokens stand in are made anew from the cache:
    ``cu_seqlens`` cuts them into sequences (default: equally many each), the ones of sequence s
    being the last of its ``seq_lens[s]``.  Called after every step's keys have been written, it
    keeps the bounds of all pages right; ``n_tokens`` None makes those of whole sequences.
    Slots behind a sequence's end have no part; a NaN among the keys stays one.
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.paged_bounds(k_cache, bounds, block_table, seq_lens, n_tokens, cu_seqlens)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_paged_bounds")
            return
    desc, table, lens = _cache(k_cache, None, block_table, seq_lens)
    device = k_cache.device
    bounds = _bounds(bounds, "k_cache", device, k_cache.dtype, desc.num_blocks, desc.Hkv, desc.D)
    cu = None
    if n_tokens is None:
        if cu_seqlens is not None:
            raise ValueError("cu_seqlens needs n_tokens")
        T = -1
    else:
        T = int(n_tokens)
        if T < 0:
            raise ValueError(f"n_tokens must not be negative, got {T}")
        if cu_seqlens is not None:
            cu = _int32(cu_seqlens, "cu_seqlens", device, desc.n_seqs + 1)
        elif T and (desc.n_seqs == 0 or T % desc.n_seqs != 0):
            raise ValueError(f"{T} tokens of {desc.n_seqs} sequences: cu_seqlens is needed")
    first, end = _span(bounds)
    for t in (k_cache, table, lens, cu):
        if t is not None and _span(t)[0] < end and first < _span(t)[1]:
            raise ValueError("bounds must not overlap what the call reads")
    status = _native.call(device, _native.library().mqk_paged_bounds, ctypes.byref(desc), lens.data_ptr(), _native.ptr(cu), T,
                          bounds.data_ptr(), _native.stream_handle(device))
    _native.check(status, "mqk_paged_bounds")


def paged_select(
    q: torch.Tensor,
    bounds: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    page: int,
    n_pages: int,
    cu_seqlens: Optional[torch.Tensor] = None,
    *,
    first: int = 1,
    recent: int = 1,
) -> torch.Tensor:
    """The pages that each token is to attend to, by the largest score that their bounds allow.

    ``q`` and its sequences as in :func:`paged_attn`, ``bounds [num_blocks, H_KV, 2, D]`` as
    :func:`paged_bounds` keeps them, ``page`` the tokens of a page (a multiple of 8).  Per token
    and key / value head the sequence's ``first`` pages and the ``recent`` last ones up to the
    token's own are taken in any case, and of those between, up to ``n_pages`` in all, the ones
    with the largest

        sum over the head's query heads h and d of max(q[h, d] * least[d], q[h, d] * largest[d])

    which no sum of these heads' scores with a key of the page exceeds (summed in 64 bits; a q
    of 0 adds nothing; equal ones: the first; a NaN counts as the largest).  Pages that are not in the table or
    the cache are not chosen.

    Returns int32 ``[..tokens of q.., H_KV, n_pages]``: the chosen pages' numbers in rising
    order, then -1 (for a token behind the last sequence, or before the first key, throughout).
    The stream's workspace holds scores, 8 bytes a page of the table, head and token, of as many
    tokens at a time as 256 MiB are enough for (4 at least).
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.paged_select(q, bounds, block_table, seq_lens, page, n_pages, cu_seqlens, first, recent)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_paged_select")
            return done
    if not isinstance(bounds, torch.Tensor):
        raise TypeError("bounds must be a torch.Tensor")
    if bounds.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"bounds must be bf16 or fp16, got {bounds.dtype}")
    if not bounds.is_cuda:
        raise ValueError(f"bounds must be on a GPU device, got {bounds.device}")
    if bounds.dim() != 4 or min(bounds.shape) < 1 or bounds.shape[2] != 2:
        raise ValueError(f"bounds must be [num_blocks, H_KV, 2, D], got {tuple(bounds.shape)}")
    blocks, H_KV, _, D = bounds.shape
    device, dtype = bounds.device, bounds.dtype
    _bounds(bounds, "q", device, dtype, blocks, H_KV, D)
    desc, table, lens = _sequences(None, None, block_table, seq_lens, device, dtype, blocks, int(page), H_KV, D)
    q3, cu = _queries(q, device, dtype, desc.n_seqs, H_KV, D, cu_seqlens)
    n_pages, first, recent = int(n_pages), int(first), int(recent)
    if first < 0 or recent < 1 or first + recent > n_pages:
        raise ValueError(f"first {first} and recent {recent} (1 at least) must fit n_pages {n_pages}")
    out = torch.empty((*q.shape[:-2], H_KV, n_pages), dtype=torch.int32, device=device)
    T, H_Q = q3.shape[:2]
    if T == 0:
        return out
    lib, stream = _native.library(), _native.stream_handle(device)
    ws = _scratch(device, stream, lib.mqk_paged_select_workspace_size(ctypes.byref(desc), T))
    status = _native.call(
        device, lib.mqk_paged_select, ctypes.byref(_desc(q3)), bounds.data_ptr(), ctypes.byref(desc), lens.data_ptr(),
        _native.ptr(cu), T, H_Q, n_pages, first, recent, out.data_ptr(), _native.ptr(ws), 0 if ws is None else ws.numel(),
        stream)
    _native.check(status, "mqk_paged_select")
    return out
