"""Attention over what the projection front returns: whole prompts, and a cache held in 4 bits.

``attn_prefill`` is the attention of the reference's ``paged_attn_prefill``
(mini_qwen/kernels/paged_attn_prefill.py:64-156) on the q / k / v that
:func:`mqk.fused_qkv_rope` (or its varlen form) returns.

The 4-bit cache keeps what the front's bf16 caches keep (pages of 16 tokens addressed by a
block table) in 4.5 bits a value instead of 16: :func:`kv4_cache` makes one,
:func:`kv4_write` fills it, :func:`kv4_attn` decodes over it (paged_attn_decode,
mini_qwen/kernels/paged_attn_decode.py:389-424), :func:`kv4_evict` brings sequences back
to a budget by the attention weight their keys got, :func:`kv4_read` gives the values back
(a prompt that continues attends over them with :func:`attn_prefill`).

A group of 64 dimensions of a token's head is kept as 4-bit codes with a scale and a least
value of the model's type: ``least = min``, ``scale = (max - min) / 15`` (rounded to float32,
then to the type), ``code = round((x - least) / scale)``, ties to even, within 0 .. 15.
The record of one page's head (kv4_device.h has its order) is ``9 * D`` elements of the
model's type; the tensor of records has that type, so that it cannot be taken for another's.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional, Tuple

import torch

from . import _native

_INT32 = torch.iinfo(torch.int32)
_DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def _heads(t, name: str, device, dtype) -> torch.Tensor:
    """``t`` as [tokens, heads, D] that the kernels can read in place (dense heads, token and
    head strides of whole 16-byte chunks); a copy where it is not."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a GPU device, got {t.device}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.dim() not in (3, 4):
        raise ValueError(f"{name} must be [T, H, D] or [B, S, H, D], got {tuple(t.shape)}")
    if t.dim() == 4:
        t = t.reshape(-1, *t.shape[2:])
    step = 16 // t.element_size()
    ok = (t.shape[2] <= 1 or t.stride(2) == 1) and t.stride(1) % step == 0 and t.stride(0) % step == 0 \
        and t.stride(0) >= 0 and t.stride(1) >= 0 and t.data_ptr() % 16 == 0
    return t if ok or t.numel() == 0 else t.clone(memory_format=torch.contiguous_format)


def _int32(t, name: str, device, numel: Optional[int] = None) -> torch.Tensor:
    """A dense int32 tensor of offsets, lengths or pages (int64 is converted: what int32 does
    not hold becomes its largest or smallest number, and so no other place)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 (or int64), got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if numel is not None and (t.dim() != 1 or t.numel() != numel):
        raise ValueError(f"{name} must have {numel} entries, got {tuple(t.shape)}")
    if t.dtype == torch.int64:
        t = t.clamp(_INT32.min, _INT32.max).to(torch.int32)
    return t.contiguous()


def _cu(t, name: str, device) -> torch.Tensor:
    t = _int32(t, name, device)
    if t.dim() != 1 or t.numel() < 2:
        raise ValueError(f"{name} must be a 1-D int32 tensor of n_seqs + 1 >= 2 offsets")
    return t


def _scale(scale, D: int) -> float:
    scale = D ** -0.5 if scale is None else float(scale)
    if not (0.0 < scale <= 1e30) or not math.isfinite(scale):
        raise ValueError(f"scale must be positive and finite, got {scale}")
    return scale


def _span(t: torch.Tensor) -> Tuple[int, int]:
    """The bytes between a tensor's first element and its last one."""
    last = sum((n - 1) * s for n, s in zip(t.shape, t.stride()))
    return t.data_ptr(), t.data_ptr() + (last + 1) * t.element_size() if t.numel() else t.data_ptr()


def _out(out, inputs, shape, dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not isinstance(out, torch.Tensor) or out.dtype != dtype or out.device != device:
        raise TypeError(f"out must be a {dtype} tensor on {device}")
    if tuple(out.shape) != tuple(shape) or not out.is_contiguous() or out.data_ptr() % 16 != 0:
        raise ValueError(f"out must be contiguous, 16-byte aligned and {tuple(shape)}, got {tuple(out.shape)}")
    first, end = _span(out)
    for t in inputs:
        a, b = _span(t)
        if first < b and a < end:
            raise ValueError("out must not overlap what the call reads")
    return out


def _desc(t: torch.Tensor):
    return _native.AttnTensor(t.data_ptr(), t.stride(0), t.stride(1))


def _scratch(device, stream, nbytes):
    """The stream's workspace; for a captured call the graph's own memory, so that replays of
    two graphs share nothing (the calls need no zeros in it)."""
    nbytes = int(nbytes)
    if nbytes and _native.capturing():
        return torch.empty(nbytes, dtype=torch.uint8, device=device)
    return _native.workspace(device, stream, nbytes)


def attn_prefill(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    *,
    cu_seqlens_k: Optional[torch.Tensor] = None,
    scale: Optional[float] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Causal attention over whole prompts with grouped heads.

    ``q [T, H_Q, D]``, ``k``/``v [Tk, H_KV, D]`` packed, with ``cu_seqlens [n_seqs + 1]``
    int32; or ``[B, S, H, D]`` with equal lengths and no ``cu_seqlens``.  bf16, fp16 or
    fp32 (all three alike), ``D`` a multiple of 8 up to 256, ``H_Q`` a multiple of
    ``H_KV``.  Slices of a packed q / k / v tensor are read where they are.

    ``cu_seqlens_k``: the keys' offsets where a sequence has other keys than queries; its
    ``n`` queries are then the last of its ``m`` tokens (a prompt that continues), query i
    seeing the first ``m - n + i + 1`` keys.  A query that sees none, or only scores of
    -infinity, gets 0.  In the
    ``[B, S, H, D]`` form k and v may simply have more tokens than q.

    ``scale``: of the scores, default ``D ** -0.5``.  ``out``: where the result goes (no part
    of q, k or v); rows behind the last sequence are left as they are in it (in a new one
    they are 0).
    Returns a tensor shaped like ``q``.  The result has no gradient.
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.attn_prefill(q, k, v, cu_seqlens, cu_seqlens_k, scale, out)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_attn_prefill")
            return done
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    device, dtype = q.device, q.dtype
    if dtype not in _DTYPES:
        raise TypeError(f"q must be bf16, fp16 or fp32, got {dtype}")
    shape = q.shape
    dims = {t.dim() for t in (q, k, v) if isinstance(t, torch.Tensor)}
    if len(dims) != 1:
        raise ValueError("q, k and v must have the same number of dimensions")
    q3, k3, v3 = _heads(q, "q", device, dtype), _heads(k, "k", device, dtype), _heads(v, "v", device, dtype)
    T, H_Q, D = q3.shape
    Tk, H_KV = k3.shape[:2]
    if k3.shape != v3.shape or k3.shape[2] != D:
        raise ValueError(f"k {tuple(k.shape)} and v {tuple(v.shape)} do not match q {tuple(shape)}")
    if H_KV < 1 or H_Q < 1 or H_Q % H_KV != 0:
        raise ValueError(f"H_Q={H_Q} must be a positive multiple of H_KV={H_KV}")
    if D < 8 or D % 8 != 0 or D > 256:
        raise ValueError(f"head_dim {D} must be a multiple of 8 up to 256")
    scale = _scale(scale, D)
    cu = cu_k = None
    if cu_seqlens is None:
        if cu_seqlens_k is not None:
            raise ValueError("cu_seqlens_k needs cu_seqlens")
        if q.dim() == 4:
            if k.shape[0] != q.shape[0]:
                raise ValueError(f"k has {k.shape[0]} sequences, q has {q.shape[0]}")
            n_seqs = q.shape[0]
        else:
            n_seqs = 1
    else:
        cu = _cu(cu_seqlens, "cu_seqlens", device)
        n_seqs = cu.numel() - 1
        if cu_seqlens_k is not None:
            cu_k = _int32(cu_seqlens_k, "cu_seqlens_k", device, n_seqs + 1)
        elif Tk != T:
            raise ValueError(f"k has {Tk} tokens, q has {T}: cu_seqlens_k is needed")
    fill = out is None
    out = _out(out, (q3, k3, v3), shape, dtype, device)
    if T == 0:
        return out
    lib, stream = _native.library(), _native.stream_handle(device)
    ws = _scratch(device, stream, _native.call(device, lib.mqk_attn_prefill_workspace_size, _DTYPES[dtype], T, Tk, n_seqs,
                                               int(cu is not None), H_Q, H_KV, D))
    status = _native.call(
        device, lib.mqk_attn_prefill, ctypes.byref(_desc(q3)), ctypes.byref(_desc(k3)),
        ctypes.byref(_desc(v3)), _DTYPES[dtype], _native.ptr(cu), _native.ptr(cu_k), T, Tk, n_seqs, H_Q, H_KV, D,
        scale, int(fill), out.data_ptr(), _native.ptr(ws), 0 if ws is None else ws.numel(), stream)
    _native.check(status, "mqk_attn_prefill")
    return out


PAGE = 16  # tokens of a page


def kv4_cache(num_blocks: int, n_kv_heads: int, head_dim: int, *, dtype=torch.bfloat16, device="cuda") -> torch.Tensor:
    """An empty 4-bit cache: ``[num_blocks, n_kv_heads, 9 * head_dim]`` of the model's type
    (bf16 or fp16), ``head_dim`` 64 or 128.  (Zeros; a page need not be cleared to be used.)"""
    if head_dim not in (64, 128):
        raise ValueError(f"head_dim {head_dim}: 64 or 128")
    if dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"a 4-bit cache is of bf16 or fp16, got {dtype}")
    if num_blocks < 1 or n_kv_heads < 1:
        raise ValueError("num_blocks and n_kv_heads must be positive")
    return torch.zeros(num_blocks, n_kv_heads, 9 * head_dim, dtype=dtype, device=device)


def _cache(cache, block_table, seq_lens):
    """Checked descriptor of a 4-bit cache and a call's sequences, and what it points to."""
    if not isinstance(cache, torch.Tensor):
        raise TypeError("cache must be a torch.Tensor (mqk.kv4_cache makes one)")
    if cache.dtype not in (torch.bfloat16, torch.float16):
        raise TypeError(f"cache must be bf16 or fp16, got {cache.dtype}")
    if not cache.is_cuda:
        raise ValueError(f"cache must be on a GPU device, got {cache.device}")
    if cache.dim() != 3 or cache.shape[2] not in (9 * 64, 9 * 128) or cache.shape[0] < 1 or cache.shape[1] < 1:
        raise ValueError(f"cache must be [num_blocks, H_KV, 9 * D] with D 64 or 128, got {tuple(cache.shape)}")
    if not cache.is_contiguous() or cache.data_ptr() % 16 != 0:
        raise ValueError("cache must be contiguous and 16-byte aligned (it is used in place)")
    device = cache.device
    table = _int32(block_table, "block_table", device)
    if table.dim() != 2 or table.shape[1] < 1:
        raise ValueError(f"block_table must be [n_seqs, pages], got {tuple(block_table.shape)}")
    n_seqs = table.shape[0]
    lens = _int32(seq_lens, "seq_lens", device, n_seqs)
    D = cache.shape[2] // 9
    desc = _native.Kv4Cache(cache.data_ptr(), table.data_ptr(), cache.shape[0], table.shape[1], n_seqs,
                            _DTYPES[cache.dtype], cache.shape[1], D)
    return desc, table, lens, D


def _scores(scores, cache, need: bool = False):
    if scores is None:
        if need:
            raise TypeError("scores must be a torch.Tensor")
        return None
    shape = (cache.shape[0], cache.shape[1], PAGE)
    if not isinstance(scores, torch.Tensor) or scores.dtype != torch.float32:
        raise TypeError("scores must be a float32 tensor")
    if scores.device != cache.device or tuple(scores.shape) != shape or not scores.is_contiguous():
        raise ValueError(f"scores must be contiguous, {shape} and on {cache.device}, got {tuple(scores.shape)}")
    return scores


def _offsets(cu_seqlens, device, n_seqs: int, T: int):
    if cu_seqlens is not None:
        return _int32(cu_seqlens, "cu_seqlens", device, n_seqs + 1)
    if T and (n_seqs == 0 or T % n_seqs != 0):
        raise ValueError(f"{T} tokens of {n_seqs} sequences: cu_seqlens is needed")
    return None


def kv4_write(
    k: torch.Tensor,
    v: torch.Tensor,
    cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    cu_seqlens: Optional[torch.Tensor] = None,
    *,
    scores: Optional[torch.Tensor] = None,
) -> None:
    """Writes ``k``/``v [T, H_KV, D]`` (or ``[B, S, H_KV, D]``) into the 4-bit cache, in place.

    The tokens of sequence s are those between ``cu_seqlens[s]`` and ``[s + 1]`` (default:
    equally many each) and become the last ones of its ``seq_lens[s]`` tokens: position p
    goes to slot ``p % 16`` of page ``block_table[s, p // 16]``.  What has no place (a
    position below 0 or past the table, a page outside the cache, a token behind the last
    sequence) is skipped, so a padded batch entry has ``seq_lens`` 0.  A page that a call
    writes to must stand in the tables once only.  ``scores`` (float32 ``[num_blocks, H_KV,
    16]``, see :func:`kv4_attn`): the written tokens' become 0.  Offsets that do not rise from
    0 to T give unspecified contents of the sequences' pages, never an access out of bounds.
    A group of 64 values that holds an infinity or a NaN reads back as NaN.
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.kv4_write(k, v, cache, block_table, seq_lens, cu_seqlens, scores)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_kv4_write")
            return
    desc, table, lens, D = _cache(cache, block_table, seq_lens)
    device = cache.device
    k3, v3 = _heads(k, "k", device, cache.dtype), _heads(v, "v", device, cache.dtype)
    if k3.shape != v3.shape or k3.shape[1:] != (cache.shape[1], D):
        raise ValueError(f"k {tuple(k.shape)} / v {tuple(v.shape)} do not match a cache of {cache.shape[1]} heads of {D}")
    T = k3.shape[0]
    cu = _offsets(cu_seqlens, device, desc.n_seqs, T)
    scores = _scores(scores, cache)
    if T == 0:
        return
    status = _native.call(device, _native.library().mqk_kv4_write, ctypes.byref(_desc(k3)), ctypes.byref(_desc(v3)),
                          ctypes.byref(desc), lens.data_ptr(), _native.ptr(cu), T, _native.ptr(scores),
                          _native.stream_handle(device))
    _native.check(status, "mqk_kv4_write")


def kv4_read(
    cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    n_tokens: int,
    cu_seqlens: Optional[torch.Tensor] = None,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """The values of ``n_tokens`` tokens that the cache holds, ``(k, v)`` of ``[n_tokens, H_KV, D]``.

    The tokens are addressed as :func:`kv4_write` addresses them: those of sequence s (cut
    by ``cu_seqlens``, default equally many each) are the last of its ``seq_lens[s]``.  For
    whole sequences ``cu_seqlens`` holds the running sum of ``seq_lens``, and its last entry
    is ``n_tokens``.  Tokens that are not there, and those behind the last sequence, give 0;
    offsets that do not rise from 0 give unspecified values.
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.kv4_read(cache, block_table, seq_lens, n_tokens, cu_seqlens)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_kv4_read")
            return done
    desc, table, lens, D = _cache(cache, block_table, seq_lens)
    device = cache.device
    T = int(n_tokens)
    if T < 0:
        raise ValueError(f"n_tokens must not be negative, got {T}")
    cu = _offsets(cu_seqlens, device, desc.n_seqs, T)
    k = torch.empty(T, cache.shape[1], D, dtype=cache.dtype, device=device)
    v = torch.empty_like(k)
    if T == 0:
        return k, v
    status = _native.call(device, _native.library().mqk_kv4_read, ctypes.byref(desc), lens.data_ptr(), _native.ptr(cu),
                          T, k.data_ptr(), v.data_ptr(), _native.stream_handle(device))
    _native.check(status, "mqk_kv4_read")
    return k, v


def kv4_attn(
    q: torch.Tensor,
    cache: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    *,
    scale: Optional[float] = None,
    scores: Optional[torch.Tensor] = None,
    out: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Decode attention over the 4-bit cache.

    ``q [B, S, H_Q, D]`` (or ``[B, H_Q, D]``: one token each), of the cache's type: the last
    S tokens of their sequences, whose keys and values have been written.  Token s of a
    sequence sees its first ``seq_lens - S + s + 1`` keys (of a length past the table those
    that the table has); one that sees none (a padded batch entry with ``seq_lens`` 0) gives
    0.  Unused slots of pages may hold anything.

    ``scores`` (float32 ``[num_blocks, H_KV, 16]``, one entry a key of a head): every key's
    softmax weight, summed over the S tokens and the query heads that share its head, is
    added to its entry, for :func:`kv4_evict`.  A page must then stand in the tables once
    only (otherwise sequences may share pages).  ``scale``: of the scores, default ``D ** -0.5``.  ``out``: where the
    result goes (no part of what is read).  Returns a tensor shaped like ``q``.
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.kv4_attn(q, cache, block_table, seq_lens, scale, scores, out)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_kv4_attn")
            return done
    desc, table, lens, D = _cache(cache, block_table, seq_lens)
    device, dtype = cache.device, cache.dtype
    if not isinstance(q, torch.Tensor):
        raise TypeError("q must be a torch.Tensor")
    if q.device != device:
        raise ValueError(f"q is on {q.device}, expected {device}")
    if q.dtype != dtype:
        raise TypeError(f"q must be {dtype} as the cache is, got {q.dtype}")
    if q.dim() not in (3, 4):
        raise ValueError(f"q must be [B, S, H_Q, D] or [B, H_Q, D], got {tuple(q.shape)}")
    B, H_Q = q.shape[0], q.shape[-2]
    S = q.shape[1] if q.dim() == 4 else 1
    if B != desc.n_seqs or q.shape[-1] != D:
        raise ValueError(f"q {tuple(q.shape)} does not match {desc.n_seqs} sequences of head_dim {D}")
    if H_Q < 1 or H_Q % desc.Hkv != 0:
        raise ValueError(f"H_Q={H_Q} must be a positive multiple of H_KV={desc.Hkv}")
    scale = _scale(scale, D)
    scores = _scores(scores, cache)
    shape = q.shape
    if not q.is_contiguous() or q.data_ptr() % 16 != 0:
        q = q.clone(memory_format=torch.contiguous_format)
    out = _out(out, (q, cache) if scores is None else (q, cache, scores), shape, dtype, device)
    if q.numel() == 0:
        return out
    lib = _native.library()
    stream = _native.stream_handle(device)
    ws = _scratch(device, stream, _native.call(device, lib.mqk_kv4_attn_workspace_size, ctypes.byref(desc), S, H_Q,
                                               int(scores is not None)))
    status = _native.call(device, lib.mqk_kv4_attn, q.data_ptr(), ctypes.byref(desc), lens.data_ptr(), S, H_Q, scale,
                          _native.ptr(scores), out.data_ptr(), _native.ptr(ws), 0 if ws is None else ws.numel(), stream)
    _native.check(status, "mqk_kv4_attn")
    return out


def kv4_evict(
    cache: torch.Tensor,
    scores: torch.Tensor,
    block_table: torch.Tensor,
    seq_lens: torch.Tensor,
    budget: int,
    *,
    recent: int = 0,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Brings sequences longer than ``budget`` tokens back to it, by their keys' accumulated
    attention weights (``scores``, see :func:`kv4_attn`), in place.

    Per key / value head the last ``recent`` tokens stay, and of the others the ``budget -
    recent`` with the largest scores (equal ones: the first; a NaN counts as the largest).
    They move to the first positions in their order, scores with them; what lies behind
    stays as it was.  Keys keep the rotation of the positions they had, and new tokens go to
    the cache position after the kept ones, while their rotation goes on from the sequence's
    own length.  A page must stand in the tables once only.  Tokens that are not there (past
    the table, or in pages outside the cache) are not kept, the recent ones among them, so a
    sequence may have fewer than ``budget`` then; and the places that kept tokens move to
    need pages: a token whose new place has none is lost (``kept`` still names it).

    Returns ``(new_lens [B] int32, kept [B, H_KV, budget] int32)``: the lengths now, and the
    positions that the kept tokens had (-1 past the length).
    """
    front = _native._front or _native.front()
    if front is not None:  # (an ordinary call in C++; None: one for the code below)
        done = front.kv4_evict(cache, scores, block_table, seq_lens, budget, recent)
        if done is not None:
            if type(done) is int:
                _native.check(done, "mqk_kv4_evict")
            return done
    desc, table, lens, D = _cache(cache, block_table, seq_lens)
    device = cache.device
    scores = _scores(scores, cache, need=True)
    budget, recent = int(budget), int(recent)
    if budget < 1 or budget > 1 << 24 or recent < 0 or recent > budget:
        raise ValueError(f"budget {budget} must be positive and recent {recent} within it")
    new_lens = torch.empty(desc.n_seqs, dtype=torch.int32, device=device)
    kept = torch.empty(desc.n_seqs, cache.shape[1], budget, dtype=torch.int32, device=device)
    if desc.n_seqs == 0:
        return new_lens, kept
    status = _native.call(device, _native.library().mqk_kv4_evict, ctypes.byref(desc), scores.data_ptr(),
                          lens.data_ptr(), budget, recent, new_lens.data_ptr(), kept.data_ptr(),
                          _native.stream_handle(device))
    _native.check(status, "mqk_kv4_evict")
    return new_lens, kept
