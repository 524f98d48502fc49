"""Attention over what the projection front returns: whole prompts, and a cache held in 4 bits.

``attn_prefill`` is the attention of the reference's ``paged_attn_prefill``
(mini_qwen/kernels/paged_attn_prefill.py:64-156) on the q / k / v that
:func:`mqk.fused_qkv_rope` (or its varlen form) returns.
"""
from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from . import _native

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
    """A dense int32 tensor of offsets or lengths (int64 is converted)."""
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 (or int64), got {t.dtype}")
    if t.device != device:
        raise ValueError(f"{name} is on {t.device}, expected {device}")
    if numel is not None and (t.dim() != 1 or t.numel() != numel):
        raise ValueError(f"{name} must have {numel} entries, got {tuple(t.shape)}")
    return t.to(torch.int32).contiguous()


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


def _out(out, q: torch.Tensor, shape, dtype, device) -> torch.Tensor:
    if out is None:
        return torch.empty(shape, dtype=dtype, device=device)
    if not isinstance(out, torch.Tensor) or out.dtype != dtype or out.device != device:
        raise TypeError(f"out must be a {dtype} tensor on {device}")
    if tuple(out.shape) != tuple(shape) or not out.is_contiguous() or out.data_ptr() % 16 != 0:
        raise ValueError(f"out must be contiguous, 16-byte aligned and {tuple(shape)}, got {tuple(out.shape)}")
    return out


def _desc(t: torch.Tensor):
    return _native.AttnTensor(t.data_ptr(), t.stride(0), t.stride(1))


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
    seeing the first ``m - n + i + 1`` keys.  A query that sees none gets 0.  In the
    ``[B, S, H, D]`` form k and v may simply have more tokens than q.

    ``scale``: of the scores, default ``D ** -0.5``.  ``out``: where the result goes; rows
    behind the last sequence are left as they are in it (in a new one they are 0).
    Returns a tensor shaped like ``q``.  The result has no gradient.
    """
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
    out = _out(out, q, shape, dtype, device)
    if T == 0:
        return out
    status = _native.call(
        device, _native.library().mqk_attn_prefill, ctypes.byref(_desc(q3)), ctypes.byref(_desc(k3)),
        ctypes.byref(_desc(v3)), _DTYPES[dtype], _native.ptr(cu), _native.ptr(cu_k), T, Tk, n_seqs, H_Q, H_KV, D,
        scale, int(fill), out.data_ptr(), _native.stream_handle(device))
    _native.check(status, "mqk_attn_prefill")
    return out
