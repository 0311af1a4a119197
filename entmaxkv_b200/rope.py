"""RMS norm of every query and key head together with the position rotation.

What lies between a layer's projection and ``PagedKVCache.append`` / ``extend``: the reference leaves it to the model
around it (its decode takes rotated keys, entmaxkv/kv_cache.py:72).
"""

from __future__ import annotations

import ctypes as C
from typing import Optional

import torch

from . import _lib

_INTS = (torch.int32, torch.int64)
_STRIDES = [C.c_int64 * (3 * n) for n in range(5)]


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` itself when its rows are 16-byte aligned and contiguous, else a copy."""
    e = t.element_size()
    s = t.stride()
    if s[3] != 1 or (s[0] | s[1] | s[2]) * e % 16 or t.data_ptr() % 16:
        return t.clone(memory_format=torch.contiguous_format)
    return t


def _strides(*tensors):
    """Batch, head and token strides of the tensors in one ctypes array, and the address of each one's three."""
    array = _STRIDES[len(tensors)](*[x for t in tensors for x in t.stride()[:3]])
    base = C.addressof(array)
    return array, [base + 24 * i for i in range(len(tensors))]


def _destination(out, like, name):
    if out is None:
        return torch.empty_like(like, memory_format=torch.contiguous_format)
    if out.shape != like.shape or out.dtype != like.dtype or out.device != like.device:
        raise ValueError(f"{name} must match its input in shape, dtype and device")
    if out.numel() and (_rows(out) is not out or any(n > 1 and st == 0 for n, st in zip(out.shape, out.stride()))):
        raise ValueError(f"{name} must have contiguous, 16-byte aligned rows of its own")
    return out


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor, inv_freq: torch.Tensor,
                 q_weight: Optional[torch.Tensor] = None, k_weight: Optional[torch.Tensor] = None,
                 eps: Optional[float] = 1e-6, interleaved: bool = False, q_out: Optional[torch.Tensor] = None,
                 k_out: Optional[torch.Tensor] = None):
    """Norm and rotate the queries [B, H_q, T, D] and keys [B, H_kv, T, D] of T tokens per sequence.

    ``y = x * rsqrt(mean(x^2) + eps) * weight`` over each head vector (``eps=None``: no norm, and no weights), then the
    first ``2 * len(inv_freq)`` elements of y are rotated by ``position * inv_freq[j]``: the pairs are (j, j + half), or
    (2j, 2j + 1) with ``interleaved``.  Computed in fp32 (the angle in 64 bits) and rounded once.  q and k may be views
    of a fused projection (any strides).  ``positions``: int32 or int64, [B, T] or [T]; ``inv_freq``: fp32, a multiple
    of 8 entries, at most D / 2; weights: [D], both in the tensors' dtype or both fp32.  ``q_out`` / ``k_out`` may be
    the inputs themselves (in place) and must not overlap them otherwise.  Returns (q_out, k_out).
    """
    index = _lib.require_on_one_device(q, k, positions, inv_freq, q_weight, k_weight)
    q_shape, k_shape = q.shape, k.shape
    if len(q_shape) != 4 or len(k_shape) != 4 or (q_shape[0], q_shape[2], q_shape[3]) != (k_shape[0], k_shape[2], k_shape[3]):
        raise ValueError("q must be [B, H_q, T, D] and k [B, H_kv, T, D]")
    B, Hq, T, D = q_shape
    dtype = q.dtype
    if k.dtype != dtype:
        raise ValueError("q and k must have one dtype")
    code = _lib.dtype_code(dtype)
    p_dtype, p_shape, p_strides = positions.dtype, positions.shape, positions.stride()
    if p_dtype not in _INTS or not (p_shape == (B, T) or p_shape == (T,)):
        raise ValueError(f"positions must be int32 or int64, [{B}, {T}] or [{T}]")
    half = inv_freq.shape[0] if inv_freq.dim() == 1 else -1
    if half < 0 or inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous() or half % 8 or 2 * half > D:
        raise ValueError("inv_freq must be contiguous fp32 with a multiple of 8 entries, at most head_dim / 2")
    weight_f32 = 0
    if q_weight is not None or k_weight is not None:
        if eps is None:
            raise ValueError("weights belong to the norm; eps=None switches it off")
        for w in (q_weight, k_weight):
            if w is not None and (w.shape != (D,) or w.dtype not in (dtype, torch.float32) or not w.is_contiguous()):
                raise ValueError(f"weights must be contiguous [{D}] tensors in the dtype of q or fp32")
        if q_weight is not None and k_weight is not None and q_weight.dtype != k_weight.dtype:
            raise ValueError("q_weight and k_weight must have one dtype")
        weight_f32 = int((k_weight if q_weight is None else q_weight).dtype == torch.float32)
    if eps is not None and not eps >= 0:
        raise ValueError("eps must be >= 0 (or None)")
    with _lib.on_device(index):
        q_out, k_out = _destination(q_out, q, "q_out"), _destination(k_out, k, "k_out")
        q, k = _rows(q), _rows(k)
        array, (qs, ks, qos, kos) = _strides(q, k, q_out, k_out)
        _lib.check(_lib.load().ekv_qk_norm_rope(
            code, B, T, Hq, k_shape[1], D, q.data_ptr(), qs, k.data_ptr(), ks, q_out.data_ptr(), qos,
            k_out.data_ptr(), kos, positions.data_ptr(), int(p_dtype == torch.int64),
            p_strides[0] if len(p_strides) == 2 else 0, p_strides[-1], inv_freq.data_ptr(), half,
            int(interleaved), _lib.ptr(q_weight), _lib.ptr(k_weight), weight_f32, int(eps is not None),
            0.0 if eps is None else eps, _lib.stream_ptr()), "ekv_qk_norm_rope")
    return q_out, k_out
