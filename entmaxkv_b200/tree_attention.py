"""Entmax attention of a tree of drafted tokens over the cache (speculative decoding).

The reference decodes one token per sequence and step (entmaxkv/attention_topk.py:8-100); a step that verifies several
drafted tokens at once attends with all of them, each seeing the cache and its own ancestors in the tree.  The drafted
keys and values stay outside the cache; ``PagedKVCache.extend`` writes the accepted ones.
"""

from __future__ import annotations

import ctypes as C
import math
from typing import Optional

import torch

from . import _lib
from .kv_cache import PagedKVCache
from .rope import _rows, _strides

#: drafted tokens per sequence
MAX_TOKENS = 256


def tree_attention_decode(q: torch.Tensor, kv_cache: PagedKVCache, k_draft: torch.Tensor, v_draft: torch.Tensor,
                          tree_mask: torch.Tensor, out: torch.Tensor, draft_lens: Optional[torch.Tensor] = None,
                          alpha: float = 1.5, taus_out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attend with T drafted tokens per sequence to the whole cache and to each token's part of the tree.

    All pages, without ALiBi: a one-token step that selects pages attends to less, and equals this one when its budget
    covers the cache.

    q, out [B, H_q, T, D]; k_draft, v_draft [B, H_kv, T, D] in the cache's dtype (any strides).  ``tree_mask``: bool,
    [T, T] or [B, T, T]: token t sees drafted token j where ``tree_mask[..., t, j]`` (itself included only where it says
    so), and every token of the cache.  ``draft_lens`` (int32 CUDA [B]): trees of different sizes; tokens from there on
    are neither keys nor rows, and their rows of ``out`` and ``taus_out`` stay as they were.

    ``p = ((alpha-1) q.k / sqrt(D) - tau)_+^(1/(alpha-1))`` with the tau that makes each row sum to one, solved until it
    no longer moves; ``out = sum p v``, written in place and returned.  A row that sees nothing gets zeros and
    ``tau = +inf``; a NaN or +inf score makes its row NaN (output and threshold), a score of -inf is as if unseen.
    ``taus_out`` (fp32 [B, H_q, T], contiguous) receives the thresholds.  Works on dense and block-table caches; the cache
    is not changed.  ``out`` must not overlap the inputs.
    A call may be captured into a graph, after ``kv_cache.reserve``: its replays read the buffers of the capture.
    Scratch comes from torch's allocator in each call: about 8 bytes per row and cached token (of the capacity, where the
    call is captured or captured calls add tokens), at most 6 GiB: then groups of rows take turns.  Little of it is touched.
    """
    if kv_cache._k is None:
        raise RuntimeError("kv_cache is not initialised")
    if not 1.0 < alpha < math.inf:
        raise ValueError("alpha must be > 1 and finite")
    index = _lib.require_on_one_device(kv_cache._k, q, k_draft, v_draft, tree_mask, out, draft_lens, taus_out)
    B, Hkv, _, D = kv_cache._k.shape
    dtype, shape = kv_cache._k.dtype, q.shape
    if len(shape) != 4 or shape[0] != B or shape[3] != D or shape[1] == 0 or shape[1] % Hkv:
        raise ValueError(f"q must be [{B}, H_q, T, {D}] with H_q a multiple of {Hkv}")
    Hq, T = shape[1], shape[2]
    if T > MAX_TOKENS:
        raise ValueError(f"at most {MAX_TOKENS} drafted tokens per sequence")
    if k_draft.shape != (B, Hkv, T, D) or v_draft.shape != (B, Hkv, T, D):
        raise ValueError(f"k_draft / v_draft must be [{B}, {Hkv}, {T}, {D}]")
    if q.dtype != dtype or k_draft.dtype != dtype or v_draft.dtype != dtype or out.dtype != dtype:
        raise ValueError("q, k_draft, v_draft and out must have the cache's dtype")
    if out.shape != shape or (not out.is_contiguous() and ((T and out.stride(-1) != 1) or any(
            n > 1 and s == 0 for n, s in zip(shape, out.stride())))):
        raise ValueError("out must match q in shape and be contiguous along head_dim")
    ms = tree_mask.stride()
    if tree_mask.dtype != torch.bool or not (tree_mask.shape == (B, T, T) or tree_mask.shape == (T, T)) or (
            T > 1 and ms[-1] != 1):
        raise ValueError(f"tree_mask must be bool [{T}, {T}] or [{B}, {T}, {T}], contiguous along its last axis")
    if draft_lens is not None and (draft_lens.dtype != torch.int32 or draft_lens.shape != (B,)
                                   or not draft_lens.is_contiguous()):
        raise ValueError(f"draft_lens must be a contiguous int32 [{B}] tensor")
    if taus_out is not None and (taus_out.shape != (B, Hq, T) or taus_out.dtype != torch.float32
                                 or not taus_out.is_contiguous()):
        raise ValueError("taus_out must be a contiguous fp32 [B, H_q, T] tensor")
    if T == 0:
        return out
    if out.data_ptr() in (q.data_ptr(), k_draft.data_ptr(), v_draft.data_ptr()):
        raise ValueError("out must not share memory with the inputs: rows are written while others still read them")
    with _lib.on_device(index):
        lib = _lib.load()
        q, k_draft, v_draft = _rows(q), _rows(k_draft), _rows(v_draft)
        # a captured call is replayed while the sequences grow, and replayed appends grow them unseen by the host: then
        # the call is sized by the capacity
        capturing = torch.cuda.is_current_stream_capturing()
        kv_cache._held_by_graphs |= capturing
        unseen = kv_cache._grows_in_graphs or capturing
        bound = kv_cache.capacity if unseen else min(kv_cache.seq_len, kv_cache.capacity)
        desc = C.byref(kv_cache.desc())
        # scratch of this call alone, from torch's stream-ordered allocator: two streams or two graphs never share it
        ws_bytes = lib.ekv_tree_workspace_bytes(desc, Hq, T, bound)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=q.device)
        array, (qs, ks, vs, os_) = _strides(q, k_draft, v_draft, out)
        _lib.check(lib.ekv_tree_decode(
            desc, q.data_ptr(), qs, Hq, T, k_draft.data_ptr(), ks, v_draft.data_ptr(), vs, tree_mask.data_ptr(),
            ms[0] if len(ms) == 3 else 0, ms[-2], _lib.ptr(draft_lens), bound, float(alpha), out.data_ptr(), os_,
            _lib.ptr(taus_out), ws.data_ptr(), ws_bytes,
            kv_cache._ctl.data_ptr(), _lib.stream_ptr()), "ekv_tree_decode")
    return out
