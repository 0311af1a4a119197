"""Paged KV cache with per-page key statistics, resident in HBM and updated in place.

Drop-in for the reference ``PagedKVCache`` (entmaxkv/kv_cache.py:16-255):
same constructor, ``initialize`` / ``append``, and the attributes callers read
(``page_size``, ``k_cache``, ``v_cache``, ``k_min``, ``k_max``, ``k_mean``,
``k_std``, ``last_num_selected_per_head``).

Differences a user can observe:
  * K/V and the statistics live in capacity-sized buffers; ``append`` writes one
    row and refreshes one statistics row per (batch, head) instead of
    concatenating the whole cache (kv_cache.py:81-82).  The public attributes are
    views ``[:, :, :seq_len]`` of those buffers, hence non-contiguous across heads.
  * sequence lengths are kept on the device (``seq_lens``), one per batch row, so a
    batch may be ragged (``initialize(..., seq_lens=...)``) and a decode step needs
    no host synchronisation.
  * ``PagedKVCache(page_size, block_table=True)`` stores K and V as a POOL of physical blocks of
    ``page_size`` rows ([num_blocks, H_kv, page_size, D]) addressed through a per-sequence block
    table, the layout serving engines hand out (the reference cache is dense,
    kv_cache.py:44-56).  Pages of one sequence are then not contiguous in memory; the page
    statistics stay dense.  ``k_cache`` / ``v_cache`` are gathered copies in that mode.
  * with ``num_blocks`` that pool is shared: pages get their blocks when tokens arrive (planned on the GPU from the
    lengths, no host synchronisation) and ``release`` gives them back.
  * ``extend`` writes several tokens per sequence: a prompt chunk, or the accepted path of a tree of drafted tokens.
"""

from __future__ import annotations

import ctypes as C
from typing import Optional, Sequence

import torch

from . import _lib


def _one_more(lens):
    return [n + 1 for n in lens]


class PagedKVCache:
    """KV cache with min/max/mean/std statistics per page of ``page_size`` keys."""

    #: rows of head-room added when a capacity is chosen automatically
    DEFAULT_HEADROOM = 1024

    def __init__(self, page_size: int = 16, capacity: Optional[int] = None, block_table: bool = False,
                 block_order: str = "interleaved", num_blocks: Optional[int] = None):
        if page_size <= 0:
            raise ValueError("page_size must be positive")
        if block_order not in ("interleaved", "random"):
            raise ValueError("block_order must be 'interleaved' or 'random'")
        if num_blocks is not None and (not block_table or num_blocks <= 0):
            raise ValueError("num_blocks must be positive and needs block_table=True")
        self.page_size = int(page_size)
        self._requested_capacity = capacity
        #: K/V live in a pool of physical blocks behind a block table (see the module docstring)
        self.block_mode = bool(block_table)
        self._block_order = block_order
        #: blocks of the shared pool; None: every sequence owns page_capacity blocks from the start
        self.num_blocks = num_blocks
        self._free = None                      # int32 [num_blocks]: the shared pool as a stack (block_tables.py)
        self._table = None                     # int32 [B, page_capacity]: page -> physical block
        self._pool_k = self._pool_v = None     # [num_blocks, H_kv, page_size, D]
        self._k = self._v = None
        self._meta = None                      # [4, B, H, page_capacity, D]: min, max, mean, std
        self.seq_lens: Optional[torch.Tensor] = None     # int32 [B] on the device
        self._host_lens: list[int] = []
        self._longest = (None, 0)              # (a _host_lens, its largest)
        self._lens_exact = True                # False: device lengths may be below the host's
        self._grows_in_graphs = False          # True: tokens are added by captured calls, whose replays the host does not see
        self._held_by_graphs = False           # True: a user's graph replays calls on the present buffers
        self._may_be_empty = False             # True: a sequence may hold no token (released, or rewound to 0)
        self._ctl = None                       # int32: [0]=status, [16:16+B] append tickets
        self.last_num_selected_per_head = None
        self._scratch: dict = {}
        self._desc = None

    # ------------------------------------------------------------------ state

    @property
    def seq_len(self) -> int:
        """Longest sequence of the batch (the reference's ``k_cache.shape[2]``)."""
        if self._longest[0] is not self._host_lens:      # the list is replaced whenever a length changes
            self._longest = (self._host_lens, max(self._host_lens) if self._host_lens else 0)
        return self._longest[1]

    @property
    def host_seq_lens(self) -> list[int]:
        return list(self._host_lens)

    @property
    def is_ragged(self) -> bool:
        return len(set(self._host_lens)) > 1

    @property
    def capacity(self) -> int:
        return 0 if self._k is None else self._k.shape[2]

    @property
    def page_capacity(self) -> int:
        return 0 if self._meta is None else self._meta.shape[3]

    @property
    def num_pages(self) -> int:
        return (self.seq_len + self.page_size - 1) // self.page_size

    def _view_rows(self, t, pool=None):
        if t is None:
            return None
        if self.block_mode:      # gather the sequence's blocks back into [B, H, S, D] (a copy)
            B, H, _, D = t.shape
            n = self.num_pages
            blocks = pool[self._table[:, :n].reshape(-1).long()]                 # [B*n, H, P, D]
            dense = blocks.view(B, n, H, self.page_size, D).permute(0, 2, 1, 3, 4).reshape(B, H, n * self.page_size, D)
            return dense[:, :, :self.seq_len]
        return t.narrow(2, 0, self.seq_len)

    @property
    def k_cache(self):
        return self._view_rows(self._k, self._pool_k)

    @property
    def v_cache(self):
        return self._view_rows(self._v, self._pool_v)

    def _meta_view(self, i):
        return None if self._meta is None else self._meta.select(0, i).narrow(2, 0, self.num_pages)

    @property
    def k_min(self):
        return self._meta_view(0)

    @property
    def k_max(self):
        return self._meta_view(1)

    @property
    def k_mean(self):
        return self._meta_view(2)

    @property
    def k_std(self):
        return self._meta_view(3)

    # ------------------------------------------------------------------ build

    def _allocate(self, B, H, D, capacity, dtype, device):
        P = self.page_size
        capacity = (capacity + P - 1) // P * P
        if self.num_blocks is not None:
            self._allocate_shared(B, H, D, capacity, dtype, device)
            return
        self._k = torch.empty(B, H, capacity, D, dtype=dtype, device=device)
        self._v = torch.empty(B, H, capacity, D, dtype=dtype, device=device)
        self._meta = torch.zeros(4, B, H, capacity // P, D, dtype=dtype, device=device)
        self._desc = None
        if self.block_mode:
            # the same memory seen as a pool of B * page_capacity blocks; _k / _v keep their dense SHAPE
            # (the wrappers read sizes from it) but their rows are only meaningful through the table
            pcap = capacity // P
            self._pool_k = self._k.view(B * pcap, H, P, D)
            self._pool_v = self._v.view(B * pcap, H, P, D)
            old = self._table
            table = torch.empty(B, pcap, dtype=torch.int32, device=device)
            if self._block_order == "interleaved":     # consecutive pages of a sequence lie B blocks apart
                table.copy_((torch.arange(pcap, device=device)[None, :] * B +
                             torch.arange(B, device=device)[:, None]).to(torch.int32))
            else:
                n_old = 0 if old is None else old.numel()
                if old is not None:
                    table[:, :old.shape[1]] = old
                g = torch.Generator(device="cpu").manual_seed(1234 + n_old)
                fresh = (torch.randperm(B * pcap - n_old, generator=g) + n_old).to(torch.int32).to(device)
                pcap_old = 0 if old is None else old.shape[1]
                table[:, pcap_old:] = fresh.view(B, pcap - pcap_old)
            self._table = table

    def _allocate_shared(self, B, H, D, capacity, dtype, device):
        """Shared pool: [num_blocks, H, P, D] behind an empty table; ``capacity`` only bounds a sequence's pages."""
        P, old = self.page_size, self._table
        if old is None:
            self._pool_k = torch.empty(self.num_blocks, H, P, D, dtype=dtype, device=device)
            self._pool_v = torch.empty_like(self._pool_k)
            self._free = torch.arange(self.num_blocks, dtype=torch.int32, device=device)
            if self._block_order == "random":
                g = torch.Generator(device="cpu").manual_seed(1234)
                self._free = torch.randperm(self.num_blocks, generator=g).to(torch.int32).to(device)
        # only the SHAPE of the dense cache (the wrappers read sizes from it); the rows live in the pool
        self._k = self._pool_k.new_empty(1).expand(B, H, capacity, D)
        self._v = self._k
        self._meta = torch.zeros(4, B, H, capacity // P, D, dtype=dtype, device=device)
        self._table = torch.full((B, capacity // P), -1, dtype=torch.int32, device=device)
        if old is not None:
            self._table[:, :old.shape[1]] = old
        self._desc = None

    def initialize(self, k: torch.Tensor, v: torch.Tensor,
                   seq_lens: Optional[Sequence[int]] = None, capacity: Optional[int] = None):
        """Copy prefill keys/values in and build every page's statistics in one launch.

        k, v: [B, H_kv, S, D] (kv_cache.py:40-70).  ``seq_lens`` (optional, length B)
        gives the valid length of each row of a padded, ragged batch.
        """
        _lib.require_cuda(k, v)
        if k.shape != v.shape or k.dim() != 4:
            raise ValueError("k and v must both be [batch, kv_heads, seq_len, head_dim]")
        _lib.dtype_code(k.dtype)
        B, H, S, D = k.shape
        lens = [S] * B if seq_lens is None else [int(x) for x in seq_lens]
        if len(lens) != B or min(lens) < 1 or max(lens) > S:
            raise ValueError("seq_lens must hold one length in [1, S] per batch row")
        cap = capacity or self._requested_capacity or (S + self.DEFAULT_HEADROOM)
        if cap < S:
            raise ValueError("capacity is smaller than the prefill length")
        if self.num_blocks is not None and sum(-(-n // self.page_size) for n in lens) > self.num_blocks:
            raise RuntimeError(f"the prefill does not fit the pool of {self.num_blocks} blocks")
        self._table = None
        self._allocate(B, H, D, cap, k.dtype, k.device)
        if self.num_blocks is not None:
            self._plan(torch.zeros(B, dtype=torch.int32, device=k.device),
                       torch.tensor(lens, dtype=torch.int32, device=k.device))
        if self.block_mode:
            self._scatter_pages(k, v, lens)
        else:
            self._k[:, :, :S].copy_(k)
            self._v[:, :, :S].copy_(v)
        self._host_lens = lens
        self._lens_exact, self._may_be_empty, self._held_by_graphs = True, False, False
        self.seq_lens = torch.tensor(lens, dtype=torch.int32, device=k.device)
        self._ctl = torch.zeros(16 + B, dtype=torch.int32, device=k.device)
        self._scratch = {}
        lib = _lib.load()
        _lib.check(lib.ekv_page_stats_init(C.byref(self.desc()), max(lens), _lib.stream_ptr()),
                   "ekv_page_stats_init")

    def _plan(self, seq_lens, new_lens, status=None):
        """Shared pool: blocks for the pages that ``new_lens`` more tokens need."""
        from .block_tables import plan_block_tables
        plan_block_tables(seq_lens, new_lens, self._table, self._free, self.page_size, status=status)

    def _scatter_pages(self, k, v, lens):
        """Block mode: copy [B, H, S, D] tensors page by page into the blocks the table assigns."""
        B, H, S, D = k.shape
        P = self.page_size
        n = (S + P - 1) // P
        ids = self._table[:, :n].reshape(-1).long()
        held = None
        if self.num_blocks is not None:        # pages behind a short sequence have no block
            held = torch.tensor([p * P < m for m in lens for p in range(n)], device=ids.device)
            ids = ids[held]
        for src, pool in ((k, self._pool_k), (v, self._pool_v)):
            if n * P != S:
                src = torch.cat([src, src.new_zeros(B, H, n * P - S, D)], dim=2)
            pages = src.reshape(B, H, n, P, D).permute(0, 2, 1, 3, 4).reshape(B * n, H, P, D)
            pool[ids] = pages if held is None else pages[held]

    def translate(self, page_indices: torch.Tensor, counts: torch.Tensor, out: Optional[torch.Tensor] = None):
        """Block mode: page numbers -> physical block ids for the first ``counts[b, h]`` entries of every
        row of a page table ([B, H_q, width] int32); the decode kernels address K/V by block id."""
        if out is None:
            out = self.scratch("phys_" + str(page_indices.shape[2]), tuple(page_indices.shape), torch.int32)
        lib = _lib.load()
        _lib.check(lib.ekv_translate_pages(C.byref(self.desc()), page_indices.shape[1], page_indices.data_ptr(),
                                           page_indices.stride(1), counts.data_ptr(), out.data_ptr(),
                                           out.stride(1), _lib.stream_ptr()), "ekv_translate_pages")
        return out

    def reserve(self, capacity: int):
        """Grow the buffers so that ``capacity`` rows fit (copies the cache once).

        Calls captured into a graph keep the addresses of the buffers that they were captured with: after a ``reserve``
        that grows them (or an ``initialize``) such graphs must not be replayed, only captured again.  While graphs of
        ``extend`` or ``tree_attention_decode`` exist, the cache does not grow by itself but raises RuntimeError."""
        if self._k is None:
            self._requested_capacity = capacity
            return
        if capacity <= self.capacity:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the cache cannot grow in a captured call: reserve() room before the capture")
        self._held_by_graphs = False
        B, H, _, D = self._k.shape
        old_k, old_v, old_meta = self._k, self._v, self._meta
        S = self.capacity if self._grows_in_graphs else self.seq_len     # (replays add rows that the host does not count)
        old_pools = (self._pool_k, self._pool_v)
        self._allocate(B, H, D, capacity, old_k.dtype, old_k.device)
        if self.num_blocks is not None:
            pass                               # the pool stays, only the table and the statistics got wider
        elif self.block_mode:
            if self._block_order == "interleaved":
                # block ids p*B + b do not depend on the capacity: the old blocks keep their numbers
                n_old = old_pools[0].shape[0]
                self._pool_k[:n_old].copy_(old_pools[0])
                self._pool_v[:n_old].copy_(old_pools[1])
            else:
                n_old = old_pools[0].shape[0]      # old table entries were kept, new pages got new blocks
                self._pool_k[:n_old].copy_(old_pools[0])
                self._pool_v[:n_old].copy_(old_pools[1])
        else:
            self._k[:, :, :S].copy_(old_k[:, :, :S])
            self._v[:, :, :S].copy_(old_v[:, :, :S])
        self._meta[:, :, :, :old_meta.shape[3]].copy_(old_meta)
        self._scratch = {}

    def append(self, k_new: torch.Tensor, v_new: torch.Tensor):
        """Append one token per sequence (k_new, v_new: [B, H_kv, 1, D]); kv_cache.py:72-116."""
        if self._k is None:
            raise RuntimeError("initialize() the cache before append()")
        _lib.require_cuda(k_new, v_new)
        B, H, _, D = self._k.shape
        if tuple(k_new.shape) != (B, H, 1, D) or tuple(v_new.shape) != (B, H, 1, D):
            raise ValueError(f"k_new / v_new must be [{B}, {H}, 1, {D}]")
        if k_new.dtype != self._k.dtype or v_new.dtype != self._k.dtype:
            raise ValueError("k_new / v_new dtype differs from the cache dtype")
        if k_new.stride(-1) != 1 or v_new.stride(-1) != 1 or k_new.stride() != v_new.stride():
            k_new, v_new = k_new.contiguous(), v_new.contiguous()
        if self.num_blocks is not None:        # a new page needs its block first
            self.extend(k_new, v_new)
            return
        lens = self._room_for(_one_more)
        capturing = torch.cuda.is_current_stream_capturing()
        self._grows_in_graphs |= capturing
        lib = _lib.load()
        _lib.check(lib.ekv_append(C.byref(self.desc()), k_new.data_ptr(), v_new.data_ptr(),
                                  k_new.stride(0), k_new.stride(1),
                                  self._ctl[16:].data_ptr(), self._ctl.data_ptr(), _lib.stream_ptr()),
                   "ekv_append")
        self._host_lens = lens
        self._may_be_empty &= capturing        # a capture appends nothing yet

    def extend(self, k_new: torch.Tensor, v_new: torch.Tensor, counts=None, index: Optional[torch.Tensor] = None,
               start=None, max_seq_len: Optional[int] = None):
        """Append several tokens per sequence and refresh the statistics of every page that they touch.

        k_new, v_new: [B, H_kv, T, D], any strides.  ``counts`` ([B]): how many rows each sequence gets (default T);
        ``index`` (int32 CUDA [B, T]): which row goes where (row ``index[b, i]`` at the i-th new position: the accepted
        path of a tree of drafted tokens; default: row i).  ``start`` ([B]): the first position to write, at most the
        current length: a smaller one rewinds the sequence, whose length becomes ``start + counts``.

        ``counts`` and ``start`` are sequences of ints, or int32 CUDA tensors.  The host does not read the latter, so
        its view of the lengths (``seq_len``, ``host_seq_lens``, the row range of ``k_cache``) becomes an upper bound:
        ``T`` more tokens for every sequence, or ``max_seq_len`` where that is given and smaller (rows past it are then
        the caller's mistake).  ``sync_lengths`` makes it exact again; call it after replays of a captured ``extend``, too,
        which the host does not count.  Scratch and work of later calls are sized by the bound, so a loop does well to
        pass ``max_seq_len`` or to call ``sync_lengths`` now and then.  Where the bound leaves no room in the buffers or in
        the pool, the call reads the lengths itself (one synchronisation) before it grows the cache or gives up.
        Values out of range are clipped on the device and show in ``device_status``.
        ``k_new`` and ``v_new`` must not be views of the cache itself.  A call may be captured into a graph, with ``counts``
        and ``start`` on the device and ``reserve`` called first: its replays write into the buffers of the capture.
        """
        if self._k is None:
            raise RuntimeError("initialize() the cache before extend()")
        dev = _lib.require_on_one_device(self._k, k_new, v_new, index)
        B, H, _, D = self._k.shape
        shape, dtype = k_new.shape, self._k.dtype
        if len(shape) != 4 or v_new.shape != shape or (shape[0], shape[1], shape[3]) != (B, H, D):
            raise ValueError(f"k_new / v_new must be [{B}, {H}, T, {D}]")
        if k_new.dtype != dtype or v_new.dtype != dtype:
            raise ValueError("k_new / v_new dtype differs from the cache dtype")
        device, T = self._k.device, shape[2]
        if max_seq_len is not None and max_seq_len < 0:
            raise ValueError("max_seq_len must be >= 0")
        if index is not None and (index.dtype != torch.int32 or index.shape != (B, T)
                                  or (T > 1 and index.stride(1) != 1)):
            raise ValueError(f"index must be int32 [{B}, {T}], contiguous along the tokens")
        counts_host, counts = self._row_lens(counts, "counts", T)
        start_host, start = self._row_lens(start, "start", None)

        if max_seq_len is not None and self._lens_exact and not self._grows_in_graphs:
            known = self._host_lens if start is None else [0] * B if start_host is None else start_host
            known = known if counts_host is None else [n + m for n, m in zip(known, counts_host)]
            if max(known) > max_seq_len:
                raise ValueError(f"a sequence will hold {max(known)} tokens, more than max_seq_len = {max_seq_len}")

        def after(lens):
            lens = lens if start_host is None else [min(s, n) for s, n in zip(start_host, lens)]
            lens = [n + T for n in lens] if counts_host is None else [n + m for n, m in zip(lens, counts_host)]
            if max_seq_len is not None and max(lens) > max_seq_len:
                lens = [n if n < max_seq_len else max_seq_len for n in lens]
            return lens

        rewound_on_device = start is not None and start_host is None
        if T == 0:
            if start is None:
                return
            k_new = v_new = k_new.new_zeros(B, H, 1, D)      # a rewind alone: no row is taken
            counts, counts_host, T, index = torch.zeros(B, dtype=torch.int32, device=device), [0] * B, 1, None
        e = k_new.element_size()
        s = k_new.stride()
        if s != v_new.stride() or s[3] != 1 or (s[0] | s[1] | s[2]) * e % 16 or (k_new.data_ptr() | v_new.data_ptr()) % 16:
            k_new, v_new = (t.clone(memory_format=torch.contiguous_format) for t in (k_new, v_new))
            s = k_new.stride()
        with _lib.on_device(dev):
            bound = self._room_for(after)
            capturing = torch.cuda.is_current_stream_capturing()
            self._grows_in_graphs |= capturing
            self._held_by_graphs |= capturing
            if self.num_blocks is not None:
                held = self.seq_lens
                if start is not None:          # what lies behind the rewind goes back first
                    from .block_tables import return_blocks
                    return_blocks(held, start, self._table, self._free, self.page_size, status=self._ctl)
                    held = torch.minimum(held, start.clamp(min=0))
                # (only what will be written is planned for: the pool's top follows from the lengths)
                more = T if counts is None else counts if counts_host is not None else counts.clamp(max=T)
                self._plan(held, more, status=self._ctl)
            _lib.check(_lib.load().ekv_extend(
                C.byref(self.desc()), k_new.data_ptr(), v_new.data_ptr(), s[0], s[1], s[2], T, _lib.ptr(counts),
                _lib.ptr(index), index.stride(0) if index is not None and B > 1 else T, _lib.ptr(start),
                self._ctl.data_ptr() + 64, self._ctl.data_ptr(), _lib.stream_ptr()), "ekv_extend")
        if counts_host is None or rewound_on_device:
            self._lens_exact = False
        if counts_host is not None and min(counts_host) > 0:
            self._may_be_empty &= capturing    # a capture writes nothing yet
        elif rewound_on_device or (start_host is not None and 0 in start_host):
            self._may_be_empty = True
        self._host_lens = bound

    def _room_for(self, after):
        """Room for the tokens of a call: ``after`` gives its lengths from those before it.  Returns them, with
        ``_host_lens`` brought up to date where it only bounded the lengths and the bound, not the tokens, leaves no room."""
        lens = after(self._host_lens)
        if max(lens) > self.capacity or not self._pool_suffices(lens):
            if (self._grows_in_graphs or not self._lens_exact) and not torch.cuda.is_current_stream_capturing():
                self.sync_lengths()
                lens = after(self._host_lens)
            self._make_room(lens)
        return lens

    def _pool_suffices(self, lens):
        return self.num_blocks is None or sum(-(-n // self.page_size) for n in lens) <= self.num_blocks

    def _make_room(self, lens):
        """Before tokens are added: room for sequences of ``lens`` tokens (upper bounds), and blocks in a shared pool."""
        if not self._pool_suffices(lens):
            raise RuntimeError(f"the pool of {self.num_blocks} blocks may not suffice: release() sequences" + (
                "" if self._lens_exact else ", or call sync_lengths() (the host knows only upper bounds of the lengths)"))
        most = max(lens)
        if most > self.capacity:
            if self._held_by_graphs:
                raise RuntimeError(f"no room for {most} tokens: captured calls hold the cache's buffers, which therefore do not "
                                   "grow by themselves; reserve() more and capture again")
            self.reserve(max(most, self.capacity + 4096, self.capacity * 5 // 4))

    def _row_lens(self, value, name, most):
        """One length per sequence, given on the host or on the device: (host list or None, int32 CUDA tensor or None)."""
        B, device = self._k.shape[0], self._k.device
        if value is None:
            return ([most] * B if most is not None else None), None
        if isinstance(value, torch.Tensor):
            _lib.require_on_one_device(self._k, value)
            if value.dtype != torch.int32 or value.shape != (B,) or not value.is_contiguous():
                raise ValueError(f"{name} must be a contiguous int32 [{B}] tensor")
            return None, value
        if torch.cuda.is_current_stream_capturing():
            raise ValueError(f"{name} must be an int32 CUDA tensor in a captured call (a list is copied at each call)")
        host = [int(x) for x in value]
        if len(host) != B or min(host) < 0 or (most is not None and max(host) > most):
            raise ValueError(f"{name} must hold one length per sequence" + (f", at most {most}" if most is not None else ""))
        beyond = lambda: any(s > n for s, n in zip(host, self._host_lens))  # noqa: E731
        if most is None and beyond():
            if self._grows_in_graphs:              # replays may have added what the host does not know of
                self.sync_lengths()
            if self._lens_exact and beyond():
                raise ValueError(f"{name} lies beyond the sequence's length")
        return host, torch.tensor(host, dtype=torch.int32, device=device)

    def sync_lengths(self) -> list[int]:
        """Read the sequence lengths back from the device (synchronises): after ``extend`` with lengths on the device the
        host's view is an upper bound."""
        self._host_lens = self.seq_lens.tolist()
        self._lens_exact, self._may_be_empty = True, min(self._host_lens) < 1
        return list(self._host_lens)

    def release(self, rows: Sequence[int]):
        """Empty the sequences ``rows``; with a shared pool their blocks go back to it.  A released sequence takes new
        tokens through ``extend`` and can be attended to once it has some."""
        if self._k is None:
            raise RuntimeError("initialize() the cache before release()")
        B = self._k.shape[0]
        rows = sorted({int(r) for r in rows})
        if rows and not 0 <= rows[0] <= rows[-1] < B:
            raise ValueError(f"rows must lie in [0, {B})")
        if not rows:
            return
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("release() belongs between captured calls, not into them")
        keep = self.seq_lens.clone()
        keep[torch.tensor(rows, device=keep.device)] = 0
        if self.num_blocks is not None:
            from .block_tables import release_block_tables
            release_block_tables(self.seq_lens, keep, self._table, self._free, self.page_size, status=self._ctl)
        else:
            self.seq_lens.copy_(keep)
        self._host_lens = [0 if i in rows else n for i, n in enumerate(self._host_lens)]
        self._may_be_empty = True

    def require_tokens(self):
        """What attends to a cache, or selects pages of it, is defined for sequences of at least one token."""
        if self._may_be_empty:
            raise ValueError("a sequence may hold no token: give it some, or call kv_cache.sync_lengths()")

    # ------------------------------------------------------------------ C ABI view

    def desc(self) -> _lib.CacheDesc:
        """The plain-C description of this cache that every entry point takes."""
        if self._desc is None:
            k, m = self._k, self._meta
            d = _lib.CacheDesc()
            kp, vp = (k, self._v) if self.num_blocks is None else (self._pool_k, self._pool_v)
            d.k, d.v = kp.data_ptr(), vp.data_ptr()
            d.k_min, d.k_max, d.k_mean, d.k_std = (m[i].data_ptr() for i in range(4))
            d.kv_stride_b, d.kv_stride_h = k.stride(0), k.stride(1)
            d.meta_stride_b, d.meta_stride_h = m.stride(1), m.stride(2)
            d.batch, d.kv_heads, d.head_dim = k.shape[0], k.shape[1], k.shape[3]
            d.page_size, d.capacity, d.page_capacity = self.page_size, k.shape[2], m.shape[3]
            d.dtype = _lib.dtype_code(k.dtype)
            if self.block_mode:
                P, H, D = self.page_size, k.shape[1], k.shape[3]
                d.kv_stride_b, d.kv_stride_h = 0, P * D
                d.block_table, d.bt_stride = self._table.data_ptr(), self._table.stride(0)
                d.kv_stride_block, d.num_blocks = H * P * D, self._pool_k.shape[0]
            self._desc = d
        self._desc.seq_lens = self.seq_lens.data_ptr()
        return self._desc

    def scratch(self, name: str, shape, dtype, zero: bool = False) -> torch.Tensor:
        """Persistent per-cache scratch tensor, reallocated only when its shape changes."""
        key = (name, tuple(shape), dtype)
        t = self._scratch.get(key)
        if t is None:
            for old in [k for k in self._scratch if k[0] == name]:
                del self._scratch[old]
            make = torch.zeros if zero else torch.empty
            t = make(tuple(shape), dtype=dtype, device=self._k.device)
            self._scratch[key] = t
        return t

    def device_status(self) -> int:
        """Status bits raised by device-side range checks of cache updates, plus ``COPY_TIMEOUT`` (16) when
        any bulk copy of this process timed out in one of the library's kernels (synchronises)."""
        bits = int(self._ctl[0].item())
        n = C.c_uint32(0)
        _lib.check(_lib.load().ekv_copy_timeouts(C.byref(n)), "ekv_copy_timeouts")
        return bits | (16 if n.value else 0)

    # ------------------------------------------------------------------ scoring helper

    def estimate_page_criticality(self, q: torch.Tensor, use_triton: bool = True,
                                  alibi_slopes=None, q_pos: int = 0,
                                  exclude_last_page: bool = False) -> torch.Tensor:
        """Key-range upper-bound score of every page, [B, H_q, pages] in q.dtype.

        kv_cache.py:118-165.  Only the decode-step form (last page excluded) exists
        as a kernel.  With ``alibi_slopes`` ([H_q]) the page bonus ``slope * (last position of
        the page - q_pos)`` is added (``q_pos``: an int for all sequences).
        """
        if not exclude_last_page:
            raise NotImplementedError("only exclude_last_page=True is implemented")
        self.require_tokens()
        from .attention_topk import _alibi_args, _score_and_select
        alibi = None
        if alibi_slopes is not None:
            B, Hq = q.shape[0], q.shape[1]
            q_len = torch.full((B,), int(q_pos) + 1, dtype=torch.int32, device=q.device)
            alibi = _alibi_args(alibi_slopes, q_len, B, Hq, q.device)
        scores = _score_and_select(q, self, token_budget=0, cache_seqlens=None, alibi=alibi)[0]
        return scores[:, :, :max(self.num_pages - 1, 0)]

    # ------------------------------------------------------------------ helpers kept from the reference object

    def select_gaussian_aware(self, q: torch.Tensor, alpha: float = 1.5, safety_margin_z: float = 0.0,
                              max_quantile: float = 0.99, gaussian_stats: Optional[dict] = None):
        """Gaussian-aware page selection on its own (kv_cache.py:205-255).

        Returns ``(page_indices int32 [B, H_q, pages], num_selected int32 [B, H_q])``: per head the
        selected pages in ascending order with the in-progress last page in the final valid slot; only
        the first ``num_selected`` entries of a row are meaningful.  ``safety_margin_z`` and
        ``max_quantile`` are derived from the batch's mean sigma exactly as the decode wrapper does, so
        the arguments have no effect (as in the reference, where the statistics dictionary overrides
        them).  Of ``gaussian_stats`` only ``threshold_excess_margin_fraction`` and
        ``tau_clamp_page_max_quantile`` are read; the statistics themselves are recomputed on the
        device (one sweep) rather than taken from the dictionary.  The statistics and tau_floor of the
        call stay in ``last_gaussian_selection``.
        """
        from .attention_gaussian import gaussian_select
        self.require_tokens()
        stats = gaussian_stats or {}
        frac = stats.get("threshold_excess_margin_fraction", 0.1)
        frac = 0.1 if frac is None else frac
        sel = gaussian_select(q, self, alpha, frac, stats.get("tau_clamp_page_max_quantile", 0.5),
                              apply_clamp=False)
        self.last_num_selected_per_head = sel["num_selected"]
        self.last_gaussian_selection = sel
        return sel["page_indices"], sel["num_selected"]

    def get_page_indices_buf(self, batch: int, num_heads: int, num_pages_to_select: int,
                             last_page_idx: int) -> torch.Tensor:
        """Persistent int32 ``[B, H, n_selected + 1]`` page table whose last column holds
        ``last_page_idx`` (kv_cache.py:167-185).  The wrappers of this library fill their own table
        on the device; the method exists for callers that build page tables themselves."""
        buf = self.scratch("user_page_indices", (batch, num_heads, num_pages_to_select + 1), torch.int32)
        buf[:, :, num_pages_to_select].fill_(last_page_idx)
        return buf

    def get_paged_decode_workspace(self, batch: int, nheads: int, dim: int, max_splits: int = 32,
                                   bins: int = 16, dtype: torch.dtype = None, device=None) -> dict:
        """The decode workspace for one shape (kv_cache.py:187-203).  The reference returns a dictionary
        of Triton intermediates; here it is one byte buffer sized by ``ekv_decode_workspace_bytes``
        (``max_splits`` and ``bins`` do not apply: splits follow the 256-token work list and the
        histogram lives in shared memory)."""
        from .attention_topk import _decode_workspace
        return {"workspace": _decode_workspace(self, batch, nheads, dim, self.capacity)}
