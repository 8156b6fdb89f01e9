"""Paged key-value cache of the decode path: the mirror of ``KvPool``, ``KvCache`` and
``BatchedKvCache`` of the reference (kernel_src/src/loquetier/utils/kvcache.py:7-50, 87-141, 143-165)
with the same constructors, properties and methods, plus the three attention-side operators
``batch_prefill``, ``batch_decode``, ``init_kv`` and ``append_kv`` of kernel_src/src/loquetier/ops/__init__.py:18-170
on the B200 kernels.

A page is one tensor ``[num_layers, 2, num_heads, page_len, head_dim]``, as in the reference.  The pool
hands pages out of large slabs instead of one device allocation per page: a slab of 180 GB-class HBM
is cut once, pages are views into it and go back to a free list, so steady-state decoding never calls
the allocator.

Beyond the reference: caches can be continued several ways (``KvCache.fork``, ``fork_caches``: full pages are shared and
counted, the filled part of a last page is copied), grow and shrink by several tokens (``extend``, ``truncate``), a
fragmented pool can be drawn together (``KvPool.compact``), ``batch_extend`` attends from a chunk of new tokens per request,
and ``norm_append_kv`` normalises queries and keys per head on their way into the cache."""
from __future__ import annotations

import bisect
from collections import Counter
from collections.abc import Iterable, Sequence
from typing import Any, List, Optional

import torch

from . import cabi
from .cabi import check, lib
from .ops import (_chk_cuda_contig, _stream, clear_recorded_workspace, device_ints, note_fresh_workspace, on_device,
                  refuse_capture, row_stride)

_DT = {torch.float16: cabi.SMLM_F16, torch.bfloat16: cabi.SMLM_BF16}


class KvPool:
    def __init__(self, num_layers: int, num_heads: int, head_dim: int, page_len: int, dtype: torch.dtype,
                 device: torch.device, pages_per_slab: int = 256):
        self.num_layers = num_layers
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.page_len = page_len
        self.dtype = dtype
        self.device = torch.device(device)
        self._page_shape = (num_layers, 2, num_heads, page_len, head_dim)
        self._page_meta = torch.empty(self._page_shape, dtype=dtype, device="meta")
        self._pages_per_slab = int(pages_per_slab)
        self._slabs: List[torch.Tensor] = []
        self._free: List[torch.Tensor] = []
        self._allocated = {}
        self._holders = {}   # address -> holders of a page that has more than one

    @property
    def page_meta(self) -> torch.Tensor:
        return self._page_meta

    @property
    def page_nbytes(self) -> int:
        return self._page_meta.nbytes

    @property
    def num_pages(self) -> int:
        return len(self._allocated)

    def allocated_pages(self) -> Iterable[torch.Tensor]:
        return iter(self._allocated.values())

    def alloc_page(self) -> torch.Tensor:
        if not self._free:
            slab = torch.empty((self._pages_per_slab,) + self._page_shape, dtype=self.dtype, device=self.device)
            self._slabs.append(slab)
            self._free.extend(slab[i] for i in range(self._pages_per_slab - 1, -1, -1))
        page = self._free.pop()
        self._allocated[page.data_ptr()] = page
        return page

    def alloc_pages(self, n: int) -> List[torch.Tensor]:
        """``n`` pages, or none where the memory does not suffice."""
        pages = []
        try:
            for _ in range(n):
                pages.append(self.alloc_page())
        except BaseException:
            for page in pages:
                self.free_page(page)
            raise
        return pages

    def free_page(self, page: torch.Tensor) -> None:
        """Gives up one hold of the page; the last one makes it free."""
        ptr = page.data_ptr()
        n = self._holders.get(ptr, 1)
        if n > 1:
            self._holders[ptr] = n - 1
            return
        del self._allocated[ptr]
        self._holders.pop(ptr, None)
        self._free.append(page)

    def share_page(self, page: torch.Tensor) -> torch.Tensor:
        """One more holder of an allocated page; each of them frees it once."""
        ptr = page.data_ptr()
        if ptr not in self._allocated:
            raise RuntimeError("the page is not allocated")
        self._holders[ptr] = self._holders.get(ptr, 1) + 1
        return page

    def page_holders(self, page: torch.Tensor) -> int:
        """How many hold the page: 0 where it is free."""
        ptr = page.data_ptr()
        return self._holders.get(ptr, 1) if ptr in self._allocated else 0

    @property
    def num_slabs(self) -> int:
        return len(self._slabs)

    def compact(self, caches: Iterable["KvCache"]) -> int:
        """Empties as many slabs as the free pages of the others allow and gives their memory back to the allocator.
        Returns their number.

        Pages move only if ``caches`` hold them alone (a page that something else holds stays, and its slab with it).  They
        are copied by one launch on the current stream and the caches' page tables follow; a ``BatchedKvCache`` made before
        has to be made again.  Work that still reads the old pages has to be on this stream or have finished."""
        caches = list({id(c): c for c in caches}.values())
        if any(c.pool is not self for c in caches):
            raise RuntimeError("every cache must be of this pool")
        if not self._slabs:
            return 0
        refuse_capture(self._slabs[0], "KvPool.compact")
        held = Counter(p.data_ptr() for c in caches for p in c.pages)
        bases = sorted((slab.data_ptr(), i) for i, slab in enumerate(self._slabs))
        starts = [b for b, _ in bases]

        def slab_of(ptr):
            return bases[bisect.bisect_right(starts, ptr) - 1][1]

        used = [[] for _ in self._slabs]
        free = [[] for _ in self._slabs]
        stays = [False] * len(self._slabs)
        for ptr, page in self._allocated.items():
            used[slab_of(ptr)].append(page)
            if held[ptr] != self._holders.get(ptr, 1):
                stays[slab_of(ptr)] = True
        for page in self._free:
            free[slab_of(page.data_ptr())].append(page)
        # the emptiest first, as long as the rest has room for what they hold
        room, load, emptied = sum(len(f) for f in free), 0, []
        for i in sorted(range(len(self._slabs)), key=lambda i: len(used[i])):
            if stays[i]:
                continue
            if load + len(used[i]) > room - len(free[i]):
                break
            room -= len(free[i])
            load += len(used[i])
            emptied.append(i)
        if not emptied:
            return 0
        gone = set(emptied)
        # into the fullest of the others first
        kept = sorted((i for i in range(len(self._slabs)) if i not in gone), key=lambda i: -len(used[i]))
        targets = [p for i in kept for p in free[i]]
        src = [p for i in emptied for p in used[i]]
        dst = targets[:len(src)]
        if src:
            copy_pages(self, *_page_tables(self.device, dst, src))
        moved = {a.data_ptr(): b for a, b in zip(src, dst)}
        for old, page in moved.items():
            del self._allocated[old]
            self._allocated[page.data_ptr()] = page
            if old in self._holders:
                self._holders[page.data_ptr()] = self._holders.pop(old)
        for c in caches:
            if any(p.data_ptr() in moved for p in c.pages):
                c._replace_pages([moved.get(p.data_ptr(), p) for p in c.pages])
        self._free = targets[len(src):][::-1]   # the fullest slabs' pages are handed out first
        for i in emptied:
            if self._slabs[i].is_cuda:   # the copies above may still read it
                self._slabs[i].record_stream(torch.cuda.current_stream(self._slabs[i].device))
        self._slabs = [slab for i, slab in enumerate(self._slabs) if i not in gone]
        return len(emptied)


class GrowableTensor:
    """A 1-D device tensor that grows by doubling (kvcache.py:52-84 of the reference)."""

    def __init__(self, data: Sequence[Any], dtype: Optional[torch.dtype] = None, device=None):
        self._buf = torch.tensor(list(data), dtype=dtype, device=device)
        self._len = len(data)
        self._pending = []   # integers of extend() that no view has asked for yet

    def view(self) -> torch.Tensor:
        self._flush()
        return self._buf[:self._len]

    def append(self, data: Any) -> None:
        self._flush()
        if self._buf.numel() < self._len + 1:
            cap = 1 << max(0, self._len).bit_length()
            new = torch.empty(max(cap, 1), dtype=self._buf.dtype, device=self._buf.device)
            new[:self._len] = self._buf[:self._len]
            self._buf = new
        self._buf[self._len] = data
        self._len += 1

    def extend(self, data: Sequence[int]) -> None:
        """Appends integers; they go to the device together when they are next looked at."""
        self._pending += data

    def _flush(self) -> None:
        if not self._pending:
            return
        refuse_capture(self._buf, "the first look at a cache's page table after it grew")
        length = self._len + len(self._pending)
        new = device_ints(self._pending, self._buf.dtype, self._buf.device)
        if self._len == 0:
            self._buf = new
        else:
            if self._buf.numel() < length:
                buf = torch.empty(1 << (length - 1).bit_length(), dtype=self._buf.dtype, device=self._buf.device)
                buf[:self._len] = self._buf[:self._len]
                self._buf = buf
            self._buf[self._len:length] = new
        self._len, self._pending = length, []

    def truncate(self, length: int) -> None:
        del self._pending[max(0, length - self._len):]
        self._len = min(self._len, length)

    def clear(self) -> None:
        self.truncate(0)


class KvCache:
    """Key-value cache for one sequence."""

    def __init__(self, pool: KvPool, init_len: int):
        if init_len < 0:
            raise ValueError("init_len must be non-negative")
        self._pool = pool
        self._pages = pool.alloc_pages((init_len + pool.page_len - 1) // pool.page_len)
        self._seqlen = init_len
        try:
            self._ptrs = GrowableTensor([t.data_ptr() for t in self._pages], dtype=torch.int64, device=pool.device)
        except BaseException:
            for page in self._pages:
                pool.free_page(page)
            raise

    pool = property(lambda self: self._pool)
    seqlen = property(lambda self: self._seqlen)
    ptrs = property(lambda self: self._ptrs.view())
    pages = property(lambda self: self._pages)
    num_pages = property(lambda self: len(self._pages))

    def acquire_one(self):
        """Reserve space for one more token."""
        last_page_offset = (self._seqlen - 1) % self._pool.page_len + 1
        if last_page_offset == self._pool.page_len:
            self._pages.append(self._pool.alloc_page())
            self._ptrs.append(self._pages[-1].data_ptr())
        self._seqlen += 1

    def extend(self, n: int):
        """Reserve space for ``n`` more tokens."""
        if n < 0:
            raise ValueError("n must be non-negative")
        need = -(-(self._seqlen + n) // self._pool.page_len) - len(self._pages)
        new = self._pool.alloc_pages(need)
        self._pages.extend(new)
        self._ptrs.extend([p.data_ptr() for p in new])
        self._seqlen += n

    def truncate(self, seqlen: int):
        """Drop the tokens behind the first ``seqlen`` (drafted ones that were rejected).  A last page that others
        hold too is replaced by a copy of what is left of it, since the next tokens go there."""
        if not 0 <= seqlen <= self._seqlen:
            raise ValueError(f"seqlen must be between 0 and {self._seqlen}")
        if seqlen == self._seqlen:
            return
        pool = self._pool
        npages, entries = -(-seqlen // pool.page_len), seqlen % pool.page_len
        own = None
        if entries and pool.page_holders(self._pages[npages - 1]) > 1:
            refuse_capture(self._pages[npages - 1], "KvCache.truncate into a shared page")
            own = pool.alloc_page()
            try:
                copy_pages(pool, *_page_tables(pool.device, [own], [self._pages[npages - 1]], [entries]))
            except BaseException:
                pool.free_page(own)
                raise
        for page in self._pages[npages - (own is not None):]:
            pool.free_page(page)
        if own is not None:
            self._replace_pages(self._pages[:npages - 1] + [own])
        else:
            del self._pages[npages:]
            self._ptrs.truncate(npages)
        self._seqlen = seqlen

    def fork(self, copies: int = 1) -> List["KvCache"]:
        """``copies`` caches with the same tokens, to be continued on their own (``fork_caches`` for several at once)."""
        return fork_caches([self], copies)[0]

    def _replace_pages(self, pages: List[torch.Tensor]):
        self._pages[:] = pages
        self._ptrs = GrowableTensor([], dtype=torch.int64, device=self._pool.device)
        self._ptrs.extend([p.data_ptr() for p in pages])

    def release(self):
        """Release all pages."""
        self._seqlen = 0
        for page in self._pages:
            self._pool.free_page(page)
        self._pages.clear()
        self._ptrs.clear()


def fork_caches(caches: Sequence[KvCache], copies: int = 1) -> List[List[KvCache]]:
    """Continues every cache ``copies`` ways: for each of them that many caches with the same tokens.  Their full pages are
    shared and counted; the filled part of a last page that is not full is copied, for all of them by one launch on the
    current stream, since the next tokens go there."""
    if copies < 0:
        raise ValueError("copies must be non-negative")
    caches = list(caches)
    if not caches:
        return []
    pool = caches[0].pool
    if any(c.pool is not pool for c in caches):
        raise RuntimeError("every cache must be of the same pool")
    partial = [c for c in caches if c.seqlen % pool.page_len]
    if partial and copies:
        refuse_capture(partial[0].pages[-1], "a fork that copies pages")
    tails = pool.alloc_pages(len(partial) * copies)
    try:
        if tails:
            src = [c.pages[-1] for c in partial for _ in range(copies)]
            entries = [c.seqlen % pool.page_len for c in partial for _ in range(copies)]
            copy_pages(pool, *_page_tables(pool.device, tails, src, entries))
    except BaseException:
        for page in tails:
            pool.free_page(page)
        raise
    rest, out = iter(tails), []
    for c in caches:
        full = c.seqlen // pool.page_len
        out.append([])
        for _ in range(copies):
            child = KvCache(pool, 0)
            pages = [pool.share_page(p) for p in c.pages[:full]]
            if c.seqlen % pool.page_len:
                pages.append(next(rest))
            child._replace_pages(pages)
            child._seqlen = c.seqlen
            out[-1].append(child)
    return out


def _page_tables(device, dst: Sequence[torch.Tensor], src: Sequence[torch.Tensor], entries: Optional[Sequence[int]] = None):
    """Device tables of page addresses (and positions) for ``copy_pages``."""
    n = len(dst)
    ptrs = device_ints([p.data_ptr() for p in dst] + [p.data_ptr() for p in src], torch.int64, device)
    return ptrs[:n], ptrs[n:], None if entries is None else device_ints(entries, torch.int32, device)


class BatchedKvCache:
    """Key-value cache for a batch of sequences: page pointers of all sequences back to back, the page
    index pointer and the number of valid entries of every last page."""

    def __init__(self, kv: Sequence[KvCache]):
        assert len(kv) > 0
        pool = kv[0].pool
        ptrs, indptr, last = [], [0], []
        for c in kv:
            assert c.pool is pool
            assert c.num_pages > 0
            ptrs.append(c.ptrs)
            indptr.append(indptr[-1] + c.num_pages)
            last.append((c.seqlen - 1) % pool.page_len + 1)
        self.pool = pool
        self.ptrs = torch.cat(ptrs)
        self.indptr = torch.tensor(indptr, dtype=torch.int32, device=pool.device)
        self.last_page_offset = torch.tensor(last, dtype=torch.int32, device=pool.device)


# ---------------------------------------------------------------------------
# operators (the reference's loquetier.ops.batch_decode / init_kv / append_kv)
# ---------------------------------------------------------------------------

_WORKSPACES = {}
_WS_HEAD = {}   # device -> bytes of tickets at the head of the workspace for the batch it last served
_WS_RECORDED = set()   # devices whose workspace was made under capture (ops.clear_recorded_workspace)


def _dtype_code(t):
    try:
        return _DT[t.dtype]
    except KeyError:
        raise RuntimeError(f"No suitable kernel. dtype={t.dtype}") from None


def decode_workspace(device, batch: int, num_qo_heads: int, num_kv_heads: int) -> Optional[torch.Tensor]:
    """Scratch of the decode kernel with its tickets zeroed, cached per device and grown on demand.  The kernel
    leaves the tickets zeroed; a batch whose tickets take another head moves the boundary between tickets and
    parked softmax states, so the head is cleared then.  Ask for it right before the launch; calls that may
    overlap on different streams need workspaces of their own."""
    shape = (int(batch), int(num_qo_heads), int(num_kv_heads))
    need = int(lib.smlm_b200_batch_decode_workspace_bytes(*shape))
    head = int(lib.smlm_b200_batch_decode_ticket_bytes(shape[0], shape[2]))
    ws = _WORKSPACES.get(device)
    if ws is None or ws.numel() < need:
        ws = torch.zeros(max(need, 1 << 16), dtype=torch.uint8, device=device)
        _WORKSPACES[device] = ws
        note_fresh_workspace(_WS_RECORDED, device, ws)
    elif device in _WS_RECORDED:
        clear_recorded_workspace(_WS_RECORDED, device, ws, head)
    elif _WS_HEAD.get(device) != head:
        with on_device(ws):
            ws[:head].zero_()
    _WS_HEAD[device] = head
    return ws


def batch_decode_into(o, q, kv_ptrs, kv_indptr, last_page_offset, num_layers, layer_idx, num_kv_heads, base, page_size,
                      workspace=None, status_word=None):
    ws = workspace if workspace is not None else decode_workspace(q.device, q.size(0), q.size(1), num_kv_heads)
    with on_device(q):
        check(lib.smlm_b200_batch_decode(o.data_ptr(), q.data_ptr(), kv_ptrs.data_ptr(), kv_indptr.data_ptr(),
                                         last_page_offset.data_ptr(), ws.data_ptr(), ws.numel(),
                                         None if status_word is None else status_word.data_ptr(),
                                         int(q.size(0)), int(kv_ptrs.numel()), int(q.size(1)), int(num_kv_heads),
                                         int(q.size(2)), int(num_layers), int(layer_idx), int(page_size), float(base),
                                         _dtype_code(q), _stream(q)), "smlm_b200_batch_decode")
    return o


def batch_decode(q: torch.Tensor, kv: BatchedKvCache, base: float, layer_idx: int) -> torch.Tensor:
    """Self-attention with rotary position encoding for a batch of one-token requests.  ``q``
    ``[batch, num_heads, head_dim]`` and the keys in ``kv`` are NOT position encoded.  Returns
    ``[batch, num_heads, head_dim]``."""
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    return batch_decode_into(o, q, kv.ptrs, kv.indptr, kv.last_page_offset, kv.pool.num_layers, layer_idx,
                             kv.pool.num_heads, base, kv.pool.page_len)


_PREFILL_WS = {}


def prefill_workspace(device, total_pages: int, page_size: int, num_kv_heads: int) -> torch.Tensor:
    """Scratch of the prefill kernels (a dense, rotated copy of the batch's keys and values), cached per
    device and grown on demand.  Calls that may overlap on different streams need workspaces of their own."""
    need = int(lib.smlm_b200_batch_prefill_workspace_bytes(int(total_pages), int(page_size), int(num_kv_heads)))
    ws = _PREFILL_WS.get(device)
    if ws is None or ws.numel() < need:
        ws = torch.empty(max(need, 1 << 20), dtype=torch.uint8, device=device)
        _PREFILL_WS[device] = ws
    return ws


def batch_prefill_into(o, q, qo_indptr, kv_ptrs, kv_indptr, last_page_offset, num_layers, layer_idx, num_kv_heads,
                       base, page_size, workspace=None, status_word=None):
    ws = workspace if workspace is not None else prefill_workspace(q.device, kv_ptrs.numel(), page_size,
                                                                   num_kv_heads)
    with on_device(q):
        check(lib.smlm_b200_batch_prefill(o.data_ptr(), q.data_ptr(), qo_indptr.data_ptr(), kv_ptrs.data_ptr(),
                                          kv_indptr.data_ptr(), last_page_offset.data_ptr(), ws.data_ptr(),
                                          ws.numel(), None if status_word is None else status_word.data_ptr(),
                                          int(last_page_offset.numel()), int(q.size(0)), int(kv_ptrs.numel()),
                                          int(q.size(1)), int(num_kv_heads), int(q.size(2)), int(num_layers),
                                          int(layer_idx), int(page_size), float(base), _dtype_code(q), _stream(q)),
              "smlm_b200_batch_prefill")
    return o


def batch_prefill(q: torch.Tensor, qo_indptr: torch.Tensor, kv: BatchedKvCache, base: float,
                  layer_idx: int) -> torch.Tensor:
    """Causal self-attention with rotary position encoding for each prompt of the batch
    (batch_prefill, kernel_src/src/loquetier/ops/__init__.py:18-57).  ``q``
    ``[sum(seqlen), num_heads, head_dim]`` and the keys in ``kv`` are NOT position encoded; request b owns
    rows ``qo_indptr[b] .. qo_indptr[b + 1]`` (int32, on the device).  Returns the attention output in the
    shape of ``q``."""
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    return batch_prefill_into(o, q, qo_indptr, kv.ptrs, kv.indptr, kv.last_page_offset, kv.pool.num_layers,
                              layer_idx, kv.pool.num_heads, base, kv.pool.page_len)


def init_kv_raw(kv_ptrs, kv_indptr, last_page_offset, k, v, seqlen_indptr, num_layers, layer_idx, num_kv_heads,
                page_size, status_word=None):
    with on_device(k):
        check(lib.smlm_b200_init_kv(kv_ptrs.data_ptr(), kv_indptr.data_ptr(), last_page_offset.data_ptr(),
                                    k.data_ptr(), v.data_ptr(), seqlen_indptr.data_ptr(),
                                    None if status_word is None else status_word.data_ptr(),
                                    int(last_page_offset.numel()), int(kv_ptrs.numel()), int(k.size(0)),
                                    int(num_layers), int(layer_idx), int(num_kv_heads), int(k.size(2)),
                                    int(page_size), _dtype_code(k), _stream(k)), "smlm_b200_init_kv")


def init_kv(kv: BatchedKvCache, k: torch.Tensor, v: torch.Tensor, seqlen_indptr: torch.Tensor, layer_idx: int):
    """Copy ``k`` and ``v`` ``[sum(seqlen), num_heads, head_dim]`` to the cache; the pages of each
    sequence are already allocated in ``kv``."""
    init_kv_raw(kv.ptrs, kv.indptr, kv.last_page_offset, k, v, seqlen_indptr, kv.pool.num_layers, layer_idx,
                kv.pool.num_heads, kv.pool.page_len)


def append_kv_raw(kv_ptrs, kv_indptr, last_page_offset, k, v, num_layers, layer_idx, num_kv_heads, page_size,
                  status_word=None):
    with on_device(k):
        check(lib.smlm_b200_append_kv(kv_ptrs.data_ptr(), kv_indptr.data_ptr(), last_page_offset.data_ptr(),
                                      k.data_ptr(), v.data_ptr(),
                                      None if status_word is None else status_word.data_ptr(), int(k.size(0)),
                                      int(kv_ptrs.numel()), int(num_layers), int(layer_idx), int(num_kv_heads),
                                      int(k.size(2)), int(page_size), _dtype_code(k), _stream(k)),
              "smlm_b200_append_kv")


def append_kv(kv: BatchedKvCache, k: torch.Tensor, v: torch.Tensor, layer_idx: int):
    """Append the new token's ``k`` and ``v`` ``[batch, num_heads, head_dim]``; the page for the new token
    of each sequence is already allocated in ``kv``."""
    append_kv_raw(kv.ptrs, kv.indptr, kv.last_page_offset, k, v, kv.pool.num_layers, layer_idx, kv.pool.num_heads,
                  kv.pool.page_len)


# ---------------------------------------------------------------------------
# operators around a cache that several continuations share
# ---------------------------------------------------------------------------

def copy_pages(pool: KvPool, dst: torch.Tensor, src: torch.Tensor, entries: Optional[torch.Tensor] = None,
               status_word: Optional[torch.Tensor] = None) -> None:
    """Copies pages of ``pool``: the page at address ``src[i]`` to the one at ``dst[i]`` (int64 tensors on the device), all
    layers and heads, the first ``entries[i]`` positions (int32; None: whole pages).  A page may be the source of several
    copies; none may be the destination of two, nor source and destination at once."""
    for t, name in ((dst, "dst"), (src, "src")):
        _chk_cuda_contig(t, name, 1)
        if t.dtype != torch.int64:
            raise RuntimeError(f"{name} must be int64")
    if dst.numel() != src.numel():
        raise RuntimeError(f"dst and src must have the same length. {dst.numel()} vs {src.numel()}")
    if entries is not None:
        _chk_cuda_contig(entries, "entries", 1)
        if entries.dtype != torch.int32 or entries.numel() != dst.numel():
            raise RuntimeError("entries must hold one int32 per page")
    _chk_same_device(dst, src=src, entries=entries, status_word=status_word)
    try:
        dtype = _DT[pool.dtype]
    except KeyError:
        raise RuntimeError(f"No suitable kernel. dtype={pool.dtype}") from None
    with on_device(dst):
        check(lib.smlm_b200_copy_pages(dst.data_ptr(), src.data_ptr(), None if entries is None else entries.data_ptr(),
                                       None if status_word is None else status_word.data_ptr(), int(dst.numel()),
                                       int(pool.num_layers), int(pool.num_heads), int(pool.head_dim), int(pool.page_len),
                                       dtype, _stream(dst)), "smlm_b200_copy_pages")


def _chk_same_device(ref: torch.Tensor, **others):
    for name, t in others.items():
        if t is not None and t.device != ref.device:
            raise RuntimeError(f"{name} must be on {ref.device}")


def batch_extend_into(o, q, qo_indptr, kv_ptrs, kv_indptr, last_page_offset, num_layers, layer_idx, num_kv_heads, base,
                      page_size, workspace=None, status_word=None):
    batch, rows, pages, heads = int(last_page_offset.numel()), int(q.size(0)), int(kv_ptrs.numel()), int(q.size(1))
    if workspace is None:   # from the allocator, call by call: streams and captured graphs each get their own
        need = int(lib.smlm_b200_batch_extend_workspace_bytes(batch, rows, pages, int(page_size), heads, int(num_kv_heads)))
        workspace = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    with on_device(q):
        check(lib.smlm_b200_batch_extend(o.data_ptr(), q.data_ptr(), qo_indptr.data_ptr(), kv_ptrs.data_ptr(),
                                         kv_indptr.data_ptr(), last_page_offset.data_ptr(),
                                         None if workspace is None else workspace.data_ptr(),
                                         0 if workspace is None else workspace.numel(),
                                         None if status_word is None else status_word.data_ptr(), batch, rows, pages, heads,
                                         int(num_kv_heads), int(q.size(2)), int(num_layers), int(layer_idx), int(page_size),
                                         float(base), _dtype_code(q), _stream(q)), "smlm_b200_batch_extend")
    return o


def batch_extend(q: torch.Tensor, qo_indptr: torch.Tensor, kv: BatchedKvCache, base: float, layer_idx: int) -> torch.Tensor:
    """Causal self-attention with rotary position encoding of a chunk of new tokens per request over its cache, which
    already holds their keys and values (drafted tokens to verify, a conversation's next turn, a prompt taken in
    pieces).  ``q`` ``[sum(new tokens), num_heads, head_dim]`` and the keys in ``kv`` are NOT position encoded; request b owns
    rows ``qo_indptr[b] .. qo_indptr[b + 1]`` (int32, on the device; it may own none), its last one stands at the cache's
    last position.  Returns the attention output in the shape of ``q``; rows of no request are not written.

    1, 2, 4 or 8 query heads per kv head, ``q`` contiguous.  Whole prompts, and many requests with 64 new tokens or more on short
    caches, are faster through ``batch_prefill``.  Batches whose row tiles times key tiles (of up to 128 rows and 64 keys, over the
    whole batch) reach 2^31 are refused."""
    _chk_cuda_contig(q, "q", 3)
    _chk_cuda_contig(qo_indptr, "qo_indptr", 1)
    pool = kv.pool
    if qo_indptr.dtype != torch.int32 or qo_indptr.numel() != kv.last_page_offset.numel() + 1:
        raise RuntimeError(f"qo_indptr must hold {kv.last_page_offset.numel() + 1} int32 values")
    if q.dtype != pool.dtype or q.size(2) != pool.head_dim:
        raise RuntimeError(f"q must be {pool.dtype} with heads of {pool.head_dim} like the cache")
    _chk_same_device(q, qo_indptr=qo_indptr, kv=kv.ptrs)
    return batch_extend_into(torch.empty_like(q), q, qo_indptr, kv.ptrs, kv.indptr, kv.last_page_offset, pool.num_layers,
                             layer_idx, pool.num_heads, base, pool.page_len)


def norm_append_kv(kv: BatchedKvCache, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_weight: torch.Tensor,
                   k_weight: torch.Tensor, eps: float, layer_idx: int, seqlen_indptr: Optional[torch.Tensor] = None,
                   status_word: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The way of new tokens into the cache for models that normalise queries and keys per head (RMSNorm over head_dim):
    returns the normalised queries and writes the normalised keys and the values into the pages, which already account
    for the tokens.  Neither is position encoded: the attention operators rotate what they read.

    ``q`` ``[tokens, num_heads, head_dim]``, ``k`` and ``v`` ``[tokens, num_kv_heads, head_dim]`` may be slices of one
    projection (rows any multiple of 8 elements apart, heads contiguous); ``q_weight`` and ``k_weight`` ``[head_dim]``.
    ``seqlen_indptr`` (int32, on the device): request b's tokens, as for ``init_kv``; None: one token per request, as for
    ``append_kv``.  Queries of rows of no request are not written."""
    pool = kv.pool
    D, dtype = pool.head_dim, pool.dtype
    strides = [row_stride(t, name, D) for t, name in ((q, "q"), (k, "k"), (v, "v"))]
    for t, name in ((q_weight, "q_weight"), (k_weight, "k_weight")):
        _chk_cuda_contig(t, name, 1)
        if t.numel() != D:
            raise RuntimeError(f"{name} must hold {D} values")
    for t, name in ((q, "q"), (k, "k"), (v, "v"), (q_weight, "q_weight"), (k_weight, "k_weight")):
        if t.dtype != dtype:
            raise RuntimeError(f"{name} must be {dtype} like the cache")
    batch, tokens = int(kv.last_page_offset.numel()), int(q.size(0))
    if k.shape != v.shape or k.size(0) != tokens or k.size(1) != pool.num_heads:
        raise RuntimeError(f"k and v must be [{tokens}, {pool.num_heads}, {D}]")
    if seqlen_indptr is not None:
        _chk_cuda_contig(seqlen_indptr, "seqlen_indptr", 1)
        if seqlen_indptr.dtype != torch.int32 or seqlen_indptr.numel() != batch + 1:
            raise RuntimeError(f"seqlen_indptr must hold {batch + 1} int32 values")
    elif tokens != batch:
        raise RuntimeError(f"without seqlen_indptr there must be one token per request. {tokens} vs {batch}")
    _chk_same_device(q, k=k, v=v, q_weight=q_weight, k_weight=k_weight, seqlen_indptr=seqlen_indptr, kv=kv.ptrs,
                     status_word=status_word)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    with on_device(q):
        check(lib.smlm_b200_norm_append_kv(out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), q_weight.data_ptr(),
                                           k_weight.data_ptr(), kv.ptrs.data_ptr(), kv.indptr.data_ptr(),
                                           kv.last_page_offset.data_ptr(),
                                           None if seqlen_indptr is None else seqlen_indptr.data_ptr(),
                                           None if status_word is None else status_word.data_ptr(), *strides, batch, tokens,
                                           int(kv.ptrs.numel()), int(q.size(1)), int(k.size(1)), D,
                                           int(pool.num_layers), int(layer_idx), int(pool.page_len), float(eps),
                                           _dtype_code(q), _stream(q)), "smlm_b200_norm_append_kv")
    return out
