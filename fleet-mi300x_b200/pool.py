"""The life of cache pages: forked, released, reserved, compacted and copied.

The caches of a model's layers share one block table, so an operation on requests is one
call for all layers. A PagePool counts on the device who holds which page; every method queues
kernels on the current stream and waits for nothing, so a decode loop calls them between
steps, also inside a captured graph:

    pool = PagePool(caches)          # one cache per layer, over one block table
    pool.reserve(1)                  # a page for the next row wherever one is needed
    pool.fork(parents, beams)        # requests become copies of others
    pool.release(finished)

The library keeps pages lowest number first; results depend on the state alone. Errors (too few
free pages, a request outside the batch) reach the host as a decode step's do: `check` as in
MlaDecodeAttention.attend. The reference keeps one flat cache per request
(src/runtime/fleet_types.h:106-111) and has no counterpart.
"""
from __future__ import annotations

import ctypes

import torch

from . import native
from .attention import _ptr, _raw_stream, _scales_ptr, host_word
from .cache import PagedLatentCache, PagedLatentCache8, _check_tensor
from .native import PAGE_SIZE


def _layers(caches) -> list[PagedLatentCache]:
    caches = [caches] if isinstance(caches, PagedLatentCache) else list(caches)
    if not 1 <= len(caches) <= native.MAX_LAYERS:
        raise ValueError(f"a pool has 1 to {native.MAX_LAYERS} layers, got {len(caches)}")
    first = caches[0]
    for c in caches:
        if type(c) is not type(first) or c.n_pages != first.n_pages or c.device != first.device:
            raise ValueError("the layers' caches must be of one class, size and device")
    if first.device.type != "cuda":
        raise RuntimeError("page operations need CUDA tensors (sm_100a); there is no CPU path")
    return caches


def _pages_struct(caches: list[PagedLatentCache]) -> native.MlaPagePool:
    p = native.new_pool()
    p.n_layers, p.n_pages = len(caches), caches[0].n_pages
    p.kv8 = int(isinstance(caches[0], PagedLatentCache8))
    for k, c in enumerate(caches):
        p.pages[k], p.scales[k] = _ptr(c.pages), _scales_ptr(c)
    return p


def _ids(x, device: torch.device) -> torch.Tensor:
    t = x if isinstance(x, torch.Tensor) and x.dtype == torch.int32 and x.device == device else \
        torch.as_tensor(x, dtype=torch.int32, device=device)
    if t.dim() != 1 or not t.is_contiguous():
        raise ValueError("request and page numbers must be one contiguous dimension")
    return t


class PagePool:
    """Who holds which page of the caches of one block table.

    caches: one cache, or one per layer (up to 64), all over the same block_table and seq_lens.
    held (int32 [batch]): pages of each request, its first block-table entries; refs (int32 [n_pages]):
    entries that hold each page, 0 = free. Without them a request holds the pages of its rows,
    ceil(seq_lens / 64), and the counts follow.
    """

    def __init__(self, caches, held: torch.Tensor | None = None, refs: torch.Tensor | None = None):
        self.caches = caches = _layers(caches)
        first = caches[0]
        if any(c.block_table.data_ptr() != first.block_table.data_ptr() or
               c.seq_lens.data_ptr() != first.seq_lens.data_ptr() for c in caches):
            raise ValueError("the layers' caches must share block_table and seq_lens")
        self.device, self.block_table, self.seq_lens = first.device, first.block_table, first.seq_lens
        if held is None:
            held = ((self.seq_lens + PAGE_SIZE - 1) // PAGE_SIZE).to(torch.int32)
        _check_tensor("held", held, torch.int32, (first.batch,))
        if refs is None:
            inside = torch.arange(first.max_blocks, device=self.device)[None, :] < held[:, None]
            refs = torch.bincount(self.block_table[inside].long(), minlength=first.n_pages).to(torch.int32)
        _check_tensor("refs", refs, torch.int32, (first.n_pages,))
        if held.device != self.device or refs.device != self.device:
            raise ValueError("held and refs must be on the caches' device")
        self.held, self.refs = held, refs
        self.error_word = torch.zeros(1, dtype=torch.int32, device=self.device)
        self.error_host = torch.zeros(1, dtype=torch.int32).pin_memory()
        self._error_host = host_word(self.error_host)
        self.lib = native.load_library()
        p = _pages_struct(caches)
        p.batch, p.max_blocks = first.batch, first.max_blocks
        p.block_table, p.seq_lens = _ptr(self.block_table), _ptr(self.seq_lens)
        p.held, p.refs = _ptr(held), _ptr(refs)
        p.error_word, p.error_host = _ptr(self.error_word), _ptr(self.error_host)
        need = ctypes.c_uint64()
        native.check(self.lib.mla_pool_scratch_size(ctypes.byref(p), ctypes.byref(need)), "mla_pool_scratch_size")
        self._scratch = torch.empty(int(need.value), dtype=torch.uint8, device=self.device)
        p.scratch, p.scratch_bytes = _ptr(self._scratch), self._scratch.numel()
        self._p = p

    def fork(self, src, dst, *, check: bool | str = True) -> None:
        """Request dst[i] becomes a copy of request src[i] as it was before the call, for all i at once:
        it shares the full pages and gets its own copy of the rows of a last page that is not
        full. Its former pages, reserved ones among them, are let go of, and entries past its new ones are -1, as after
        release. src[i] == dst[i] changes nothing; a request may
        be both a source and a destination. Too few free pages: nothing changes, MLA_DEV_NO_PAGE."""
        src, dst = _ids(src, self.device), _ids(dst, self.device)
        if src.numel() != dst.numel():
            raise ValueError(f"{src.numel()} sources for {dst.numel()} destinations")
        self._call("mla_pool_fork", check, _ptr(src), _ptr(dst), src.numel())

    def release(self, requests, *, check: bool | str = True) -> None:
        """Let go of the requests' pages; they hold nothing and have no rows afterwards, and their
        block-table entries are -1: a step on one of them, before pages are reserved for it, is an
        error (MLA_DEV_BAD_PAGE) and stores no row."""
        requests = _ids(requests, self.device)
        self._call("mla_pool_release", check, _ptr(requests), requests.numel())

    def reserve(self, tokens: int, requests=None, *, check: bool | str = True) -> None:
        """Pages for `tokens` more rows of the requests (default: all), where they hold too few. Too few
        free pages in all: nothing changes, MLA_DEV_NO_PAGE."""
        ids = None if requests is None else _ids(requests, self.device)
        if ids is None or ids.numel():
            self._call("mla_pool_reserve", check, _ptr(ids), 0 if ids is None else ids.numel(), int(tokens))

    def compact(self, *, check: bool | str = True) -> None:
        """Move the held pages to the lowest numbers, block table and counts with them."""
        self._call("mla_pool_compact", check)

    def free_pages(self) -> int:
        """How many pages nobody holds (waits for the device)."""
        return int((self.refs == 0).sum())

    def _call(self, name: str, check, *args) -> None:
        if check and self._error_host.value and not torch.cuda.is_current_stream_capturing():
            self.raise_pending()
        code = getattr(self.lib, name)(self._p, *args, _raw_stream(self.device))
        if code:
            native.check(code, name)
        if check == "sync" and not torch.cuda.is_current_stream_capturing():
            torch.cuda.current_stream(self.device).synchronize()
            self.raise_pending()

    def raise_pending(self) -> None:
        """Raise MlaError if an earlier call recorded a device error (no synchronisation; see
        MlaDecodeAttention.raise_pending). Clears both words before raising."""
        code = self._error_host.value
        if code:
            self.error_host.zero_()
            if not torch.cuda.is_current_stream_capturing():
                self.error_word.zero_()
            raise native.MlaError(code, "device (a page operation since the last check)")


def copy_pages(src_caches, src, dst_caches, dst, *, error_word: torch.Tensor | None = None) -> None:
    """Page src[i] of every source cache into page dst[i] of the destination cache beside it (one cache each,
    or lists of layers; the two may be the same): a swap to another pool, or a move within one.
    No destination may appear twice, nor be a source of the same call. Counts and block tables
    are the caller's. A page number outside its pool is skipped and recorded in error_word."""
    a = _layers(src_caches)
    b = a if dst_caches is src_caches else _layers(dst_caches)
    if len(a) != len(b) or type(a[0]) is not type(b[0]) or a[0].device != b[0].device:
        raise ValueError("copies go between caches of one class, device and number of layers")
    src, dst = _ids(src, a[0].device), _ids(dst, a[0].device)
    if src.numel() != dst.numel():
        raise ValueError(f"{src.numel()} sources for {dst.numel()} destinations")
    p = _pages_struct(a)
    q = p if b is a else _pages_struct(b)
    q.error_word = _ptr(error_word)
    native.check(native.load_library().mla_copy_pages(q, p, _ptr(src), _ptr(dst), src.numel(),
                                                      _raw_stream(a[0].device)), "mla_copy_pages")
