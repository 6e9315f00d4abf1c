"""Paged latent KV cache of one layer and its block table.

The reference keeps one flat cache per layer, `[max_pos][kv_lora + qk_rope]` bf16
(src/runtime/fleet_types.h:106-111, src/host/kv_convert.py:36-59), appended in place
at `pos` (reference_decode.py:236-237). Here the same 576-wide rows (c_kv | k_pe,
k_pe already RoPE'd) live in 64-row pages `[n_pages][64][576]` bf16; request b's
logical row t is page `block_table[b][t // 64]`, slot `t % 64`. `seq_lens[b]` is the
number of rows already cached, i.e. the position of the token being decoded.
"""
from __future__ import annotations

import torch

from .native import KV_LORA, PAGE8_BYTES, PAGE_SIZE, QK_ROPE, ROW, SCALE_BLOCK


def _check_tensor(name: str, t: torch.Tensor, dtype: torch.dtype, shape: tuple) -> None:
    """Dtype, shape (None: any positive size) and contiguity of a caller's tensor."""
    if t.dtype != dtype or t.dim() != len(shape) or any(
            n <= 0 if want is None else n != want for n, want in zip(t.shape, shape)):
        raise ValueError(f"{name} must be {dtype} [{', '.join('*' if n is None else str(n) for n in shape)}], "
                         f"got {t.dtype} {tuple(t.shape)}")
    if not t.is_contiguous():
        raise ValueError(f"{name} must be contiguous")


class PagedLatentCache:
    def __init__(self, n_pages: int, batch: int, max_blocks: int, device: torch.device | str = "cuda",
                 zero: bool = True):
        if n_pages <= 0 or batch <= 0 or max_blocks <= 0:
            raise ValueError("n_pages, batch and max_blocks must be positive")
        alloc = torch.zeros if zero else torch.empty
        self.pages = alloc(n_pages, PAGE_SIZE, ROW, dtype=torch.bfloat16, device=device)
        self.block_table = torch.zeros(batch, max_blocks, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)

    @classmethod
    def from_tensors(cls, pages: torch.Tensor, block_table: torch.Tensor, seq_lens: torch.Tensor
                     ) -> "PagedLatentCache":
        """A cache over tensors that the caller keeps (its own page pool, a block table and row
        counts shared by the layers of a model): nothing is copied."""
        _check_tensor("pages", pages, torch.bfloat16, (None, PAGE_SIZE, ROW))
        return cls._adopt(pages, block_table, seq_lens)

    @classmethod
    def _adopt(cls, pages, block_table, seq_lens):
        _check_tensor("block_table", block_table, torch.int32, (None, None))
        _check_tensor("seq_lens", seq_lens, torch.int32, (block_table.shape[0],))
        if not pages.device == block_table.device == seq_lens.device:
            raise ValueError("pages, block_table and seq_lens must be on one device")
        self = cls.__new__(cls)
        self.pages, self.block_table, self.seq_lens = pages, block_table, seq_lens
        return self

    @property
    def batch(self) -> int:
        return self.block_table.shape[0]

    @property
    def n_pages(self) -> int:
        return self.pages.shape[0]

    @property
    def max_blocks(self) -> int:
        return self.block_table.shape[1]

    @property
    def device(self) -> torch.device:
        return self.pages.device

    @classmethod
    def for_lengths(cls, lengths, *, extra_tokens: int = 1, spare_pages: int = 0, permute: bool = True,
                    generator: torch.Generator | None = None, device="cuda", zero: bool = True
                    ) -> "PagedLatentCache":
        """A cache whose request b can hold lengths[b] + extra_tokens rows, with
        seq_lens = lengths. Pages are handed out in a random permutation when
        `permute` (the fragmented layout of a long-running server)."""
        lengths = [int(x) for x in lengths]
        need = [(n + extra_tokens + PAGE_SIZE - 1) // PAGE_SIZE for n in lengths]
        total = max(1, sum(need) + spare_pages)
        max_blocks = max(1, max(need))
        cache = cls(total, len(lengths), max_blocks, device=device, zero=zero)
        order = (torch.randperm(total, generator=generator) if permute else torch.arange(total))
        order = order.to(torch.int32)
        bt = torch.zeros(len(lengths), max_blocks, dtype=torch.int32)
        off = 0
        for b, n in enumerate(need):
            bt[b, :n] = order[off:off + n]
            off += n
        cache.block_table.copy_(bt)
        cache.seq_lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        return cache

    def _flat_index(self, b: int, start: int, n: int) -> torch.Tensor:
        t = torch.arange(start, start + n, device=self.device)
        pages = self.block_table[b].to(torch.int64)[t // PAGE_SIZE]
        return pages * PAGE_SIZE + (t % PAGE_SIZE)

    def write_rows(self, b: int, start: int, rows: torch.Tensor) -> None:
        """Store rows [n, 576] as request b's logical rows start..start+n-1 (set-up helper)."""
        flat = self.pages.view(-1, ROW)
        flat[self._flat_index(b, start, rows.shape[0])] = rows.to(device=self.device, dtype=torch.bfloat16)

    def read_rows(self, b: int, start: int, n: int) -> torch.Tensor:
        """Request b's logical rows start..start+n-1, [n, 576] bf16."""
        return self.pages.view(-1, ROW)[self._flat_index(b, start, n)]

    def advance(self, n: int = 1) -> None:
        """Count the rows appended by the last step (the reference's caller advances pos)."""
        self.seq_lens += n


class PagedLatentCache8(PagedLatentCache):
    """The same cache held in 8 bits: half the bytes per row.

    `pages` is uint8 [n_pages, 36864]: per page the latent part [64][512], then the rotary part
    [64][64], both e4m3. `scales` is int8 [n_pages, 4, 2]: per block of 16 rows the exponents of the
    power-of-two scales of the two parts, value = e4m3 * 2**exponent. An exponent is the smallest
    one, at least -64, that brings the block's largest finite magnitude to at most 448; a row that joins a
    started block may raise it, and the block's earlier rows are then held anew under it (a row that is
    stored again in its place, as by a repeated step, leaves the raised one).
    Infinities and NaN are held as NaN. Rows are stored by the decode step
    (MlaDecodeAttention) and by rows_to_pages; both take this class as they take
    PagedLatentCache. Pages that two requests share (PagePool.fork) must not be appended to.
    """

    def __init__(self, n_pages: int, batch: int, max_blocks: int, device: torch.device | str = "cuda",
                 zero: bool = True):
        if n_pages <= 0 or batch <= 0 or max_blocks <= 0:
            raise ValueError("n_pages, batch and max_blocks must be positive")
        alloc = torch.zeros if zero else torch.empty
        self.pages = alloc(n_pages, PAGE8_BYTES, dtype=torch.uint8, device=device)
        self.scales = alloc(n_pages, PAGE_SIZE // SCALE_BLOCK, 2, dtype=torch.int8, device=device)
        self.block_table = torch.zeros(batch, max_blocks, dtype=torch.int32, device=device)
        self.seq_lens = torch.zeros(batch, dtype=torch.int32, device=device)

    @classmethod
    def from_tensors(cls, pages: torch.Tensor, scales: torch.Tensor, block_table: torch.Tensor,
                     seq_lens: torch.Tensor) -> "PagedLatentCache8":
        """A cache over tensors that the caller keeps; nothing is copied."""
        _check_tensor("pages", pages, torch.uint8, (None, PAGE8_BYTES))
        _check_tensor("scales", scales, torch.int8, (pages.shape[0], PAGE_SIZE // SCALE_BLOCK, 2))
        if scales.device != pages.device:
            raise ValueError("pages and scales must be on one device")
        self = cls._adopt(pages, block_table, seq_lens)
        self.scales = scales
        return self

    def write_rows(self, b: int, start: int, rows: torch.Tensor) -> None:
        """Store rows [n, 576] as request b's logical rows start..start+n-1 (on the GPU only:
        the rounding and the blocks' scales are the library's). Waits for the device; rows without a place in
        the block table or a page of the pool raise MlaError."""
        from .handoff import rows_to_pages
        from .native import MlaError
        one = PagedLatentCache8.from_tensors(self.pages, self.scales, self.block_table[b:b + 1],
                                             self.seq_lens[b:b + 1])
        word = torch.zeros(1, dtype=torch.int32, device=self.device)
        rows_to_pages(one, rows.to(device=self.device, dtype=torch.bfloat16).contiguous(), [0, rows.shape[0]], [start],
                      error_word=word)
        if int(word):
            raise MlaError(int(word), "device (write_rows)")

    def read_rows(self, b: int, start: int, n: int) -> torch.Tensor:
        """The values of request b's logical rows start..start+n-1, [n, 576] f32."""
        flat = self._flat_index(b, start, n)
        page, slot = flat // PAGE_SIZE, flat % PAGE_SIZE
        e4m3 = self.pages.view(torch.float8_e4m3fn)
        parts = (e4m3[:, :PAGE_SIZE * KV_LORA].unflatten(1, (PAGE_SIZE, KV_LORA)),
                 e4m3[:, PAGE_SIZE * KV_LORA:].unflatten(1, (PAGE_SIZE, QK_ROPE)))
        scale = torch.exp2(self.scales[page, slot // SCALE_BLOCK].float())
        return torch.cat([part.view(torch.uint8)[page, slot].view(torch.float8_e4m3fn).float() * scale[:, k:k + 1]
                          for k, part in enumerate(parts)], dim=1)
