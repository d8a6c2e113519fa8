"""
A paged cache: K and V rows of any number of sequences in pages of a common pool, for batches whose sequences have lengths of
their own and come and go. The reference's caches are contiguous, one row of slots per batch element; this is for a serving
loop around the same layers.

The pool is two tensors ``(num_pages, n_query_groups, page_size, row)``: bfloat16 or float16 rows, or uint8 rows of 8-bit or
packed 4-bit codes with their ``QuantState`` of ``(num_pages, n_query_groups, page_size)`` arrays (the codes, scales and zero
points of ``RowQuantizer``, one block per row). Which pages a sequence has is a row of an int32 block table: token ``t`` of
sequence ``b`` lies in page ``block_table[b, t // page_size]`` at place ``t % page_size``; its slot is ``page * page_size + place``.
Handing out pages is the caller's: any order, pages shared between sequences (a common prompt) included, as long as no slot is
written twice in one call.

A layer's step for one new token a sequence is ``longctx.ops.rotary_``, ``paged_write``, ``attention.ops.paged_decode``. A later
chunk of a prompt attends over ``paged_read`` rows with ``attention.ops.prefill_core``, one sequence a call: ``prefill_core`` has one
position for its whole batch, and the zero rows that ``paged_read`` puts behind shorter sequences are keys like any others to it. Tables, lengths, slots and positions
stay on the device and are read by the kernels alone, so the calls can be captured into a graph and replayed with others in
their place (graphs that share a memory pool in the order of their capture, as torch asks for: a later one's tensors may lie where
an earlier one had its workspace). There is no CPU path.
"""
from typing import Optional, Tuple

import torch

from .. import _lib
from ..attention import ops

PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)


def paged_write(key: torch.Tensor, value: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, slots: torch.Tensor,
                quant: Optional[ops.QuantState] = None) -> None:
    """Write rows ``key`` / ``value`` (tokens, n_query_groups, head_size), views with contiguous rows, to the slots ``slots`` (tokens,)
    int64. Rows of a negative slot, or of one behind the pool's last, are dropped. With ``quant`` (pages of codes) the rows are quantised
    on the way in, bit for bit as ``RowQuantizer`` does, and ``quant`` gets their scales and zero points."""
    _lib.host().paged_write(key, value, key_pages, value_pages, slots, quant)


def paged_read(key_pages: torch.Tensor, value_pages: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, length: int, head_size: Optional[int] = None,
               dtype: Optional[torch.dtype] = None, quant: Optional[ops.QuantState] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The first ``length`` rows of every sequence, ``(key, value)`` of shape (sequences, n_query_groups, length, head_size): rows behind
    ``lens`` (int32, on the device) are zero (an attention that takes them for keys has to mask them). Pages of codes need ``quant``, and ``head_size`` and ``dtype`` of the rows
    they stand for; of plain pages both are known."""
    if quant is None:
        head_size = key_pages.shape[-1] if head_size is None else head_size
        dtype = key_pages.dtype if dtype is None else dtype
    elif head_size is None or dtype is None:
        raise ValueError("pages of codes: head_size and dtype of their rows must be given")
    return _lib.host().paged_read(key_pages, value_pages, block_table, lens, length, head_size, dtype, quant)


class PagedKVCacheBuffers:
    """The pool of one layer and its operators. ``num_bits``: None for plain rows, 8 or 4 for codes. A new pool holds zeros."""

    def __init__(self, num_pages: int, page_size: int, n_query_groups: int, head_size: int, dtype: torch.dtype = torch.bfloat16, num_bits: Optional[int] = None,
                 device: Optional[torch.device] = None):
        if num_pages < 1 or n_query_groups < 1:
            raise ValueError(f"num_pages = {num_pages}, n_query_groups = {n_query_groups}: must be positive")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"page_size = {page_size}, must be one of {PAGE_SIZES}")
        if head_size not in ops.ALLOWED_HEAD_SIZES:
            raise NotImplementedError(f"head_size = {head_size} not in {ops.ALLOWED_HEAD_SIZES}")
        if dtype not in ops.ALLOWED_DTYPES:
            raise NotImplementedError(f"dtype = {dtype} not in {ops.ALLOWED_DTYPES}")
        if num_bits not in (None, 8, 4):
            raise ValueError(f"num_bits = {num_bits}, must be None, 8 or 4")
        self.device = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        if self.device.type != "cuda":
            raise RuntimeError("PagedKVCacheBuffers lives on a ROCm device only")
        self.num_pages, self.page_size, self.n_query_groups, self.head_size = num_pages, page_size, n_query_groups, head_size
        self.dtype, self.num_bits = dtype, num_bits
        rows = (num_pages, n_query_groups, page_size)
        kept = dtype if num_bits is None else torch.uint8
        self.k, self.v = (torch.zeros(*rows, head_size if num_bits != 4 else head_size // 2, dtype=kept, device=self.device) for _ in range(2))
        self.quant = None
        if num_bits is not None:
            self.quant = ops.QuantState(*(torch.zeros(rows, dtype=t, device=self.device) for t in (torch.float32, torch.int32) * 2))

    def slots(self, block_table: torch.Tensor, positions: torch.Tensor) -> torch.Tensor:
        """Slots of the tokens at ``positions`` (sequences, tokens) of the sequences of ``block_table``, flat int64; -1 for a negative position and
        for one behind the table. Once per step: the layers share them."""
        if block_table.dim() != 2 or block_table.shape[1] == 0:
            raise ValueError(f"block_table must be (sequences, pages), got shape {tuple(block_table.shape)}")
        if positions.dim() != 2 or positions.shape[0] != block_table.shape[0]:
            raise ValueError(f"positions must be ({block_table.shape[0]}, tokens), got shape {tuple(positions.shape)}")
        pos = positions.long()
        page = torch.div(pos.clamp(min=0), self.page_size, rounding_mode="floor")
        there = (pos >= 0) & (page < block_table.shape[1])
        at = block_table.long().gather(1, page.clamp(max=block_table.shape[1] - 1))
        return torch.where(there & (at >= 0), at * self.page_size + pos % self.page_size, -1).flatten()

    def write(self, key: torch.Tensor, value: torch.Tensor, slots: torch.Tensor) -> None:
        """See :func:`paged_write`."""
        paged_write(key, value, self.k, self.v, slots, self.quant)

    def read(self, block_table: torch.Tensor, lens: torch.Tensor, length: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """See :func:`paged_read`."""
        return paged_read(self.k, self.v, block_table, lens, length, self.head_size, self.dtype, self.quant)

    def decode(self, query: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, scale: Optional[float] = None,
               return_lse: bool = False) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """See :func:`keys_values_amd.attention.ops.paged_decode`."""
        return ops.paged_decode(query, self.k, self.v, block_table, lens, ops.default_scale(self.head_size) if scale is None else scale, return_lse, self.quant)

    def size_estimate(self) -> int:
        """Bits that the pool takes."""
        state = self.quant or ()
        return sum(8 * t.numel() * t.element_size() for t in (self.k, self.v, *state))
