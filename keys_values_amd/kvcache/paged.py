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

Long sequences need not be read whole for a token. With the lowest and the highest of each page's keys at hand (``paged_bounds``, twice a row's bytes a page),
``attention.ops.paged_select`` finds the pages that can matter to a query, and ``attention.ops.paged_decode_chosen`` attends to those. A layer's step is
then ``paged_append`` (rotation and write in one launch), ``paged_bounds`` of the page written to (``tokens=1``), ``paged_select``, ``paged_decode_chosen``; a pool made
with ``bounds=True`` has them as methods. Several new tokens of a sequence: one append, one ``paged_bounds`` with the sequence's new length and ``tokens`` their number, then the
row of the table once a token, with the token's own length, in the other two.
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


def paged_append(qkv: torch.Tensor, n_head: int, n_query_groups: int, head_size: int, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float,
                 cos: torch.Tensor, sin: torch.Tensor, positions: torch.Tensor, key_pages: torch.Tensor, value_pages: torch.Tensor, slots: torch.Tensor,
                 quant: Optional[ops.QuantState] = None, interleaved: bool = False) -> None:
    """What a layer does with the projections of new tokens, in one launch: ``longctx.ops.rotary_`` of qkv's query heads, in place, and of its key heads on their
    way to the slots ``slots`` (int64, one a token), to which its value heads go too, as :func:`paged_write` stores them. Bit for bit what the two calls give, but
    that the key heads of qkv (and its value heads) stay as they are. Tokens of a negative position, or of one behind the tables, are padding: nothing of them is changed or
    stored, whatever their slot. Those with a position and without a slot have their queries turned."""
    _lib.host().paged_append(qkv, n_head, n_query_groups, head_size, q_weight, k_weight, eps, cos, sin, positions, key_pages, value_pages, slots, quant, interleaved)


def paged_bounds(key_pages: torch.Tensor, bounds: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, tokens: Optional[int] = None,
                 quant: Optional[ops.QuantState] = None) -> None:
    """Bring ``bounds`` (num_pages, n_query_groups, 2, head_size), of the rows' type, in line with the pages that hold the last ``tokens`` of the first
    ``lens`` tokens of every sequence (None: all of them): the lowest [.., 0, :] and the highest [.., 1, :] of the page's keys among these, value by value, of codes as
    :func:`paged_read` gives their rows (rounded to nearest, so that the rows that attention takes may lie half a step outside). A NaN among the keys makes a bound NaN.
    ``tokens`` is the most that any sequence has got since the last call: pages of sequences that got fewer are looked at again, which changes nothing. Sequences that share a
    page should share it whole, or have as many tokens in it: where they have not, its bounds are one's or parts of each. A sequence with several new tokens is given once, with
    all of them counted, also where ``attention.ops.paged_select`` is then given its row of the table once a token: a page's bounds hold for any of its tokens."""
    _lib.host().paged_bounds(key_pages, bounds, block_table, lens, tokens, quant)


class PagedKVCacheBuffers:
    """The pool of one layer and its operators. ``num_bits``: None for plain rows, 8 or 4 for codes; ``bounds``: whether it keeps the bounds of its pages' keys, which
    :meth:`select` goes by. A new pool holds zeros."""

    def __init__(self, num_pages: int, page_size: int, n_query_groups: int, head_size: int, dtype: torch.dtype = torch.bfloat16, num_bits: Optional[int] = None,
                 device: Optional[torch.device] = None, bounds: bool = False):
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

        self.bounds = torch.zeros(num_pages, n_query_groups, 2, head_size, dtype=dtype, device=self.device) if bounds else None

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

    def append(self, qkv: torch.Tensor, n_head: int, q_weight: Optional[torch.Tensor], k_weight: Optional[torch.Tensor], eps: float, cos: torch.Tensor, sin: torch.Tensor,
               positions: torch.Tensor, slots: torch.Tensor, interleaved: bool = False) -> None:
        """See :func:`paged_append`."""
        paged_append(qkv, n_head, self.n_query_groups, self.head_size, q_weight, k_weight, eps, cos, sin, positions, self.k, self.v, slots, self.quant, interleaved)

    def _bounds(self) -> torch.Tensor:
        if self.bounds is None:
            raise ValueError("the pool keeps no bounds: make it with bounds=True")
        return self.bounds

    def update_bounds(self, block_table: torch.Tensor, lens: torch.Tensor, tokens: Optional[int] = None) -> None:
        """See :func:`paged_bounds`."""
        paged_bounds(self.k, self._bounds(), block_table, lens, tokens, self.quant)

    def select(self, query: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, count: int, first: int = 1, last: int = 1) -> torch.Tensor:
        """See :func:`keys_values_amd.attention.ops.paged_select`."""
        return ops.paged_select(query, self._bounds(), block_table, lens, self.page_size, count, first, last)

    def read(self, block_table: torch.Tensor, lens: torch.Tensor, length: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """See :func:`paged_read`."""
        return paged_read(self.k, self.v, block_table, lens, length, self.head_size, self.dtype, self.quant)

    def decode(self, query: torch.Tensor, block_table: torch.Tensor, lens: torch.Tensor, scale: Optional[float] = None, return_lse: bool = False,
               chosen: Optional[torch.Tensor] = None) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
        """See :func:`keys_values_amd.attention.ops.paged_decode`; with ``chosen`` pages :func:`keys_values_amd.attention.ops.paged_decode_chosen`."""
        scale = ops.default_scale(self.head_size) if scale is None else scale
        if chosen is not None:
            return ops.paged_decode_chosen(query, self.k, self.v, block_table, lens, chosen, scale, return_lse, self.quant)
        return ops.paged_decode(query, self.k, self.v, block_table, lens, scale, return_lse, self.quant)

    def size_estimate(self) -> int:
        """Bits that the pool takes."""
        more = (*(self.quant or ()), *(() if self.bounds is None else (self.bounds,)))
        return sum(8 * t.numel() * t.element_size() for t in (self.k, self.v, *more))
