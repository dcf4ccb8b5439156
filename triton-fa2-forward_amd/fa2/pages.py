"""The pages of a serving step on AMD MI355X (gfx950): which pages of a cache are free, on the GPU.

A PagePool holds the numbers of the pages that no sequence has. pages_extend() takes pages for a step's new tokens from
it, enters them into the sequences' block table and gives what the step's other operators are called with (row starts,
lengths, positions, slots); pages_release() gives pages back. Both work from lengths on the device: nothing is
copied to the host. They change the block table and the pool's stack in place and return new lengths and a new count: go on
with the pool that a call returns, the one it was given is used up. A captured graph copies the new lengths and count to
where its next replay reads them. The HIP kernels are csrc/serve_pages.hip
behind include/fa2_fwd.h.
"""

from typing import NamedTuple

import torch

from . import _lib
from .packed import _index


class PagePool(NamedTuple):
    """free: int32 [pages] on the GPU, dense, whose first count entries are the free pages, a stack with its top at the end;
    count: int32 [1]."""
    free: torch.Tensor
    count: torch.Tensor

    @classmethod
    def full(cls, pages, device="cuda"):
        """All of a cache's pages, free."""
        return cls(torch.arange(pages, dtype=torch.int32, device=device),
                   torch.full((1,), pages, dtype=torch.int32, device=device))


class Step(NamedTuple):
    """What pages_extend gives: the pool with fewer pages, cu_seqlens int32 [S + 1] and seqlens int32 [S] as cache_write and
    attention_paged take them, positions int32 [n_tokens] of the new tokens in their sequences (as rotary takes them),
    and slots int64 [n_tokens], page * page_size + the place in the page. Both are -1 for rows of no sequence, a slot
    also for a token without a page."""
    pool: PagePool
    cu_seqlens: torch.Tensor
    seqlens: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor


def _check(pool, block_table):
    """The pool's and the table's types and places; the device."""
    device = pool.free.device
    assert pool.free.dim() == 1 and pool.free.dtype == torch.int32, "a pool's free is int32 [pages]"
    assert pool.count.dtype == torch.int32 and pool.count.numel() == 1, "a pool's count is int32 [1]"
    assert block_table.dim() == 2 and block_table.dtype == torch.int32, "block_table is int32 [S, pages]"
    if not (pool.free.is_cuda and pool.count.device == device and block_table.device == device):
        raise RuntimeError(f"the pool and block_table must be on one GPU, got {device}, {pool.count.device} and "
                           f"{block_table.device}")
    S, P = block_table.shape
    if not pool.free.is_contiguous():
        raise ValueError("a pool's free is written in place: it must be dense")
    # (written in place, so never copied)
    if (P > 1 and block_table.stride(1) != 1) or (S > 1 and P > 0 and block_table.stride(0) < P):
        raise ValueError(f"block_table must have a unit stride in its rows and no shared elements, got {block_table.stride()}")
    return device


def pages_extend(pool, block_table, seqlens, new_tokens, page_size, n_tokens):
    """Pages for the new tokens of a step: a Step.

    block_table: int32 [S, pages] (S up to 2^20), whose rows hold the pages of seqlens[s] tokens in order; the new ones are entered
    behind them, in place. seqlens: int32 [S], tokens in the cache; new_tokens: int32 [S], to be added to each (negative
    numbers count as 0). page_size: a power of two up to 2^20. n_tokens: rows of positions and slots (the sum of new_tokens, which is
    not copied to the host to find out; or more).
    The pages are the topmost of the pool, in the order of the sequences. Where too few are free the last tokens get
    none: their entries are -1, cache_write leaves them out, and rows that see them are NaN in attention_paged. Tokens past the
    end of their row of the table need no page.
    """
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.pages_extend(*pool, block_table, seqlens, new_tokens, page_size, n_tokens)
        if result is not None:
            return Step(PagePool(pool.free, result[0]), *result[1:])
    device = _check(pool, block_table)
    S = block_table.shape[0]
    assert seqlens.shape == new_tokens.shape == (S,), "seqlens and new_tokens hold an entry per row of block_table"
    if page_size < 1 or page_size & (page_size - 1) or page_size > 1 << 20:
        raise ValueError(f"page_size must be a power of two up to 2^20, got {page_size}")
    if n_tokens < 0:
        raise ValueError(f"n_tokens must not be negative, got {n_tokens}")
    lens, new = _index(seqlens, "seqlens", device), _index(new_tokens, "new_tokens", device)

    def empty(n, dtype=torch.int32):
        return torch.empty(n, dtype=dtype, device=device)

    count, cu, after, positions, slots = empty(1), empty(S + 1), empty(S), empty(n_tokens), empty(n_tokens, torch.int64)
    if S == 0:
        count.copy_(pool.count.view(1))
        for t, x in ((cu, 0), (positions, -1), (slots, -1)):
            t.fill_(x)
    else:
        with torch.cuda.device(device):
            _lib.pages_extend(pool.free, pool.count, count, block_table, page_size, lens, new, after, cu, positions, slots,
                              torch.cuda.current_stream(device).cuda_stream)
    return Step(PagePool(pool.free, count), cu, after, positions, slots)


def pages_release(pool, block_table, first, last):
    """The pool with entries first[s] .. last[s] - 1 of every sequence's row of block_table given back to it (int32 [S] each;
    empty ranges for sequences that keep theirs): 0 .. ceil(length / page_size) for a sequence that has ended, from the
    shared pages' number on where it shares a prefix, the pages that have left a window.

    They go on top of the stack in the order of the sequences and entries; entries that are no page of the pool's are left
    out. The table is left as it is. A page that is given back twice is free twice: the caller's to avoid.
    """
    if _lib.native is not None:  # the common call, made natively; None: not one of those
        result = _lib.native.pages_release(*pool, block_table, first, last)
        if result is not None:
            return PagePool(pool.free, result)
    device = _check(pool, block_table)
    S = block_table.shape[0]
    assert first.shape == last.shape == (S,), "first and last hold an entry per row of block_table"
    first, last = _index(first, "first", device), _index(last, "last", device)
    if S == 0:
        return PagePool(pool.free, pool.count.clone())
    count, counts = (torch.empty(n, dtype=torch.int32, device=device) for n in (1, S + 1))
    with torch.cuda.device(device):
        _lib.pages_release(pool.free, pool.count, count, block_table, first, last, counts,
                           torch.cuda.current_stream(device).cuda_stream)
    return PagePool(pool.free, count)
