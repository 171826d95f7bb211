"""Block tables and slot maps of one serving step, built on the GPU.

A step adds query_lens[b] rows to request b, which has seq_lens[b] rows in the
paged caches.  `step_layout` hands out the new pages, extends the block tables
in place and says for every new row where it goes and what it sees: the slots
that `index_cache_append` and `latent_cache_append` write to, the positions that
`apply_rope` turns to, and the request and visible length of each query token
that `shared_prefix_attention` takes.  Nothing is read back to the host, so a
captured step follows the lengths.  The reference has no counterpart (its caller
passes finished tables and indices, solution/triton/kernel.py:184-332).
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _lib


class StepLayout(NamedTuple):
    """The new rows of a step in request order, [num_tokens] int32 each (rows
    behind the last request: slot -1, position 0, request 0, length 0)."""
    slots: torch.Tensor          # flat cache slot page*64 + row
    positions: torch.Tensor      # prefix_len + row in the request
    token_request: torch.Tensor  # request (row of the block table)
    token_lens: torch.Tensor     # own rows the token sees, itself included
    pages_used: torch.Tensor     # [1]: free pages taken


def step_layout(seq_lens, query_lens, block_table, free_pages, num_tokens, *, prefix_len=None, out=None,
                device_error=None) -> StepLayout:
    """Lay out a step: pages for the new rows, and where each new row goes.

    seq_lens, query_lens [B]: rows in the cache and rows that the step adds;
    block_table [B, W] int32, extended IN PLACE with pages from the front of
    free_pages [F] (entries of pages that the requests have already stay);
    num_tokens: rows of the outputs, at least sum(query_lens) or a fixed
    capacity for a captured graph; prefix_len: optional [1] int32 tensor, rows
    of a shared prefix in front of every request (added to the positions only).
    out: a StepLayout of [num_tokens] int32 contiguous tensors to write into.
    device_error: optional int32 tensor that collects DSA_DEVERR_* bits (4: out
    of pages, table columns or rows; 1: a negative entry of an older page).
    Calling it again with the same lengths and free pages gives the same result.
    """
    seq_lens, query_lens = _lib.int32(seq_lens, "seq_lens"), _lib.int32(query_lens, "query_lens")
    free_pages = _lib.int32(free_pages, "free_pages")
    assert seq_lens.dim() == 1 and query_lens.dim() == 1 and free_pages.dim() == 1
    num_tokens = int(num_tokens)
    batch, width = block_table.shape
    assert seq_lens.shape[0] == batch and query_lens.shape[0] == batch and num_tokens >= 0
    assert block_table.dtype == torch.int32 and (width <= 1 or block_table.stride(1) == 1), \
        "block_table must be int32 with contiguous rows"
    assert prefix_len is None or isinstance(prefix_len, torch.Tensor), "prefix_len must be one int32 on the GPU"
    index = _lib.same_device(block_table, seq_lens, query_lens, free_pages, prefix_len, device_error)
    if prefix_len is not None:
        assert prefix_len.dtype == torch.int32 and prefix_len.numel() == 1, "prefix_len must be one int32"
    if device_error is not None:
        assert device_error.dtype == torch.int32 and device_error.numel() >= 1, "device_error must be int32"
    if out is None:
        buf = block_table.new_empty(4 * num_tokens + 1)
        out = StepLayout(*buf.split_with_sizes((num_tokens, num_tokens, num_tokens, num_tokens, 1)))
        at = buf.data_ptr()
        outs = tuple(at + 4 * num_tokens * i for i in range(5))
    else:
        assert _lib.same_device(*out) == index, "out: on the inputs' device"
        for t, n in zip(out, (num_tokens,) * 4 + (1,)):
            assert t.dtype == torch.int32 and t.numel() == n and t.is_contiguous(), "out: int32, contiguous"
        outs = tuple(t.data_ptr() for t in out)
    _lib.call_on(index, "dsa_step_layout", seq_lens.data_ptr(), query_lens.data_ptr(), batch,
                 block_table.data_ptr(), block_table.stride(0), width, free_pages.data_ptr(),
                 free_pages.shape[0], prefix_len.data_ptr() if prefix_len is not None else None, num_tokens,
                 *outs, device_error.data_ptr() if device_error is not None else None)
    return out
