"""Dense MLA attention over the paged latent cache for a batch that shares a
long prefix: the prefix's rows are read once for all the tokens.

Stands beside `kernel()`, which attends to 2048 selected rows of the same cache:
this one attends to every row of the shared prefix and of the request's own
pages (short contexts, exact attention behind a common system prompt or
document).  The reference has no counterpart.
"""
from __future__ import annotations

import ctypes
import threading

import torch

from . import _lib
from .kernel import HEAD_DIM_CKV, HEAD_DIM_KPE, NUM_HEADS, PAGE_SIZE

_workspaces: dict[int, torch.Tensor] = {}  # per device: the word that collects device errors
_lock = threading.Lock()
_size_cache: dict[tuple, int] = {}


def prefix_workspace_size(num_tokens: int, heads: int = NUM_HEADS, device=None) -> int:
    """Bytes of the workspace that a call of this shape needs on `device` (an
    index or torch.device; default: the current device)."""
    index = _index(device)
    nbytes = _size_cache.get((index, num_tokens, heads))
    if nbytes is None:
        n = ctypes.c_size_t(0)
        with torch.cuda.device(index):
            _lib.call("dsa_shared_prefix_attention_workspace_size", num_tokens, heads, ctypes.byref(n))
        nbytes = _size_cache[(index, num_tokens, heads)] = n.value
    return nbytes


def _index(device) -> int:
    if isinstance(device, int):
        return device
    index = torch.device(device).index if device is not None else None
    return index if index is not None else torch.cuda.current_device()


def _error_word(index: int) -> torch.Tensor:
    """The device's error word for calls without a workspace of their own.  It
    stays, since a captured graph may hold its address."""
    word = _workspaces.get(index)
    if word is None:
        with _lock, torch.cuda.device(index):
            word = _workspaces.get(index)
            if word is None:
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("the error word cannot be made during stream capture: make one call on the "
                                       "device before the capture, or pass workspace=")
                word = torch.zeros(64, dtype=torch.int32, device=f"cuda:{index}")
                torch.cuda.current_stream().synchronize()  # zero before a call on another stream can set it
                _workspaces[index] = word
    return word


def shared_prefix_attention(q_nope, q_pe, ckv_cache, kpe_cache, prefix_pages, prefix_len, block_table, token_lens,
                            sm_scale, *, token_request=None, output=None, lse=None, workspace=None):
    """Attention of every token over the shared prefix and its request's own rows;
    returns (output [T,H,512] bf16, lse [T,H] fp32 base 2).

    q_nope [T,H,512], q_pe [T,H,64], ckv_cache [P,64,512], kpe_cache [P,64,64]
    bf16, H a multiple of 16.  prefix_pages [n] int32 and prefix_len (an int or
    a [1] int32 CUDA tensor, at most 64 n): the prefix, which may end inside a
    page.  block_table [B,W] int32: own pages of each request, own row 0 first.
    token_lens [T] int32: own rows that token t sees (0: only the prefix).
    token_request [T] int32: block-table row of token t (default: row t).
    `step_layout` makes token_lens and token_request.  A token that sees no row
    gets output 0 and lse -inf.  Rows past a length are never read.

    output/lse write into existing tensors.  Plan and partials take about 40 MB
    of torch's memory for the time of the call, so calls on several streams or
    threads and captured graphs do not meet (the first call on a device must not
    be a captured one).  workspace: a zeroed, 256-byte aligned uint8 CUDA tensor of
    prefix_workspace_size(T, H) bytes to use instead; calls that share it must not
    overlap.  Errors found on the device (page ids or requests outside their
    range: those rows are skipped) are read by `read_prefix_error`, those of calls
    with a workspace of their own in its first int32.
    """
    tokens, heads, dim = q_nope.shape
    num_pages = ckv_cache.shape[0]
    assert heads % NUM_HEADS == 0 and heads > 0, "heads must be a multiple of 16"
    assert dim == HEAD_DIM_CKV and q_pe.shape == (tokens, heads, HEAD_DIM_KPE)
    assert ckv_cache.shape == (num_pages, PAGE_SIZE, HEAD_DIM_CKV)
    assert kpe_cache.shape == (num_pages, PAGE_SIZE, HEAD_DIM_KPE)
    length = prefix_len if isinstance(prefix_len, torch.Tensor) else None
    index = _lib.same_device(q_nope, q_pe, ckv_cache, kpe_cache, prefix_pages, length, block_table, token_lens,
                             token_request, output, lse, workspace)
    bf16 = torch.bfloat16
    assert q_nope.dtype == bf16 and q_pe.dtype == bf16 and ckv_cache.dtype == bf16 and kpe_cache.dtype == bf16, \
        "queries and caches must be bfloat16"
    requests, width = block_table.shape
    assert token_lens.shape == (tokens,), "token_lens must be [tokens]"
    assert prefix_pages.dim() == 1, "prefix_pages must be one list of pages"
    prefix_pages, token_lens = _lib.int32(prefix_pages, "prefix_pages"), _lib.int32(token_lens, "token_lens")
    if length is not None:
        assert length.numel() == 1 and length.dtype == torch.int32, "prefix_len must be an int or one int32"
        bound = prefix_pages.shape[0] * PAGE_SIZE
    else:
        bound = int(prefix_len)
        assert 0 <= bound <= prefix_pages.shape[0] * PAGE_SIZE, "prefix_len does not fit prefix_pages"
    if token_request is not None:
        assert token_request.shape == (tokens,), "token_request must be [tokens]"
        token_request = _lib.int32(token_request, "token_request")
    else:
        assert requests >= tokens, "without token_request the block table needs a row for every token"
    if output is None:
        output = torch.empty_like(q_nope, memory_format=torch.contiguous_format)
        out_token, out_head = heads * HEAD_DIM_CKV, HEAD_DIM_CKV
    else:
        assert output.shape == (tokens, heads, HEAD_DIM_CKV) and output.dtype == bf16
        out_token, out_head, last = output.stride()
        assert last == 1 and out_token % 8 == 0 and out_head % 8 == 0 and output.data_ptr() % 16 == 0, \
            "output rows must be contiguous and 16-byte aligned"
        assert (out_token > 0 or tokens <= 1) and out_head > 0, "output is an expanded tensor"
    if lse is None:
        lse = q_nope.new_empty((tokens, heads), dtype=torch.float32)
        lse_token, lse_head = heads, 1
    else:
        assert lse.shape == (tokens, heads) and lse.dtype == torch.float32
        lse_token, lse_head = lse.stride()
        assert (lse_token > 0 or tokens <= 1) and lse_head > 0, "lse is an expanded tensor"
    if tokens == 0:
        return output, lse
    assert num_pages > 0, "the cache has no pages"
    if block_table.dtype != torch.int32 or (width > 1 and block_table.stride(1) != 1):
        block_table = _lib.int32(block_table, "block_table")
    ckv_strides, kpe_strides = _tile_strides(ckv_cache), _tile_strides(kpe_cache)
    assert ckv_strides and kpe_strides, "cache rows must be contiguous, 16-byte aligned and apart"
    (c_page, c_row), (e_page, e_row) = ckv_strides, kpe_strides
    q_nope, qn_token, qn_head = _tiled(q_nope)
    q_pe, qp_token, qp_head = _tiled(q_pe)
    args = (q_nope.data_ptr(), qn_token, qn_head, q_pe.data_ptr(), qp_token, qp_head, ckv_cache.data_ptr(), c_page, c_row,
            kpe_cache.data_ptr(), e_page, e_row, prefix_pages.data_ptr(), bound,
            length.data_ptr() if length is not None else None, block_table.data_ptr(), block_table.stride(0), requests,
            width, token_request.data_ptr() if token_request is not None else None, token_lens.data_ptr(), tokens, heads,
            num_pages, sm_scale, output.data_ptr(), out_token, out_head, lse.data_ptr(), lse_token, lse_head)
    if workspace is None:
        _lib.call_with_scratch(index, "dsa_shared_prefix_attention_scratch", prefix_workspace_size(tokens, heads, index),
                               _error_word(index).data_ptr(), *args)
    elif workspace.dtype == torch.uint8 and workspace.is_contiguous():
        _lib.call_on(index, "dsa_shared_prefix_attention", *args, workspace.data_ptr(), workspace.numel())
    else:
        raise ValueError("workspace must be a contiguous uint8 tensor on the inputs' device")
    return output, lse


def _tile_strides(t: torch.Tensor):
    """(outer, inner stride) of t [A, B, width] if the TMA can read its rows where
    they are, else None."""
    if t.is_contiguous() and t.data_ptr() % 16 == 0:
        _, rows, width = t.shape
        return rows * width, width
    outer, inner, last = t.stride()
    if last == 1 and inner % 8 == 0 and inner >= t.shape[2] and t.data_ptr() % 16 == 0 and (
            t.shape[0] == 1 or (outer >= inner and outer % 8 == 0)):
        return outer, inner
    return None


def _tiled(t: torch.Tensor):
    """(t, outer, inner stride), of a contiguous copy if the TMA cannot read t itself."""
    strides = _tile_strides(t)
    if strides is None:
        t = t.clone(memory_format=torch.contiguous_format)
        strides = t.stride()[:2]
    return t, *strides


def read_prefix_error(device=None, clear=True) -> int:
    """Synchronise the current stream and return the DSA_DEVERR_* bits raised by
    shared_prefix_attention calls without a workspace of their own."""
    index = _index(device)
    word = _workspaces.get(index)
    if word is None:
        return 0
    bits = ctypes.c_int(0)
    with torch.cuda.device(index):
        _lib.call("dsa_read_device_error", word.data_ptr(), int(clear), ctypes.byref(bits),
                  torch.cuda.current_stream().cuda_stream)
    return bits.value
