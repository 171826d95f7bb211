"""ctypes binding of libdsa_b200.so (the C ABI declared in include/dsa_b200.h).

The library is built in-tree by flashinfer_repo_b200.build.  There is no
fallback: if the library is missing or a call fails, an exception is raised.
"""
from __future__ import annotations

import ctypes
import os

import torch

from . import build as _build

_lib = None

I64 = ctypes.c_int64
P = ctypes.c_void_p
SZ = ctypes.c_size_t
F32 = ctypes.c_float
INT = ctypes.c_int

class Options(ctypes.Structure):
    """struct dsa_options (include/dsa_b200.h)."""
    _fields_ = [("attention_kernel", ctypes.c_int), ("attention_stages", ctypes.c_int),
                ("attention_ctas", ctypes.c_int), ("attention_min_tiles", ctypes.c_int),
                ("attention_grids", ctypes.c_int), ("merge_pdl", ctypes.c_int),
                ("indexer_tiles_per_cta", ctypes.c_int), ("attention_cluster", ctypes.c_int)]


# name -> argtypes; every function returns int (dsa_status) except the message.
SIGNATURES = {
    "dsa_sparse_attention_workspace_size": [I64, I64, I64, ctypes.POINTER(SZ)],
    "dsa_set_options": [ctypes.POINTER(Options)],
    "dsa_get_options": [ctypes.POINTER(Options)],
    "dsa_sparse_attention": [P, I64, I64, P, I64, I64, P, I64, I64, P, I64, I64, P, I64,
                             I64, I64, I64, I64, I64, F32, P, I64, I64, P, I64, I64, P, SZ, P],
    "dsa_sparse_attention_noalloc": [P, I64, I64, P, I64, I64, P, I64, I64, P, I64, I64, P, I64,
                                     I64, I64, I64, I64, I64, F32, P, I64, I64, P, I64, I64, P],
    "dsa_sparse_attention_noalloc_read_error": [INT, ctypes.POINTER(INT), P],
    "dsa_sparse_attention_scatter": [P, I64, I64, P, I64, I64, P, I64, I64, P, I64, I64, P, I64,
                                     I64, I64, I64, I64, I64, F32, P, I64, I64, P, I64, I64, INT,
                                     P, SZ, P],
    "dsa_sparse_attention_scatter_sync": [P, I64, I64, P, I64, I64, P, I64, I64, P, I64, I64, P, I64,
                                          I64, I64, I64, I64, I64, F32, P, I64, I64, P, I64, I64,
                                          INT, P, INT, INT, P, SZ, P],
    "dsa_peer_alloc": [SZ, ctypes.POINTER(P), P],
    "dsa_peer_open": [P, ctypes.POINTER(P)],
    "dsa_peer_close": [P],
    "dsa_peer_free": [P],
    "dsa_peer_barrier": [P, INT, INT, P, P],
    "dsa_read_device_error": [P, INT, ctypes.POINTER(INT), P],
    "dsa_indexer_scores": [P, P, I64, P, I64, P, P, I64, P, I64, I64, I64, I64, I64, P, I64, P, P],
    "dsa_index_cache_append": [P, I64, P, P, I64, P, I64, I64, P, P],
    "dsa_topk_select": [P, I64, P, P, I64, I64, I64, P, P, INT, P],
    "dsa_indexer_topk": [P, P, I64, P, I64, P, P, I64, P, I64, I64, I64, I64, I64, I64, P, P, P,
                         INT, P, P],
    "dsa_step_layout": [P, P, I64, P, I64, I64, P, I64, P, I64, P, P, P, P, P, P, P],
    "dsa_apply_rope": [P, I64, I64, P, I64, I64, INT, I64, I64, I64, I64, I64, P, INT, P, INT, INT, F32,
                       P],
    "dsa_latent_cache_append": [P, I64, INT, P, INT, I64, P, INT, P, P, P, I64, I64, P, I64, I64, I64,
                                F32, INT, F32, P, P],
    "dsa_shared_prefix_attention_workspace_size": [I64, I64, ctypes.POINTER(SZ)],
    "dsa_shared_prefix_attention": [P, I64, I64, P, I64, I64, P, I64, I64, P, I64, I64, P, I64, P, P, I64,
                                    I64, I64, P, P, I64, I64, I64, F32, P, I64, I64, P, I64, I64, P, SZ,
                                    P],
    "dsa_shared_prefix_attention_scratch": [P, I64, I64, P, I64, I64, P, I64, I64, P, I64, I64, P, I64, P, P,
                                            I64, I64, I64, P, P, I64, I64, I64, F32, P, I64, I64, P, I64, I64,
                                            P, SZ, P, P],
}


class DSAError(RuntimeError):
    """A failing call of the native library (status code + message)."""

    def __init__(self, fn, code, msg):
        super().__init__(f"{fn} failed with status {code}: {msg}")
        self.code = code


def lib_path() -> str:
    return _build.LIB


def load(build_if_missing: bool = True):
    global _lib
    if _lib is not None:
        return _lib
    path = lib_path()
    if not os.path.exists(path):
        if not build_if_missing:
            raise OSError(f"{path} is missing; run python -m flashinfer_repo_b200.build")
        _build.build()
    lib = ctypes.CDLL(path)
    lib.dsa_last_error_message.restype = ctypes.c_char_p
    lib.dsa_last_error_message.argtypes = []
    for name, args in SIGNATURES.items():
        f = getattr(lib, name)
        f.argtypes = args
        f.restype = INT
    _lib = lib
    return lib


def check(fn_name: str, rc: int):
    if rc != 0:
        msg = load().dsa_last_error_message().decode(errors="replace")
        raise DSAError(fn_name, rc, msg)


def call(fn_name: str, *args):
    check(fn_name, getattr(load(), fn_name)(*args))


_bound = {}
# the raw getters: torch.cuda.current_stream builds an object, 1.5 us a call
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else None
_current_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


def call_on(index: int, fn_name: str, *args):
    """`call` with CUDA device `index` current and torch's current stream of that
    device as the last argument."""
    f = _bound.get(fn_name)
    if f is None:
        f = _bound[fn_name] = getattr(load(), fn_name)
    if _current_device() == index:
        rc = f(*args, _current_stream(index))
    else:
        with torch.cuda.device(index):
            rc = f(*args, _current_stream(index))
    if rc != 0:
        check(fn_name, rc)


# memory of torch's allocator without a tensor around it: 0.5 us, a tensor takes 1.6
_alloc = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_alloc", None)
_free = getattr(torch._C, "_cuda_cudaCachingAllocator_raw_delete", None)


def call_with_scratch(index: int, fn_name: str, nbytes: int, error: int, *args):
    """`call_on` of a function whose last arguments are a workspace, its size, a
    device error word and the stream.  The workspace is torch's memory of that
    stream (of the graph, in a capture) and goes back to it in stream order."""
    if _current_device() != index:
        with torch.cuda.device(index):
            return call_with_scratch(index, fn_name, nbytes, error, *args)
    stream = _current_stream(index)
    f = _bound.get(fn_name)
    if f is None:
        f = _bound[fn_name] = getattr(load(), fn_name)
    scratch = _alloc(nbytes, stream)
    try:
        rc = f(*args, scratch, nbytes, error, stream)
        if rc != 0:
            check(fn_name, rc)
    finally:
        _free(scratch)


def same_device(first, *others) -> int:
    """Index of the one CUDA device that all tensors (None is skipped) are on;
    RuntimeError if they are on several or on the CPU."""
    index = first.get_device()
    for t in others:
        if t is not None and t.get_device() != index:
            index = -1
            break
    if index < 0:
        where = [str(t.device) for t in (first, *others) if t is not None]
        raise RuntimeError(f"all tensors must be on one CUDA device (no CPU path), got {where}")
    return index


def int32(t, name: str):
    """Contiguous int32 copy of an id or length tensor (itself if it is one);
    64-bit values past 32 bits are cut to the range's ends, not wrapped around."""
    if t.dtype == torch.int32:
        return t if t.is_contiguous() else t.contiguous()
    assert t.dtype == torch.int64, f"{name} must be int32 or int64"
    return t.clamp(-2 ** 31, 2 ** 31 - 1).to(torch.int32).contiguous()
