"""Writer of the paged MLA latent cache that `kernel()` and
`shared_prefix_attention` read: latent norm, rotary key and paged store in one
pass over the projection's rows.  The reference takes a filled cache
(solution/triton/kernel.py:138) and has no writer.
"""
from __future__ import annotations

import torch

from . import _lib
from .kernel import HEAD_DIM_CKV, HEAD_DIM_KPE, PAGE_SIZE
from .rope import DTYPES, LAYOUTS, _check_rotation


def latent_cache_append(kv, norm_weight, positions, slots, inv_freq, ckv_cache, kpe_cache, *, eps=1e-6,
                        layout="interleaved", rope_scale=1.0, device_error=None) -> None:
    """Write rows of kv [T, 576] (512 latent values, 64 rotary key values) at
    flat slot ids slots [T] (-1 = skip) of ckv_cache [P, 64, 512] and kpe_cache
    [P, 64, 64] (bf16):

        ckv = x * rsqrt(mean(x^2) + eps) * norm_weight,   kpe = rope(x[512:]) * rope_scale

    kv may be a strided view (a slice of a wider projection) in bf16, fp16 or
    fp32; norm_weight [512] likewise; positions [T] int32 or int64; inv_freq [32]
    float64 (`rope_frequencies(64)`).  Sums and products in 32 bits, one rounding
    to bf16.  Slots must be distinct (-1 apart).  device_error: optional int32
    tensor that collects DSA_DEVERR_* bits (1: a slot outside the cache, skipped).
    """
    tokens, width = kv.shape
    num_pages = ckv_cache.shape[0]
    kv_type, norm_type = DTYPES.get(kv.dtype), DTYPES.get(norm_weight.dtype)
    assert width == HEAD_DIM_CKV + HEAD_DIM_KPE, "kv must be [tokens, 576]"
    assert kv_type is not None and norm_type is not None, "kv and norm_weight: bf16, fp16 or fp32"
    assert norm_weight.shape == (HEAD_DIM_CKV,)
    assert ckv_cache.dtype == torch.bfloat16 and kpe_cache.dtype == torch.bfloat16, "the caches are bf16"
    assert ckv_cache.shape == (num_pages, PAGE_SIZE, HEAD_DIM_CKV)
    assert kpe_cache.shape == (num_pages, PAGE_SIZE, HEAD_DIM_KPE)
    assert slots.shape == (tokens,), "slots must be [tokens]"
    assert inv_freq.shape == (HEAD_DIM_KPE // 2,), "inv_freq must have 32 values"
    index = _lib.same_device(kv, norm_weight, positions, slots, inv_freq, ckv_cache, kpe_cache, device_error)
    positions, inv_freq = _check_rotation(positions, inv_freq, tokens, layout)
    if device_error is not None:
        assert device_error.dtype == torch.int32 and device_error.numel() >= 1, "device_error must be int32"
    if kv.stride(1) != 1:
        kv = kv.contiguous()
    norm_weight = norm_weight.contiguous()
    slots = _lib.int32(slots, "slots")
    c_page, c_row, c_last = ckv_cache.stride()
    e_page, e_row, e_last = kpe_cache.stride()
    assert c_last == 1 and e_last == 1, "cache rows must be contiguous"
    _lib.call_on(index, "dsa_latent_cache_append", kv.data_ptr(), kv.stride(0), kv_type, norm_weight.data_ptr(), norm_type,
                 tokens, positions.data_ptr(), positions.dtype == torch.int64, slots.data_ptr(), inv_freq.data_ptr(),
                 ckv_cache.data_ptr(), c_page, c_row, kpe_cache.data_ptr(), e_page, e_row, num_pages, eps,
                 LAYOUTS[layout], rope_scale, device_error.data_ptr() if device_error is not None else None)
