"""Rotary positions for queries and keys of the DSA step.

The reference takes rotated q_pe, k_pe and index queries (solution/triton/
kernel.py:138, indexer_kernel.py:345) and has no operator that makes them.
Angles are position * inv_freq with inv_freq in 64 bits, reduced on the device
before they are rounded, so far positions lose nothing and there is no table of
cosines to size or gather.
"""
from __future__ import annotations

import math

import torch

from . import _lib

LAYOUTS = {"interleaved": 0, "half": 1}
DTYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}


def rope_frequencies(rot_dim, base=10000.0, *, scaling=None, factor=1.0, original_context=4096, beta_fast=32.0,
                     beta_slow=1.0, device="cuda") -> torch.Tensor:
    """inv_freq [rot_dim/2] float64 = base^(-2i/rot_dim), stretched for long contexts:

    scaling None      as they are
    "linear"          every frequency divided by `factor`
    "ntk"             the base grows, base * factor^(rot_dim/(rot_dim-2))
    "yarn"            by parts: pairs that turn more than beta_fast times over
                      original_context stay, those under beta_slow turns are
                      divided by `factor`, a linear ramp between
    """
    rot_dim = int(rot_dim)
    assert rot_dim >= 2 and rot_dim % 2 == 0, "rot_dim must be even"
    if scaling not in (None, "linear", "ntk", "yarn"):
        raise ValueError(f"unknown scaling {scaling!r}")
    if scaling is not None and not factor >= 1.0:
        raise ValueError("factor must be at least 1")
    if scaling == "ntk":
        assert rot_dim > 2, "ntk scaling needs more than one pair"
        base = base * factor ** (rot_dim / (rot_dim - 2))
    i = torch.arange(0, rot_dim, 2, dtype=torch.float64)
    inv = base ** (-i / rot_dim)
    if scaling == "linear":
        inv = inv / factor
    elif scaling == "yarn":
        def pair(turns):  # the (fractional) pair that makes `turns` turns over the original context
            return rot_dim * math.log(original_context / (turns * 2 * math.pi)) / (2 * math.log(base))
        low, high = max(math.floor(pair(beta_fast)), 0), min(math.ceil(pair(beta_slow)), rot_dim - 1)
        ramp = ((torch.arange(rot_dim // 2, dtype=torch.float64) - low) / max(high - low, 1e-3)).clamp(0, 1)
        inv = inv * (1 - ramp) + inv / factor * ramp
    return inv.to(device)


def _check_rotation(positions, inv_freq, tokens, layout):
    if layout not in LAYOUTS:
        raise ValueError(f"layout must be one of {sorted(LAYOUTS)}, got {layout!r}")
    assert positions.shape == (tokens,) and positions.dtype in (torch.int32, torch.int64), \
        "positions must be [tokens] int32 or int64"
    assert inv_freq.dim() == 1 and inv_freq.dtype == torch.float64, "inv_freq must be [rot_dim/2] float64"
    return positions.contiguous(), inv_freq.contiguous()


class _Turn(torch.autograd.Function):
    """The turn with its gradient, the turn back."""

    @staticmethod
    def forward(ctx, x, positions, inv_freq, layout, offset, inverse, scale):
        ctx.save_for_backward(positions, inv_freq)
        ctx.turn = layout, offset, inverse, scale
        return apply_rope(x, positions, inv_freq, layout=layout, offset=offset, inverse=inverse, scale=scale)

    @staticmethod
    def backward(ctx, grad):
        positions, inv_freq = ctx.saved_tensors
        layout, offset, inverse, scale = ctx.turn
        grad = apply_rope(grad, positions, inv_freq, layout=layout, offset=offset, inverse=not inverse, scale=scale)
        return grad, None, None, None, None, None, None


def apply_rope(x, positions, inv_freq, *, layout="interleaved", offset=0, inverse=False, scale=1.0, out=None):
    """Turn the slice [offset, offset + rot_dim) of every head of x [T, H, D]
    (or [T, D]) to its token's position, rot_dim = 2 * len(inv_freq); the other
    values are copied.

    positions [T] int32 or int64; inv_freq float64 (`rope_frequencies`).
    layout "interleaved" pairs values (2i, 2i+1) of the slice, "half" (i, i +
    rot_dim/2).  scale multiplies the turned slice (the attention factor of
    scaled frequencies).  inverse=True turns back: with the same scale it is the
    gradient of the forward turn, which autograd records for an x that requires
    one.  out: a tensor of x's shape and type to write into, x itself for in
    place (nothing can be recorded then); any other overlap with x is not allowed.
    bf16, fp16 or fp32; products in 32 bits, one rounding.
    """
    if torch.is_grad_enabled() and (x.requires_grad or inv_freq.requires_grad):
        if out is not None or inv_freq.requires_grad:
            raise RuntimeError("apply_rope records gradients of x only, and not into out=: use torch.no_grad()")
        return _Turn.apply(x, positions, inv_freq, layout, offset, inverse, scale)
    shape = x.shape
    assert len(shape) in (2, 3), "x must be [tokens, heads, dim] or [tokens, dim]"
    dtype = DTYPES.get(x.dtype)
    assert dtype is not None, f"x must be bf16, fp16 or fp32, got {x.dtype}"
    index = _lib.same_device(x, positions, inv_freq, out)
    positions, inv_freq = _check_rotation(positions, inv_freq, shape[0], layout)
    rot = 2 * inv_freq.shape[0]
    assert 0 <= offset and offset + rot <= shape[-1], "the rotated slice reaches past the head"
    x_at = x.stride()
    if x_at[-1] != 1:
        assert out is None or out.data_ptr() != x.data_ptr(), "in place needs contiguous heads"
        x = x.contiguous()
        x_at = x.stride()
    if out is None:
        out = x.new_empty(shape)
        o_at = out.stride()
    else:
        o_at = out.stride()
        assert out.shape == shape and out.dtype == x.dtype and o_at[-1] == 1
        assert all(st > 0 for st, n in zip(o_at, shape) if n > 1), "out is an expanded tensor"
        assert out.data_ptr() != x.data_ptr() or o_at == x_at, "out shares x's memory with other strides"
    heads, x_head, o_head = (shape[1], x_at[1], o_at[1]) if len(shape) == 3 else (1, 0, 0)
    _lib.call_on(index, "dsa_apply_rope", x.data_ptr(), x_at[0], x_head, out.data_ptr(), o_at[0], o_head, dtype,
                 shape[0], heads, shape[-1], offset, rot, positions.data_ptr(), positions.dtype == torch.int64,
                 inv_freq.data_ptr(), LAYOUTS[layout], bool(inverse), scale)
    return out
