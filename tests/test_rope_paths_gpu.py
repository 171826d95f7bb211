"""The rotary turn's kernels by launch: four units a lane (many tokens), one (few), value by value; in place and not."""
from __future__ import annotations

import pytest
import torch

import flashinfer_repo_b200 as fi

pytestmark = pytest.mark.gpu


def _turn64(x, pos, inv, layout, offset, inverse, scale):
    """The slice turned in 64 bits and |a| + |b| of its pairs."""
    ang = pos.double()[:, None, None] * inv * (-1 if inverse else 1)
    c, s, r = torch.cos(ang), torch.sin(ang), 2 * inv.numel()
    z = x[..., offset:offset + r].double()
    a, b = (z[..., 0::2], z[..., 1::2]) if layout == "interleaved" else z.chunk(2, -1)
    join = (lambda u, v: torch.stack((u, v), -1).flatten(-2)) if layout == "interleaved" else \
        (lambda u, v: torch.cat((u, v), -1))
    m = (a.abs() + b.abs()) * abs(scale)
    return join((a * c - b * s) * scale, (b * c + a * s) * scale), join(m, m)


def _check(got, x, pos, inv, layout, offset, inverse, scale):
    want, mag = _turn64(x, pos, inv, layout, offset, inverse, scale)
    r = 2 * inv.numel()
    f = torch.finfo(x.dtype)
    # one rounding to the type; half a turn rounded (2^-24 half turns, 1.9e-7 rad), cos and sin to 2 ulp, their scaling,
    # two products and a sum in 32 bits: below 7e-7 of |a| + |b|; a denormal's step
    tol = f.eps / 2 * want.abs() + 7e-7 * mag + f.smallest_normal * f.eps
    assert ((got[..., offset:offset + r].double() - want).abs() <= tol).all()
    assert torch.equal(got[..., :offset], x[..., :offset]) and torch.equal(got[..., offset + r:], x[..., offset + r:])


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,heads,dim,offset,rot", [
    (1500, 64, 128, 0, 64),   # half of every head turned, the rest copied
    (703, 33, 192, 128, 64),  # an odd number of heads, the slice behind
    (1100, 20, 64, 0, 64),    # all turned
    (2500, 1, 576, 512, 64),  # one head, a short slice of a long row
    (900, 17, 160, 16, 128),
    (600, 128, 48, 8, 32),
    (64, 16, 192, 128, 64),   # few tokens: one unit a lane
    (3, 7, 128, 64, 64)])
def test_aligned_heads(tokens, heads, dim, offset, rot, layout, dtype):
    g = torch.Generator(device="cuda").manual_seed(tokens)
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 1 << 18, (tokens,), generator=g, device="cuda", dtype=torch.int32)
    inv = fi.rope_frequencies(rot, 500000.0)
    got = fi.apply_rope(x, pos, inv, layout=layout, offset=offset)
    _check(got, x, pos, inv, layout, offset, False, 1.0)
    back = fi.apply_rope(x, pos.long(), inv, layout=layout, offset=offset, inverse=True, scale=0.7)
    _check(back, x, pos, inv, layout, offset, True, 0.7)
    # in place, and in place in the middle of a wider buffer: the same values, and nothing beside them is written
    same = x.clone()
    assert fi.apply_rope(same, pos, inv, layout=layout, offset=offset, out=same) is same
    assert torch.equal(same, got)
    wide = torch.randn((tokens, heads + 2, dim + 32), generator=g, device="cuda").to(dtype)
    part = wide[:, 1:heads + 1, 16:16 + dim]
    part.copy_(x)
    want = wide.clone()
    want[:, 1:heads + 1, 16:16 + dim] = got
    fi.apply_rope(part, pos, inv, layout=layout, offset=offset, out=part)
    assert torch.equal(wide, want)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_values_one_by_one(layout, dtype):
    """Widths and starts off a 16-byte boundary, and a half layout of 48 values: many tokens, in place and not."""
    g = torch.Generator(device="cuda").manual_seed(3)
    for tokens, heads, dim, offset, rot in ((2000, 9, 99, 1, 62), (1300, 16, 144, 96, 48), (777, 5, 130, 2, 128)):
        x = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(dtype)
        pos = torch.randint(0, 1 << 18, (tokens,), generator=g, device="cuda", dtype=torch.int32)
        inv = fi.rope_frequencies(rot)
        got = fi.apply_rope(x, pos, inv, layout=layout, offset=offset)
        _check(got, x, pos, inv, layout, offset, False, 1.0)
        assert torch.equal(fi.apply_rope(x, pos, inv, layout=layout, offset=offset, out=x), got)
