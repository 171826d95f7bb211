"""The serving-step operators at the edges of what their documentation allows."""
from __future__ import annotations

import math

import pytest
import torch

import flashinfer_repo_b200 as fi

from . import prefix_oracle as P

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192.0)
I32 = torch.int32


def _put(*v):
    return torch.tensor(v, dtype=I32, device="cuda")


def _attend(c, **kw):
    a = {"pages": c["pages"], "prefix": c["prefix"], "ckv": c["ckv"], "kpe": c["kpe"], **kw}
    extra = {k: a[k] for k in ("output", "lse", "workspace") if k in a}
    return fi.shared_prefix_attention(c["qn"], c["qp"], a["ckv"], a["kpe"], a["pages"], a["prefix"], c["table"], c["lens"],
                                      SCALE, token_request=c["request"], **extra)


# ------------------------------------------------------------- step layout
@pytest.mark.parametrize("seq,q,width,slots", [
    (641, 1, 10, [-1]),            # the row's page is a column past the table and was there before
    (700, 3, 8, [-1, -1, -1]),
    (639, 2, 10, [5 * 64 + 63, -1]),  # the second row would need a new one past the table
    (638, 2, 10, [5 * 64 + 62, 5 * 64 + 63])])
def test_layout_flags_rows_past_the_table(seq, q, width, slots):
    table = torch.full((1, width), 5, dtype=I32, device="cuda")
    err = torch.zeros(1, dtype=I32, device="cuda")
    lay = fi.step_layout(_put(seq), _put(q), table, _put(7, 8, 9), q, device_error=err)
    assert lay.slots.tolist() == slots and err.item() == (4 if -1 in slots else 0)
    assert (table == 5).all()


# ------------------------------------------------------ shared-prefix attention
def test_prefix_pages_must_be_one_list():
    c = P.make_case(1, 3, 16, 200, [1, 0, 70])
    for pages in (c["pages"][None], c["pages"][:, None]):
        for prefix in (c["prefix"], 64):
            with pytest.raises(AssertionError, match="prefix_pages"):
                _attend(c, pages=pages, prefix=prefix)


def test_outputs_shared_by_rows_are_refused():
    c = P.make_case(2, 3, 32, 100, [1, 0, 70])
    for output in (torch.empty((1, 32, 512), dtype=torch.bfloat16, device="cuda").expand(3, 32, 512),
                   torch.empty((3, 1, 512), dtype=torch.bfloat16, device="cuda").expand(3, 32, 512)):
        with pytest.raises(AssertionError, match="expanded"):
            _attend(c, output=output)
    for lse in (torch.empty((1, 32), device="cuda").expand(3, 32), torch.empty((3, 1), device="cuda").expand(3, 32)):
        with pytest.raises(AssertionError, match="expanded"):
            _attend(c, lse=lse)
    # a single token or any strides that keep rows apart are fine
    one = {**c, "qn": c["qn"][:1], "qp": c["qp"][:1], "lens": c["lens"][:1], "request": c["request"][:1]}
    P.check(one, _attend(one, output=torch.empty((1, 32, 512), dtype=torch.bfloat16, device="cuda").expand(1, 32, 512)), SCALE)
    turned = torch.empty((32, 3, 512), dtype=torch.bfloat16, device="cuda").transpose(0, 1)
    P.check(c, _attend(c, output=turned, lse=torch.empty((32, 3), device="cuda").T), SCALE)


def test_refused_caches_are_not_copied():
    """A cache that the loads cannot read is refused, without a copy of it being made first."""
    pages = 2000
    c = P.make_case(3, 2, 16, 100, [1, 70])
    wide = torch.zeros((pages, 64, 580), dtype=torch.bfloat16, device="cuda")
    good = torch.zeros((pages, 64, 576), dtype=torch.bfloat16, device="cuda")
    shifted = torch.zeros(pages * 64 * 512 + 8, dtype=torch.bfloat16, device="cuda")[4:pages * 64 * 512 + 4]
    _attend(c)
    for ckv, kpe in ((wide[..., :512], wide[..., 512:576]), (shifted.view(pages, 64, 512), good[..., 512:]),
                     (good[..., :512], wide[..., 516:])):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        with pytest.raises(AssertionError, match="cache rows"):
            _attend(c, ckv=ckv, kpe=kpe)
        assert torch.cuda.max_memory_allocated() - before < 2 ** 20


@pytest.mark.parametrize("heads,live,padded,own", [(16, 5, 3, 6000), (16, 3, 13, 700), (32, 2, 6, 1000)])
def test_padded_rows_leave_the_pages_of_a_request_shared(heads, live, padded, own):
    """One request with several tokens and rows behind the last one (request 0, length 0, as step_layout makes them):
    its own pages are in the list of the row block once, not once a token."""
    tokens = live + padded
    c = P.make_case(4, 1, heads, 200, [own])
    c["lens"] = _put(*(own - live + 1 + i for i in range(live)), *[0] * padded)
    c["request"] = torch.zeros(tokens, dtype=I32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(5)
    c["qn"] = torch.randn((tokens, heads, 512), generator=g, device="cuda").to(torch.bfloat16)
    c["qp"] = torch.randn((tokens, heads, 64), generator=g, device="cuda").to(torch.bfloat16)
    ws = torch.zeros(fi.prefix_workspace_size(tokens, heads), dtype=torch.uint8, device="cuda")
    got = _attend(c, workspace=ws)
    P.check(c, got, SCALE)
    blocks = -(-tokens * (heads // 16) // 8)
    tiles = ws[256:256 + 8 * (blocks + 1)].view(torch.int64).diff().tolist()
    # the prefix, the pages that all live tokens see whole, and one more for each token, two pages a tile
    assert tiles[0] <= (4 + own // 64 + 2 * live + 1) // 2 + 1, tiles


def test_empty_rows_between_the_tokens_of_a_request():
    c = P.make_case(6, 2, 16, 130, [400, 90])
    c["lens"], c["request"] = _put(300, 0, 399, 400, 0, 0, 90, 0, 77), _put(0, 0, 0, 0, 1, 0, 1, 1, 1)
    g = torch.Generator(device="cuda").manual_seed(7)
    c["qn"] = torch.randn((9, 16, 512), generator=g, device="cuda").to(torch.bfloat16)
    c["qp"] = torch.randn((9, 16, 64), generator=g, device="cuda").to(torch.bfloat16)
    P.check(c, _attend(c), SCALE)
    c["prefix"].zero_()
    P.check(c, _attend(c), SCALE)
    assert fi.read_prefix_error() == 0


# ------------------------------------------------------------------ rotary
def _turn64(x, pos, inv, layout, offset, scale):
    ang = pos.double()[:, None, None] * inv
    c, s, r = torch.cos(ang), torch.sin(ang), 2 * inv.numel()
    z = x[..., offset:offset + r]
    a, b = (z[..., 0::2], z[..., 1::2]) if layout == "interleaved" else z.chunk(2, -1)
    y = ((a * c - b * s) * scale, (b * c + a * s) * scale)
    y = torch.stack(y, -1).flatten(-2) if layout == "interleaved" else torch.cat(y, -1)
    return torch.cat((x[..., :offset], y, x[..., offset + r:]), -1)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("flat", [False, True])
def test_rope_gradient_follows_the_result(layout, flat):
    """A tensor that requires gradients gets the formula's, through a strided view and a second time over."""
    g = torch.Generator(device="cuda").manual_seed(8)
    leaf = torch.randn((9, 5, 104), generator=g, device="cuda", requires_grad=True)
    pos, inv = torch.arange(9, device="cuda", dtype=I32) * 7919, fi.rope_frequencies(64)
    dy = torch.randn((9, 5, 96), generator=g, device="cuda")
    view = leaf[..., 8:]
    if flat:
        view, dy = view[:, 2], dy[:, 2].contiguous()
    y = fi.apply_rope(view, pos, inv, layout=layout, offset=16, scale=1.3)
    (grad,) = torch.autograd.grad(y, leaf, dy, create_graph=False)
    l64 = leaf.detach().double().requires_grad_()
    v64 = l64[..., 8:]
    ref = _turn64(v64[:, 2][:, None] if flat else v64, pos, inv, layout, 16, 1.3)
    (want,) = torch.autograd.grad(ref, l64, (dy[:, None] if flat else dy).double())
    # |a| + |b| of two normal values stays below 12, scaled by 1.3; 7e-7 of it: the angle's rounding and the products
    assert (grad.double() - want).abs().max() <= 1.3 * 12 * 7e-7 + 12 * 2 ** -24
    assert (y.detach().double() - (ref[:, 0] if flat else ref)).abs().max() <= 1.3 * 12 * 7e-7 + 12 * 2 ** -24
    # against differences: the turn is linear, so they are exact up to rounding
    step = torch.randn(leaf.shape, generator=g, device="cuda")
    with torch.no_grad():
        moved = (leaf + step)[..., 8:]
        moved = fi.apply_rope(moved[:, 2] if flat else moved, pos, inv, layout=layout, offset=16, scale=1.3)
        slope, along = ((moved - y) * dy).double().sum(), (grad * step).double().sum()
    n = dy.numel()
    assert (slope - along).abs() <= n ** 0.5 * 8 * 12 * 12 * 1e-6


def test_rope_gradient_is_recorded_only_where_wanted():
    x = torch.randn((4, 2, 64), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    pos, inv = _put(1, 2, 3, 4), fi.rope_frequencies(64)
    y = fi.apply_rope(x, pos, inv)
    assert y.requires_grad and y.dtype == torch.bfloat16
    with torch.no_grad():
        z = fi.apply_rope(x, pos, inv)
        fi.apply_rope(x, pos, inv, out=x)  # in place is fine where nothing is recorded
    assert not z.requires_grad and torch.equal(y, z) and torch.equal(x, z)
    assert not fi.apply_rope(x.detach(), pos, inv).requires_grad
    for out in (x, torch.empty_like(x)):
        with pytest.raises(RuntimeError, match="grad"):
            fi.apply_rope(x, pos, inv, out=out)
    with pytest.raises(RuntimeError, match="grad"):
        fi.apply_rope(x.detach(), pos, inv.clone().requires_grad_())
    # twice differentiable: the turn of the turned-back gradient
    dy = torch.randn((4, 2, 64), device="cuda", dtype=torch.bfloat16, requires_grad=True)
    (g,) = torch.autograd.grad(fi.apply_rope(x, pos, inv), x, dy, create_graph=True)
    (h,) = torch.autograd.grad(g, dy, torch.ones_like(g))
    assert torch.equal(h, fi.apply_rope(torch.ones_like(x), pos, inv).detach())
