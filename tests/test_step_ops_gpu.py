"""The serving-step operators against plain 64-bit implementations: step layout,
rotary positions, latent-cache writer, shared-prefix attention, and a run of them
together.  Tolerances count roundings: half a step of a type is eps/2 of the value."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

import flashinfer_repo_b200 as fi
from flashinfer_repo_b200.pipeline import run_shared_prefix_step

pytestmark = pytest.mark.gpu
PAGE, DC, DP = 64, 512, 64
SCALE = 1 / math.sqrt(192.0)
I32 = torch.int32


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _put(a, t=I32):
    return torch.as_tensor(np.ascontiguousarray(a)).to("cuda", t)


# ------------------------------------------------------------- step layout
def _layout_oracle(seq, q, table, free, rows, prefix):
    table = table.copy()
    out = np.zeros((4, rows), np.int64)
    out[0] = -1
    row = used = 0
    bits = 0
    for b in range(len(seq)):
        for i in range(max(q[b], 0)):
            pos = max(seq[b], 0) + i
            if pos % PAGE == 0:  # a new page
                page = free[used] if used < len(free) else -1
                bits |= 4 * (used >= len(free) or pos // PAGE >= table.shape[1])
                used += 1
                if pos // PAGE < table.shape[1]:
                    table[b, pos // PAGE] = page
            page = table[b, pos // PAGE] if pos // PAGE < table.shape[1] else -1
            if row < rows:
                out[:, row] = page * PAGE + pos % PAGE if page >= 0 else -1, prefix + pos, b, pos + 1
            else:
                bits |= 4
            row += 1
    return table, out, min(used, len(free)), bits


def _check_layout(seq, q, width, nfree, rows, prefix, seed=0, poison=None):
    rng = np.random.default_rng(seed)
    seq, q = np.asarray(seq), np.asarray(q)
    table = rng.integers(0, 1 << 20, (len(seq), width))
    if poison is not None:
        table[poison] = -5
    free = rng.permutation(1 << 16)[:nfree]
    dev = _put(table)
    err = torch.zeros(1, dtype=I32, device="cuda")
    want_table, want, used, bits = _layout_oracle(seq, q, table, free, rows, prefix)
    for _ in range(2):  # the second call finds its own pages in the table: the same result
        lay = fi.step_layout(_put(seq), _put(q), dev, _put(free), rows, prefix_len=_put([prefix]), device_error=err)
        got = np.stack([t.cpu().numpy() for t in lay[:4]])
        assert np.array_equal(dev.cpu().numpy(), want_table)
        assert np.array_equal(got, want)
        assert lay.pages_used.item() == used
    return err.item(), bits


@pytest.mark.parametrize("seq,q,rows,prefix", [
    ([5], [1], 1, 0), ([64], [1], 1, 7), ([63], [2], 2, 0), ([0], [0], 0, 0), ([0, 0, 0], [0, 200, 1], 230, 1000),
    ([130, 0, 64, 63, 1], [1, 64, 65, 1, 0], 140, 64)])
def test_layout_small(seq, q, rows, prefix):
    err, bits = _check_layout(seq, q, 12, 40, rows, prefix)
    assert err == 0 and bits == 0


@pytest.mark.parametrize("batch", [1, 31, 511, 512, 513, 2048, 5000])
def test_layout_many_requests(batch):
    """Batches around the chunk of the scan, decode rows with some chunks and idle requests."""
    rng = np.random.default_rng(batch)
    seq = rng.integers(0, 700, batch)
    q = rng.choice([0, 1, 1, 1, 3, 150], batch)
    assert _check_layout(seq, q, 16, 20000, int(q.sum()) + 77, 4096, batch)[0] == 0


def test_layout_one_long_request():
    assert _check_layout([100], [70000], 1200, 1200, 70000, 0)[0] == 0


def test_layout_runs_out():
    """Too few free pages, table columns or rows: -1 slots or dropped rows, and the flag."""
    for width, nfree, rows in ((8, 2, 300), (2, 40, 300), (8, 40, 100), (8, 0, 300)):
        err, bits = _check_layout([10, 60, 128], [100, 90, 110], width, nfree, rows, 0)
        assert bits == 4 and err == 4


def test_layout_bad_entry_and_negative_lengths():
    err, _ = _check_layout([70, -3, 5], [1, 2, -9], 4, 8, 4, 0, poison=(0, 1))
    assert err == 1


def test_layout_out_int64_and_padding():
    out = fi.StepLayout(*(torch.full((n,), 99, dtype=I32, device="cuda") for n in (4, 4, 4, 4, 1)))
    table = torch.zeros((2, 3), dtype=I32, device="cuda")
    got = fi.step_layout(_put([3, 64], torch.int64), _put([1, 1], torch.int64), table, _put([9, 8], torch.int64), 4,
                         out=out)
    assert got is out and out.slots.tolist() == [3, 9 * 64, -1, -1] and out.pages_used.tolist() == [1]
    assert out.positions.tolist() == [3, 64, 0, 0] and out.token_lens.tolist() == [4, 65, 0, 0]
    assert out.token_request.tolist() == [0, 1, 0, 0] and table.tolist() == [[0, 0, 0], [0, 9, 0]]


# ------------------------------------------------------------------ rotary
def _rope64(x, pos, inv, layout, offset, inverse, scale):
    y = x.double().clone()
    r = 2 * inv.numel()
    z = y[..., offset:offset + r]
    ang = pos.double()[:, None, None] * inv * (-1 if inverse else 1)
    c, s = torch.cos(ang), torch.sin(ang)
    a, b = (z[..., 0::2], z[..., 1::2]) if layout == "interleaved" else z.chunk(2, -1)
    ra, rb = (a * c - b * s) * scale, (b * c + a * s) * scale
    y[..., offset:offset + r] = torch.stack((ra, rb), -1).flatten(-2) if layout == "interleaved" \
        else torch.cat((ra, rb), -1)
    # what the products are made of, for the 32-bit share of the tolerance
    mag = torch.zeros_like(y)
    m = (a.abs() + b.abs()) * abs(scale)
    mag[..., offset:offset + r] = torch.stack((m, m), -1).flatten(-2) if layout == "interleaved" else torch.cat((m, m), -1)
    return y, mag


def _close_rope(got, x, pos, inv, layout, offset, inverse, scale):
    want, mag = _rope64(x, pos, inv, layout, offset, inverse, scale)
    # one rounding to the type; in 32 bits: half a turn rounded (2^-24 half turns, pi * 2^-24 = 1.9e-7 rad),
    # cos and sin to 2 ulp, their scaling, two products and a sum: below 8 * 2^-24 = 4.8e-7 of |a| + |b|
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps  # a denormal's step
    tol = torch.finfo(x.dtype).eps / 2 * want.abs() + 7e-7 * mag + tiny
    assert ((got.double() - want).abs() <= tol).all()
    r = 2 * inv.numel()
    assert torch.equal(got[..., :offset], x[..., :offset]) and torch.equal(got[..., offset + r:], x[..., offset + r:])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("tokens,heads,dim,offset,rot", [
    (1, 1, 64, 0, 64), (3, 16, 192, 128, 64), (65, 5, 128, 0, 64), (130, 7, 96, 3, 62), (2, 128, 576, 512, 64),
    (9, 3, 2, 0, 2), (5, 2, 512, 0, 512), (33, 4, 72, 8, 48)])
def test_rope(tokens, heads, dim, offset, rot, layout, dtype):
    g = _gen(tokens + dim)
    x = torch.randn((tokens, heads, dim), generator=g, device="cuda").to(dtype)
    pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda", dtype=I32)
    pos[0] = 0
    inv = fi.rope_frequencies(rot, scaling="yarn", factor=4.0) if rot > 2 else fi.rope_frequencies(rot)
    for inverse, scale in ((False, 1.0), (True, 0.7)):
        got = fi.apply_rope(x, pos, inv, layout=layout, offset=offset, inverse=inverse, scale=scale)
        _close_rope(got, x, pos, inv, layout, offset, inverse, scale)


@pytest.mark.parametrize("layout", ["interleaved", "half"])
def test_rope_views(layout):
    """Strided views, rows off a 16-byte boundary, in place, 2-D, 64-bit positions, empty batches."""
    g = _gen(5)
    big = torch.randn((40, 8, 200), generator=g, device="cuda").to(torch.bfloat16)
    pos = torch.randint(0, 1 << 22, (40,), generator=g, device="cuda", dtype=torch.int64)
    inv = fi.rope_frequencies(64)
    for view in (big[..., 8:200], big[..., 3:195], big[::2, 1:7, :128], big.transpose(0, 1)[:, :8, 72:136],
                 big[..., 1:193:2]):
        p = pos[:view.shape[0]]
        _close_rope(fi.apply_rope(view, p, inv, layout=layout), view, p, inv, layout, 0, False, 1.0)
    before, part = big.clone(), big[5:25, 2:6, 101:165]
    got = fi.apply_rope(part, pos[5:25], inv, layout=layout, out=part)
    assert got is part
    _close_rope(part, before[5:25, 2:6, 101:165], pos[5:25], inv, layout, 0, False, 1.0)
    before[5:25, 2:6, 101:165] = part
    assert torch.equal(before, big)  # nothing outside the view is written
    flat = big[:, 0, :128].contiguous()
    got = fi.apply_rope(flat, pos, inv, layout=layout, offset=64)
    _close_rope(got[:, None], flat[:, None], pos, inv, layout, 64, False, 1.0)
    assert fi.apply_rope(big[:0], pos[:0], inv).shape == (0, 8, 200)


def test_rope_is_its_inverse_and_gradient():
    """The inverse turn is the transpose: checked as the gradient of the plain formula."""
    g = _gen(6)
    x = torch.randn((12, 3, 96), generator=g, device="cuda", dtype=torch.float32)
    dy = torch.randn((12, 3, 96), generator=g, device="cuda", dtype=torch.float32)
    pos = torch.arange(12, device="cuda", dtype=I32) * 977
    inv = fi.rope_frequencies(64)
    leaf = x.double().requires_grad_()
    y, _ = (lambda v: _rope64_autograd(v, pos, inv, 16, 1.3))(leaf)
    y.backward(dy.double())
    got = fi.apply_rope(dy, pos, inv, layout="half", offset=16, inverse=True, scale=1.3)
    # |a| + |b| of two normal values stays below 12; 7e-7 of it as above
    assert (got.double() - leaf.grad).abs().max() <= 1.3 * 12 * 7e-7 + 12 * 2 ** -24
    back = fi.apply_rope(fi.apply_rope(x, pos, inv), pos, inv, inverse=True)
    assert (back - x).abs().max() <= 2 * 12 * 7e-7


def _rope64_autograd(v, pos, inv, offset, scale):
    ang = pos.double()[:, None, None] * inv
    c, s = torch.cos(ang), torch.sin(ang)
    r = 2 * inv.numel()
    a, b = v[..., offset:offset + r].chunk(2, -1)
    y = torch.cat((v[..., :offset], (a * c - b * s) * scale, (b * c + a * s) * scale, v[..., offset + r:]), -1)
    return y, None


# ------------------------------------------------------ latent cache writer
def _append64(kv, w, pos, inv, layout, eps, scale):
    x = kv.double()
    c = x[:, :DC] * torch.rsqrt(x[:, :DC].pow(2).mean(-1, keepdim=True) + eps) * w.double()
    e, mag = _rope64(kv[:, None, DC:], pos, inv, layout, 0, False, scale)
    return c, e[:, 0], mag[:, 0]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("tokens,layout", [(1, "interleaved"), (7, "half"), (64, "interleaved"), (1003, "half")])
def test_append(tokens, layout, dtype):
    g = _gen(tokens)
    wide = torch.randn((tokens, 600), generator=g, device="cuda").to(dtype)
    for kv in (wide[:, 24:], wide[:, 5:581], wide[:, :576].contiguous()):  # aligned, not aligned, dense
        kv = kv[:, :576]
        w = (1 + torch.randn(DC, generator=g, device="cuda") * 0.1).to(dtype)
        pages = tokens // PAGE + 3
        both = torch.randn((pages, PAGE, 576), generator=g, device="cuda").to(torch.bfloat16)
        ckv, kpe = both[..., :DC], both[..., DC:]  # one buffer for both: strided rows
        slots = torch.randperm(pages * PAGE, generator=g, device="cuda")[:tokens].to(I32)
        if tokens > 5:
            slots[4] = -1
        pos = torch.randint(0, 1 << 20, (tokens,), generator=g, device="cuda", dtype=I32)
        inv = fi.rope_frequencies(DP, scaling="linear", factor=2.0)
        before = both.clone()
        err = torch.zeros(1, dtype=I32, device="cuda")
        if tokens > 5:
            kv[3, :DC] = 0  # an all-zero latent: eps alone
        fi.latent_cache_append(kv, w, pos, slots, inv, ckv, kpe, eps=1e-5, layout=layout, rope_scale=1.1,
                               device_error=err)
        c, e, mag = _append64(kv, w, pos, inv, layout, 1e-5, 1.1)
        live = slots >= 0
        at = slots[live].long()
        got_c, got_e = ckv.reshape(-1, DC)[at].double(), kpe.reshape(-1, DP)[at].double()
        # bf16 rounding; in 32 bits the sum of 512 squares (21 additions deep), root, two products: below 32 * 2^-24
        assert ((got_c - c[live]).abs() <= (2 ** -8 + 2e-6) * c[live].abs() + 1e-38).all()
        assert ((got_e - e[live]).abs() <= 2 ** -8 * e[live].abs() + 7e-7 * mag[live] + 1e-38).all()
        rest = torch.ones(pages * PAGE, dtype=torch.bool, device="cuda")
        rest[at] = False
        assert torch.equal(both.view(-1, 576)[rest], before.view(-1, 576)[rest])  # other rows as they were
        assert err.item() == 0


def test_ids_past_32_bits_are_flagged_not_wrapped():
    kv = torch.ones((2, 576), device="cuda", dtype=torch.bfloat16)
    ckv = torch.zeros((2, PAGE, DC), device="cuda", dtype=torch.bfloat16)
    kpe = torch.zeros((2, PAGE, DP), device="cuda", dtype=torch.bfloat16)
    err = torch.zeros(1, dtype=I32, device="cuda")
    fi.latent_cache_append(kv, torch.ones(DC, device="cuda"), _put([0, 0], torch.int64),
                           torch.tensor([1 << 32, -(1 << 40)], device="cuda"), fi.rope_frequencies(DP), ckv, kpe,
                           device_error=err)
    assert err.item() == 1 and ckv.count_nonzero().item() == 0
    table = torch.zeros((1, 2), dtype=I32, device="cuda")
    lay = fi.step_layout(_put([0]), _put([1]), table, torch.tensor([1 << 33], device="cuda"), 1, device_error=err.zero_())
    assert err.item() == 1 and lay.slots.tolist() == [-1]


def test_append_bad_slots_and_int64():
    kv = torch.ones((3, 576), device="cuda", dtype=torch.bfloat16)
    ckv = torch.zeros((2, PAGE, DC), device="cuda", dtype=torch.bfloat16)
    kpe = torch.zeros((2, PAGE, DP), device="cuda", dtype=torch.bfloat16)
    err = torch.zeros(1, dtype=I32, device="cuda")
    fi.latent_cache_append(kv, torch.ones(DC, device="cuda"), _put([0, 0, 0], torch.int64),
                           _put([128, 5, -2], torch.int64), fi.rope_frequencies(DP), ckv, kpe, device_error=err)
    assert err.item() == 1 and (ckv[0, 5] == 1).all() and (kpe[0, 5] == 1).all()
    assert ckv.count_nonzero().item() == DC and kpe.count_nonzero().item() == DP


# --------------------------------------------------- shared-prefix attention
def _case(seed, tokens, heads, prefix, lens, per=1, max_prefix=None, stale=0.0, pages_extra=3):
    """Shuffled pages; the rows behind each length hold `stale`."""
    g, host = _gen(seed), np.random.default_rng(seed)
    lens = np.asarray(lens, np.int64)
    first = -(-(max_prefix if max_prefix is not None else prefix) // PAGE)
    requests = tokens // per
    own = -(-lens.reshape(requests, per).max(1) // PAGE)
    pages = host.permutation(first + int(own.sum()) + pages_extra)
    table = np.zeros((requests, max(1, int(own.max(initial=0)) + 1)), np.int64)
    table[np.arange(table.shape[1])[None, :] < own[:, None]] = pages[first:first + int(own.sum())]
    mk = lambda *s: torch.randn(s, generator=g, device="cuda")  # noqa: E731
    ckv = (mk(len(pages), PAGE, DC) * 0.5).to(torch.bfloat16)
    kpe = (mk(len(pages), PAGE, DP) * 0.5).to(torch.bfloat16)
    used = torch.zeros(len(pages) * PAGE, dtype=torch.bool, device="cuda")
    rows = np.arange(prefix)
    used[_put(pages[:first][rows // PAGE] * PAGE + rows % PAGE, torch.int64)] = True
    for r in range(requests):
        rows = np.arange(lens.reshape(requests, per)[r].max())
        used[_put(table[r][rows // PAGE] * PAGE + rows % PAGE, torch.int64)] = True
    ckv.view(-1, DC)[~used] = stale
    kpe.view(-1, DP)[~used] = stale
    return dict(qn=mk(tokens, heads, DC).to(torch.bfloat16), qp=mk(tokens, heads, DP).to(torch.bfloat16), ckv=ckv,
                kpe=kpe, pages=_put(pages[:first]), prefix=_put([prefix]), table=_put(table), lens=_put(lens),
                request=_put(np.repeat(np.arange(requests), per)))


def _attend64(c, scale=SCALE):
    """(out, lse, sum p|v| / sum p, sum |q||k| * scale) in 64 bits, one token after the other."""
    ckv, kpe = c["ckv"].reshape(-1, DC).double(), c["kpe"].reshape(-1, DP).double()
    col = torch.arange(PAGE, device="cuda")
    pre = (c["pages"].long()[:, None] * PAGE + col).flatten()[:c["prefix"].item()]
    out, lse, mag, dot = [], [], [], []
    for t in range(c["qn"].shape[0]):
        own = (c["table"][c["request"][t].item()].long()[:, None] * PAGE + col).flatten()[:c["lens"][t].item()]
        at = torch.cat((pre, own))
        k, e = ckv[at], kpe[at]
        z = (c["qn"][t].double() @ k.T + c["qp"][t].double() @ e.T) * scale
        p = torch.softmax(z, -1) if at.numel() else z
        out.append(p @ k)
        mag.append(p @ k.abs())
        lse.append(torch.logsumexp(z, -1) / math.log(2.0))
        d = c["qn"][t].double().abs() @ k.abs().T + c["qp"][t].double().abs() @ e.abs().T
        dot.append(d.amax(-1) * abs(scale) if at.numel() else torch.zeros(z.shape[0], device="cuda", dtype=torch.float64))
    return torch.stack(out), torch.stack(lse), torch.stack(mag), torch.stack(dot)


def _attend(c, scale=SCALE, **kw):
    return fi.shared_prefix_attention(c["qn"], c["qp"], c["ckv"], c["kpe"], c["pages"], c["prefix"], c["table"],
                                      c["lens"], scale, token_request=c["request"], **kw)


def _check_attention(c, got, scale=SCALE):
    out, lse, mag, dot = _attend64(c, scale)
    # scores: 576 products summed in 32 bits, at most 576 * 2^-24 of sum |q||k| (3.5e-5), and their scaling
    ds = 3.6e-5 * dot
    # weights to bf16 for the matrix product (2^-8 each), the scores' errors (numerator and sum), exponentials and
    # sums in 32 bits (1e-5), one rounding of the output
    tol = 2 ** -8 * out.abs() + (2 ** -8 + 1e-5 + 2 * ds[..., None]) * (mag + out.abs()) + 1e-30
    assert got[0].isfinite().all()
    err = (got[0].double() - out).abs()
    assert (err <= tol).all(), (err - tol).max()
    assert torch.equal(torch.isneginf(got[1]), torch.isneginf(lse))
    fin = ~torch.isneginf(lse)
    # the sum of up to 2^18 terms in 32 bits, split and joined: 1e-5; lse itself to 32 bits
    tol = (ds + 1e-5) / math.log(2.0) + lse.abs() * 2 ** -22
    assert ((got[1].double() - lse).abs()[fin] <= tol[fin]).all()


@pytest.mark.parametrize("tokens,heads,prefix,lens,per", [
    (1, 16, 1, [0], 1), (1, 16, 0, [1], 1), (1, 16, 64, [64], 1), (1, 16, 65, [63], 1), (1, 128, 127, [129], 1),
    (3, 16, 0, [0, 5, 200], 1), (3, 16, 130, [0, 0, 0], 1), (2, 16, 5000, [1, 700], 1), (8, 16, 1000, [1, 2, 3, 64, 65, 128, 129, 500], 1),
    (9, 16, 300, [7] * 9, 1), (5, 48, 200, [0, 100, 64, 1, 333], 1), (7, 32, 129, [0, 1, 2, 3, 400, 5, 6], 1),
    (3, 144, 100, [65, 0, 1], 1), (6, 64, 77, [5, 6, 64, 65, 200, 201], 2), (12, 16, 640, [10, 11, 12, 63, 64, 65, 0, 1, 2, 127, 128, 129], 3),
    (70, 16, 513, [i * 3 % 200 for i in range(70)], 1), (33, 128, 257, [i * 5 % 90 for i in range(33)], 1)])
def test_prefix_attention(tokens, heads, prefix, lens, per):
    c = _case(tokens + heads + prefix, tokens, heads, prefix, lens, per)
    _check_attention(c, _attend(c))
    assert fi.read_prefix_error() == 0


def test_prefix_long_and_batched():
    """Row blocks split over many CTAs and CTAs that work on several row blocks."""
    for tokens, heads, prefix, own in ((2, 16, 40000, 3000), (100, 16, 3000, 600), (24, 128, 1500, 300)):
        lens = np.random.default_rng(tokens).integers(0, own, tokens)
        c = _case(3, tokens, heads, prefix, lens)
        _check_attention(c, _attend(c))
    assert fi.read_prefix_error() == 0


def _runs_case(seed, heads, prefix, groups, order=None):
    """Requests with several tokens each: groups = [[lengths of the tokens of request 0], ...]."""
    lens = [n for g in groups for n in g]
    request = [r for r, g in enumerate(groups) for _ in g]
    host = np.random.default_rng(seed)
    c = _case(seed, len(groups), heads, prefix, [max(g) for g in groups])
    g = _gen(seed + 1)
    order = list(range(len(lens))) if order is None else host.permutation(len(lens)).tolist()
    c["lens"], c["request"] = _put(np.array(lens)[order]), _put(np.array(request)[order])
    c["qn"] = torch.randn((len(lens), heads, DC), generator=g, device="cuda").to(torch.bfloat16)
    c["qp"] = torch.randn((len(lens), heads, DP), generator=g, device="cuda").to(torch.bfloat16)
    return c


@pytest.mark.parametrize("heads,groups,order", [
    (16, [[300, 301, 302, 303, 304, 305, 306, 307, 308, 309]], None), (16, [[5, 6, 7], [190, 191, 192, 193, 194], [64, 128]], None),
    (16, [[128, 0, 129, 64, 63, 1, 65]], None), (32, [[700, 701, 702], [63, 64, 65, 66]], None), (48, [[130, 131], [1], [257, 256]], None),
    (128, [[100, 101, 102], [0, 0], [64]], None), (16, [[500, 501, 502], [100, 101], [64, 65, 66, 67]], "mixed")])
def test_prefix_tokens_of_one_request(heads, groups, order):
    """Tokens of a request side by side share its pages, each up to its own length."""
    for prefix in (0, 100):
        c = _runs_case(21, heads, prefix, groups, order)
        _check_attention(c, _attend(c))
    assert fi.read_prefix_error() == 0


def test_prefix_later_rows_of_the_same_request_are_not_seen():
    """Rows that a later token of the request sees hold NaN: the earlier tokens' outputs stay as they are."""
    c = _runs_case(22, 16, 70, [[125, 126, 127, 128, 129, 200]])
    want = _attend(c)
    for row in (125, 128, 150):
        d = {k: v.clone() for k, v in c.items()}
        d["ckv"][d["table"][0, row // PAGE], row % PAGE] = float("nan")
        out, lse = _attend(d)
        sees = d["lens"] > row
        assert torch.equal(out[~sees], want[0][~sees]) and torch.equal(lse[~sees], want[1][~sees])
        assert out[sees].isnan().all() and lse[sees].isnan().all()


def test_prefix_many_row_blocks():
    """More row blocks than threads of a CTA, most of them finished by one pair."""
    lens = np.random.default_rng(5).integers(0, 150, 4200)
    c = _case(23, 4200, 16, 90, lens)
    _check_attention(c, _attend(c))
    c = _case(24, 600, 128, 65, lens[:600] // 4)
    _check_attention(c, _attend(c))


@pytest.mark.parametrize("stale", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_prefix_rows_behind_a_length_are_not_read(stale):
    c = _case(11, 10, 16, 100, [0, 1, 63, 64, 65, 100, 5, 7, 190, 2], stale=stale)
    _check_attention(c, _attend(c))


def test_prefix_requests_do_not_disturb_each_other():
    """A request whose own rows hold NaN and infinities spoils its own outputs alone."""
    c = _case(12, 9, 16, 200, [10, 70, 3, 130, 9, 64, 1, 5, 80])
    page = c["table"][3, 0].item()
    c["ckv"][page, 5, 100], c["ckv"][page, 9, 3], c["kpe"][page, 7, 2] = float("nan"), float("inf"), -float("inf")
    out, lse = _attend(c)
    assert out[3].isnan().any()
    keep = torch.tensor([t for t in range(9) if t != 3], device="cuda")
    c["ckv"][page, 5, 100], c["ckv"][page, 9, 3], c["kpe"][page, 7, 2] = 0, 0, 0
    want, wlse = _attend(c)
    assert torch.equal(out[keep], want[keep]) and torch.equal(lse[keep], wlse[keep])


def test_prefix_extreme_scores():
    """Scores in the thousands, of one sign and of both, and all equal: the maximum is taken out."""
    for scale in (8.0, -8.0, 0.0):
        c = _case(13, 4, 16, 500, [3, 64, 100, 0])
        _check_attention(c, _attend(c, scale), scale)


def test_prefix_rising_maximum():
    """The largest score comes last and is far above the others: everything before it is rescaled."""
    c = _case(14, 2, 16, 700, [300, 130])
    c["qn"].fill_(0.25)
    c["qp"].zero_()
    rows = torch.linspace(-2, 2, 700, device="cuda").to(torch.bfloat16)
    at = (c["pages"].long()[:, None] * PAGE + torch.arange(PAGE, device="cuda")).flatten()[:700]
    c["ckv"].view(-1, DC)[at] += rows[:, None]
    _check_attention(c, _attend(c, 1.0), 1.0)


def test_prefix_strides_and_outputs():
    """Queries out of a wider projection, both caches in one buffer, permuted requests, given outputs, 64-bit ids."""
    c = _case(15, 6, 32, 150, [9, 64, 100, 3, 0, 77])
    wide = torch.randn((6, 40, 600), device="cuda").to(torch.bfloat16)
    wide[:, 4:36, 8:584] = torch.cat((c["qn"], c["qp"]), -1)
    both = torch.cat((c["ckv"], c["kpe"]), -1)
    perm = _put([5, 3, 1, 0, 2, 4], torch.int64)
    out = torch.zeros((6, 32, 600), device="cuda", dtype=torch.bfloat16)
    lse = torch.zeros((6, 33), device="cuda")
    table = torch.zeros_like(c["table"])
    table[perm] = c["table"]
    got = fi.shared_prefix_attention(wide[:, 4:36, 8:520], wide[:, 4:36, 520:584], both[..., :DC], both[..., DC:],
                                     c["pages"].long(), 150, table.long(), c["lens"].long(), SCALE,
                                     token_request=perm, output=out[..., 16:528], lse=lse[:, :32])
    _check_attention(c, got)
    assert (out[..., :16] == 0).all() and (out[..., 528:] == 0).all() and (lse[:, 32] == 0).all()


def test_prefix_length_on_the_device():
    """A shorter length on the device than the page list allows, zero and past the list (cut to it)."""
    for prefix in (0, 1, 100, 192):
        c = _case(16, 3, 16, prefix, [5, 0, 70], max_prefix=192)
        _check_attention(c, _attend(c))
    c["prefix"].fill_(10 ** 6)
    got = _attend(c)
    c["prefix"].fill_(192)
    assert torch.equal(got[0], _attend(c)[0])


def test_prefix_bad_ids_are_skipped_and_flagged():
    c = _case(17, 4, 16, 200, [70, 5, 130, 9])
    for row, what in ((0, "table"), (2, "request"), (1, "lens")):
        d = {k: v.clone() for k, v in c.items()}
        if what == "table":
            d["table"][row, 1] = 10 ** 7
        elif what == "request":
            d["request"][row] = 77
        else:
            d["lens"][row] = 64 * d["table"].shape[1] + 1
        out, lse = _attend(d)
        assert fi.read_prefix_error() == 1 and fi.read_prefix_error() == 0
        keep = [t for t in range(4) if t != row]
        _check_attention({**c, **{k: c[k][keep] for k in ("qn", "qp", "lens", "request")}}, (out[keep], lse[keep]))
        assert out.isfinite().all()
        if what == "table":  # the rows of the good page stay
            d["lens"][row] = 64
            assert torch.allclose(out[row].float(), _attend(d)[0][row].float(), atol=0.02)
            assert fi.read_prefix_error() == 0
    c["pages"][1] = -1
    assert _attend(c)[0].isfinite().all() and fi.read_prefix_error() == 1


def test_prefix_repeats_bit_for_bit_and_private_workspace():
    c = _case(18, 40, 16, 2000, np.arange(40) * 7)
    a = _attend(c)
    for _ in range(3):
        b = _attend(c)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    ws = torch.zeros(fi.prefix_workspace_size(40, 16), dtype=torch.uint8, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # beside a call on another stream
        b = _attend(c, workspace=ws)
    d = _attend(c)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a[0], b[0]) and torch.equal(a[0], d[0])
    with pytest.raises(Exception, match="workspace"):
        _attend(c, workspace=ws[:128])


def test_wrappers_refuse_on_the_gpu():
    c = _case(20, 2, 16, 10, [3, 4])
    with pytest.raises(RuntimeError, match="CUDA"):
        _attend({**c, "pages": c["pages"].cpu()})
    with pytest.raises(AssertionError):
        _attend({**c, "qn": c["qn"].half()})
    with pytest.raises(AssertionError):
        fi.shared_prefix_attention(c["qn"], c["qp"], c["ckv"], c["kpe"], c["pages"], 65, c["table"], c["lens"], SCALE)
    with pytest.raises(AssertionError):
        fi.apply_rope(c["qp"], _put([1]), fi.rope_frequencies(64))
    x = torch.zeros((2, 4, 64), device="cuda")
    with pytest.raises(AssertionError):
        fi.apply_rope(x, _put([1, 2]), fi.rope_frequencies(64), out=x.as_strided((2, 4, 64), (64, 128, 1)))
    with pytest.raises(AssertionError):
        fi.apply_rope(x, _put([1, 2]), fi.rope_frequencies(64), out=torch.zeros((2, 1, 64), device="cuda").expand(2, 4, 64))
    with pytest.raises(AssertionError):
        fi.step_layout(_put([1]), _put([1]), torch.zeros((1, 2), dtype=I32, device="cuda"), _put([1]), 1, prefix_len=3)
    with pytest.raises(RuntimeError, match="capture"):
        graph = torch.cuda.CUDAGraph()
        big = torch.zeros((1 << 15, 16, 512), dtype=torch.bfloat16, device="cuda")
        fi.prefix._workspaces.pop(0, None)  # as in a process whose first call is the captured one
        with torch.cuda.graph(graph):
            fi.shared_prefix_attention(big, big[..., :64], c["ckv"], c["kpe"], c["pages"], 10, c["table"],
                                       torch.zeros(1 << 15, dtype=I32, device="cuda"), SCALE,
                                       token_request=torch.zeros(1 << 15, dtype=I32, device="cuda"))


# ------------------------------------------------------------ all together
def _step_inputs(seed, batch, q, seq, prefix, heads=16, capacity=None):
    g, host = _gen(seed), np.random.default_rng(seed)
    tokens = capacity if capacity is not None else int(np.sum(q))
    first, width = -(-prefix // PAGE), 8
    have = -(-np.asarray(seq) // PAGE)
    pages = host.permutation(first + batch * width)
    table = np.zeros((batch, width), np.int64)
    table[np.arange(width)[None, :] < have[:, None]] = pages[first:first + have.sum()]
    mk = lambda *s: torch.randn(s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    return dict(q_nope=mk(tokens, heads, DC), q_pe=mk(tokens, heads, DP), kv=mk(tokens, 576),
                norm_weight=mk(DC), inv_freq=fi.rope_frequencies(DP, scaling="yarn", factor=40.0),
                ckv_cache=mk(len(pages), PAGE, DC) * 0.5, kpe_cache=mk(len(pages), PAGE, DP) * 0.5,
                seq_lens=_put(seq), query_lens=_put(q), block_table=_put(table),
                free_pages=_put(pages[first + have.sum():]), prefix_pages=_put(pages[:first]),
                prefix_len=_put([prefix]), sm_scale=SCALE)


def _step_oracle(a, lay):
    """The step from its inputs in 64 bits up to the caches and queries, which are then rounded to bf16."""
    ckv, kpe = a["ckv_cache"].clone(), a["kpe_cache"].clone()
    c, e, _ = _append64(a["kv"], a["norm_weight"], lay.positions, a["inv_freq"], "interleaved", 1e-6, 1.0)
    live = lay.slots >= 0
    ckv.view(-1, DC)[lay.slots[live].long()] = c[live].to(torch.bfloat16)
    kpe.view(-1, DP)[lay.slots[live].long()] = e[live].to(torch.bfloat16)
    qp = _rope64(a["q_pe"], lay.positions, a["inv_freq"], "interleaved", 0, False, 1.0)[0].to(torch.bfloat16)
    return dict(qn=a["q_nope"], qp=qp, ckv=ckv, kpe=kpe, pages=a["prefix_pages"], prefix=a["prefix_len"],
                table=a["block_table"], lens=lay.token_lens, request=lay.token_request)


def _close_step(c, out, lse):
    """As _check_attention, with the caches and turned queries one bf16 step apart at worst where the 32- and 64-bit
    values round to different sides: a share of 2^-7 of the values and of the scores' few largest terms."""
    want, wlse, mag, dot = _attend64(c)
    assert ((out.double() - want).abs() <= 2 ** -8 * want.abs() + (2 ** -7 + 1e-2) * (mag + want.abs())).all()
    assert ((lse.double() - wlse).abs() <= 1e-3 * (1 + dot)).all()


def test_step_decode_and_chunks():
    a = _step_inputs(30, 5, [1, 3, 0, 70, 1], [63, 64, 5, 10, 0], 300)
    out, lse, lay = run_shared_prefix_step(**a)
    assert lay.token_lens.tolist() == [64, 65, 66, 67] + list(range(11, 81)) + [1]
    _close_step(_step_oracle(a, lay), out, lse)
    # a second step on top of the first
    b = _step_inputs(31, 5, [1] * 5, [64, 67, 5, 80, 1], 300)
    for k in ("ckv_cache", "kpe_cache", "block_table", "prefix_pages"):
        b[k] = a[k]
    b["free_pages"] = a["free_pages"][lay.pages_used.item():]
    out, lse, lay = run_shared_prefix_step(**b)
    _close_step(_step_oracle(b, lay), out, lse)


def test_step_captured_follows_lengths():
    """One captured step replayed with other lengths, tokens and prefix; the padded rows see the prefix alone."""
    a = _step_inputs(32, 4, [1, 1, 1, 1], [10, 63, 64, 130], 500, capacity=8)
    a["prefix_len"].fill_(500)
    run_shared_prefix_step(**a)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, lse, lay = run_shared_prefix_step(**a)
    for seq, q, prefix in (([10, 63, 64, 130], [1, 1, 1, 1], 500), ([11, 60, 65, 100], [2, 0, 5, 1], 449),
                           ([0, 0, 0, 0], [0, 1, 0, 0], 1)):
        a["seq_lens"].copy_(_put(seq))
        a["query_lens"].copy_(_put(q))
        a["prefix_len"].fill_(prefix)
        a["q_nope"].normal_(generator=_gen(sum(q)))
        graph.replay()
        torch.cuda.synchronize()
        assert lay.token_lens[sum(q):].tolist() == [0] * (8 - sum(q))
        eager = run_shared_prefix_step(**a)
        assert torch.equal(out, eager[0]) and torch.equal(lse, eager[1])
        _close_step(_step_oracle(a, lay), out, lse)
    assert fi.read_prefix_error() == 0


# ------------------------------------------------- offsets past 32 bits, last:
# its gigabytes stay in torch's cache, from which the next module's test of free
# device memory takes its own temporaries (a graph capture empties that cache)
def test_prefix_far_pages():
    """Cache offsets past 2^31 elements and 2^32 bytes."""
    pages = 70000
    ckv = torch.empty((pages, PAGE, DC), dtype=torch.bfloat16, device="cuda")
    kpe = torch.empty((pages, PAGE, DP), dtype=torch.bfloat16, device="cuda")
    c = _case(19, 3, 16, 130, [70, 5, 64])
    n = c["ckv"].shape[0]
    ckv[pages - n:], kpe[pages - n:] = c["ckv"], c["kpe"]
    got = fi.shared_prefix_attention(c["qn"], c["qp"], ckv, kpe, c["pages"] + (pages - n), c["prefix"],
                                     c["table"] + (pages - n), c["lens"], SCALE)
    _check_attention(c, got)
    # and the writer: the last row of the cache
    kv = torch.randn((1, 576), device="cuda").to(torch.bfloat16)
    w = torch.ones(DC, device="cuda")
    fi.latent_cache_append(kv, w, _put([3]), _put([pages * PAGE - 1]), fi.rope_frequencies(DP), ckv, kpe)
    e = _append64(kv, w, _put([3]), fi.rope_frequencies(DP), "interleaved", 1e-6, 1.0)[0]
    assert ((ckv[-1, -1].double() - e[0]).abs() <= (2 ** -8 + 2e-6) * e[0].abs()).all()
