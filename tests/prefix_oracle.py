"""Shared-prefix attention in 64 bits with a tolerance that shrinks as rows are added.

The weights are rounded to bf16 for the matrix product, each by at most 2^-8 of
itself and independently of the others, so what they do to an output grows with
the root of the sum of squares of p v and not with the sum of p |v|: by
Hoeffding's inequality the error passes 8 * 2^-8 * sqrt(sum p^2 v^2) with a
probability below 2 exp(-32) = 3e-14.  (For few rows the plain sum is smaller.)"""
from __future__ import annotations

import math

import torch

PAGE, DC, DP = 64, 512, 64


def rows_of(case, t):
    """Flat cache rows that token t sees, in list order."""
    device = case["ckv"].device
    col = torch.arange(PAGE, device=device)
    pre = (case["pages"].long()[:, None] * PAGE + col).flatten()[:int(case["prefix"].item())]
    own = (case["table"][case["request"][t].item()].long()[:, None] * PAGE + col).flatten()[:case["lens"][t].item()]
    return torch.cat((pre, own))


def attend64(case, scale, tokens=None, values=None):
    """(out, lse base 2, tolerance of out, tolerance of lse) of the given tokens, one after the other.
    values: cache rows whose values are taken in place of those seen (to plant a mistake), as a function of them."""
    ckv, kpe = case["ckv"].reshape(-1, DC), case["kpe"].reshape(-1, DP)
    results = []
    for t in range(case["qn"].shape[0]) if tokens is None else tokens:
        at = rows_of(case, t)
        qn, qp = case["qn"][t].double(), case["qp"][t].double()
        if at.numel() == 0:
            zero = torch.zeros_like(qn)
            results.append((zero, torch.full_like(zero[:, 0], -math.inf), zero, zero[:, 0]))
            continue
        k, e = ckv[at].double(), kpe[at].double()
        v = k if values is None else ckv[values(at)].double()
        z = (qn @ k.T + qp @ e.T) * scale
        p = torch.softmax(z, -1)
        # scores: 576 products summed in 32 bits, at most 576 * 2^-24 of sum |q||k| (3.5e-5), and their scaling
        ds = 3.6e-5 * (qn.abs() @ k.abs().T + qp.abs() @ e.abs().T) * abs(scale)
        out, mag = p @ v, p @ v.abs()
        rt = (p.square() @ v.square()).sqrt()
        # what each weight can be off by: its rounding, its score's error and that of the sum it is divided by
        w = p * (2 ** -8 + 2 * ds)
        linear = w @ v.abs() + w.sum(-1, keepdim=True) * out.abs()
        root = 8 * ((w.square() @ v.square()).sqrt() + w.square().sum(-1, keepdim=True).sqrt() * out.abs())
        # one rounding of the output; the weights; exponentials and sums in 32 bits (1e-5) and n / 16 additions to
        # the accumulator of a value that stays below |out| + 8 rt, 2^-23 of it each
        tol = (2 ** -8 * out.abs() + torch.minimum(linear, root) + 1e-5 * (mag + out.abs()) +
               at.numel() * 2 ** -27 * (out.abs() + 8 * rt) + 1e-30)
        lse = torch.logsumexp(z, -1) / math.log(2.0)
        # the scores' errors; the sum of the weights in 32 bits, split and joined (1e-5); lse itself in 32 bits
        results.append((out, lse, tol, ((p * ds).sum(-1) + 1e-5) / math.log(2.0) + lse.abs() * 2 ** -22))
    return tuple(torch.stack(r) for r in zip(*results))


def check(case, got, scale, tokens=None):
    out, lse, tol, ltol = attend64(case, scale, tokens)
    if tokens is not None:
        got = got[0][list(tokens)], got[1][list(tokens)]
    assert got[0].isfinite().all()
    err = (got[0].double() - out).abs()
    assert (err <= tol).all(), ((err / tol).max().item(), (err > tol).sum().item())
    assert torch.equal(torch.isneginf(got[1]), torch.isneginf(lse))
    fin = ~torch.isneginf(lse)
    assert ((got[1].double() - lse).abs()[fin] <= ltol[fin]).all()
    return (err / tol).max().item()


def make_case(seed, tokens, heads, prefix, lens, per=1, device="cuda"):
    """Shuffled pages, random rows; lens are the tokens' own rows, `per` tokens a request."""
    gen = torch.Generator(device=device).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    lens = torch.as_tensor(lens, dtype=torch.int64)
    requests, first = tokens // per, -(-prefix // PAGE)
    own = (lens.reshape(requests, per).amax(1) + PAGE - 1) // PAGE
    pages = torch.randperm(first + int(own.sum()) + 2, generator=host)
    table = torch.zeros((requests, int(own.max()) + 1), dtype=torch.int64)
    table[torch.arange(table.shape[1])[None, :] < own[:, None]] = pages[first:first + int(own.sum())]
    mk = lambda *s: torch.randn(s, generator=gen, device=device)  # noqa: E731
    put = lambda v: v.to(device, torch.int32)  # noqa: E731
    return dict(qn=mk(tokens, heads, DC).to(torch.bfloat16), qp=mk(tokens, heads, DP).to(torch.bfloat16),
                ckv=(mk(len(pages), PAGE, DC) * 0.5).to(torch.bfloat16), kpe=(mk(len(pages), PAGE, DP) * 0.5).to(torch.bfloat16),
                pages=put(pages[:first]), prefix=put(torch.tensor([prefix])), table=put(table), lens=put(lens),
                request=put(torch.arange(requests).repeat_interleave(per)))
