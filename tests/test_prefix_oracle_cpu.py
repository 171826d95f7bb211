"""The tolerance of prefix_oracle sees what a mistake in the kernel's bookkeeping would do to an output."""
from __future__ import annotations

import math

import torch

from . import prefix_oracle as P

SCALE = 1 / math.sqrt(192.0)


def _case():
    return P.make_case(1, 1, 16, 20000, [100], device="cpu")


def _misses(c, values):
    out, _, tol, _ = P.attend64(c, SCALE)
    wrong = P.attend64(c, SCALE, values=values)[0]
    return ((wrong - out).abs() > tol).sum().item()


def test_honest_weights_pass():
    """Weights rounded to bf16, the sum of them as they are: a fraction of the tolerance."""
    c = _case()
    at = P.rows_of(c, 0)
    k, e = c["ckv"].reshape(-1, P.DC)[at].double(), c["kpe"].reshape(-1, P.DP)[at].double()
    z = (c["qn"][0].double() @ k.T + c["qp"][0].double() @ e.T) * SCALE
    w = torch.exp(z - z.amax(-1, keepdim=True))
    got = (w.to(torch.bfloat16).double() @ k / w.sum(-1, keepdim=True)).to(torch.bfloat16).double()
    out, _, tol, _ = P.attend64(c, SCALE)
    assert ((got - out[0]).abs() / tol[0]).max() < 0.6


def test_wrong_values_fail():
    """The values of a tile, of a page and of the rows behind a page's middle taken from elsewhere."""
    c = _case()
    for rows, first in ((128, 6400), (64, 640), (32, 19232)):
        def values(at):
            at = at.clone()
            at[first:first + rows] = at[:rows]
            return at
        assert _misses(c, values) > 0, rows
