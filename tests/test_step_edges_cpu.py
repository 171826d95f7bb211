"""Refusals of the serving-step operators at their edges, without a GPU."""
from __future__ import annotations

import pytest

from flashinfer_repo_b200 import _lib

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
X = 4096  # an aligned non-NULL address that is never read


def _scratch(q=X, table=X, tokens=1, heads=16, out=X, ws=X, err=None):
    return _lib.load().dsa_shared_prefix_attention_scratch(
        q, 16 * 512, 512, q, 16 * 64, 64, X, 64 * 512, 512, X, 64 * 64, 64, X, 64, None, table, 4, 4, 4, None, X, tokens,
        heads, 8, 0.1, out, 16 * 512, 512, out, 16, 1, ws, 1 << 40, err, None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(q=X + 8), dict(table=None), dict(tokens=-1), dict(heads=24),
                                dict(out=None), dict(ws=None)])
def test_scratch_entry_refuses(kw):
    assert _scratch(**kw) == INVALID


def test_scratch_entry_takes_no_error_word():
    assert _scratch(tokens=0) == 0
