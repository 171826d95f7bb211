"""The serving-step operators at their edges, without a GPU: refusals, the middle of the frequency ramp."""
from __future__ import annotations

import math

import pytest

import flashinfer_repo_b200 as fi
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


def test_yarn_ramp_pair_by_pair():
    """The share of the plain frequency falls along a line of the pair's number, from the pair that makes beta_fast
    turns over the original context (rounded down) to the one that makes beta_slow (rounded up)."""
    for rot, base, factor, context, fast, slow in ((64, 10000.0, 40.0, 4096, 32.0, 1.0), (128, 500000.0, 8.0, 8192, 32.0, 1.0),
                                                   (32, 10000.0, 4.0, 2048, 16.0, 2.0)):
        got = fi.rope_frequencies(rot, base, scaling="yarn", factor=factor, original_context=context, beta_fast=fast,
                                  beta_slow=slow, device="cpu").tolist()
        # turns over the context of the (fractional) pair i: context * base^(-2i/rot) / 2 pi
        at = [math.log(context / (2 * math.pi * turns), base) * rot / 2 for turns in (fast, slow)]
        first, last = math.floor(at[0]), math.ceil(at[1])
        assert 0 < first < last < rot // 2
        between = 0
        for i, f in enumerate(got):
            plain = base ** (-2 * i / rot)
            share = 1.0 if i <= first else 0.0 if i >= last else (last - i) / (last - first)
            between += 0 < share < 1
            assert math.isclose(f, plain * share + plain / factor * (1 - share), rel_tol=1e-13), (i, share)
        assert between >= 3  # the last of the three: pairs 6, 7 and 8 between 5 and 9
