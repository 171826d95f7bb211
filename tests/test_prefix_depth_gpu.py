"""Shared-prefix attention where a pair of CTAs walks many tiles and rescales what it has: long stretches of one
row block, maxima that rise along them, the cuts of the plan.  Against 64 bits, with the tolerance of prefix_oracle."""
from __future__ import annotations

import math

import pytest
import torch

import flashinfer_repo_b200 as fi

from . import prefix_oracle as P

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192.0)
SLOT_BYTES = (2 * 64 * 512 + 4 * 64) * 4  # a partial: O, m and l of 128 rows


def _attend(c, scale=SCALE, **kw):
    return fi.shared_prefix_attention(c["qn"], c["qp"], c["ckv"], c["kpe"], c["pages"], c["prefix"], c["table"], c["lens"],
                                      scale, token_request=c["request"], **kw)


def _pairs():
    """Pairs of CTAs on the device: the workspace holds two partials for each."""
    return fi.prefix_workspace_size(1, 16) // (2 * SLOT_BYTES)


def _planned(c, scale=SCALE):
    """(result, tiles of each row block, pairs that each row block has of its own or 0) of a call."""
    tokens, heads = c["qn"].shape[:2]
    blocks = -(-tokens * (heads // 16) // 8)
    ws = torch.zeros(fi.prefix_workspace_size(tokens, heads), dtype=torch.uint8, device="cuda")
    got = _attend(c, scale, workspace=ws)
    plan = ws[256:256 + 8 * (blocks + 2)].view(torch.int64).tolist()
    assert ws[:4].view(torch.int32).item() == 0
    return got, [b - a for a, b in zip(plan[:blocks], plan[1:blocks + 1])], plan[-1]


def test_many_tiles_a_stretch():
    """More than the 16 tiles whose page ids are looked up at once, and more than 40 partials of a row block."""
    c = P.make_case(1, 2, 16, 170001, [3000, 65])
    got, tiles, share = _planned(c)
    assert share == _pairs() and tiles[0] > 16 * share > 16 * 40
    P.check(c, got, SCALE)
    c = P.make_case(2, 80, 128, 4500, [i * 7 % 300 for i in range(80)])
    got, tiles, share = _planned(c)
    assert len(tiles) >= _pairs() and min(tiles) > 32
    P.check(c, got, SCALE, range(0, 80, 3))


def _slopes(c, values, where="prefix"):
    """Add values[i] to row i of the prefix, all latents alike; with queries of ones the scores follow them."""
    n = values.numel()
    col = torch.arange(P.PAGE, device="cuda")
    at = (c["pages"].long()[:, None] * P.PAGE + col).flatten()[:n]
    c["qn"].fill_(0.25)
    c["qp"].zero_()
    c["ckv"].view(-1, P.DC)[at] += values[:, None].to("cuda", torch.bfloat16)


@pytest.mark.parametrize("shape", ["rising", "falling", "steps", "spikes", "zigzag"])
def test_maximum_moves_along_a_stretch(shape):
    """Scores that move by hundreds along the 12 tiles of a pair: O in tensor memory is rescaled, by little and by all."""
    n = 1500
    i = torch.arange(n, dtype=torch.float32)
    values = {"rising": i / n * 3 - 1.5, "falling": 1.5 - i / n * 3, "steps": (i // 200) * 0.05,
              "spikes": torch.where(i % 377 == 376, i / n, torch.zeros(())), "zigzag": (i % 400) / 400 + i / n}[shape]
    c = P.make_case(3, 80, 128, n, [i % 70 for i in range(80)])
    _slopes(c, values)
    got, tiles, share = _planned(c, 0.3)
    assert share <= 1 and min(tiles) >= 12  # a row block is one pair's, or two cut it
    P.check(c, got, 0.3, range(0, 80, 5))


def test_maximum_rises_behind_a_prefix_that_is_all_masked_low():
    """Scores near -1e4 for the whole prefix, ordinary ones in the own rows: what came before weighs nothing."""
    c = P.make_case(4, 80, 128, 1300, [130] * 80)
    _slopes(c, torch.full((1300,), -100.0))
    got = _attend(c, 1.0)
    P.check(c, got, 1.0, range(0, 80, 5))
