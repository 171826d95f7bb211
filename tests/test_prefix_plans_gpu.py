"""Shared-prefix attention over the plans: pairs of their own for each row block, the even cut of the line of all
tiles with fewer and with more row blocks than pairs, the numbers of row blocks at which planning and merging change.
The plan that a case is meant for is read back from its workspace."""
from __future__ import annotations

import math

import pytest
import torch

import flashinfer_repo_b200 as fi

from . import prefix_oracle as P

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192.0)
SLOT_BYTES = (2 * 64 * 512 + 4 * 64) * 4  # a partial: O, m and l of 128 rows


def _pairs():
    """Pairs of CTAs on the device: the workspace holds two partials for each."""
    return fi.prefix_workspace_size(1, 16) // (2 * SLOT_BYTES)


def _planned(c):
    """(result, tiles of each row block, pairs that each row block has of its own or 0) of a call."""
    tokens, heads = c["qn"].shape[:2]
    blocks = -(-tokens * (heads // 16) // 8)
    ws = torch.zeros(fi.prefix_workspace_size(tokens, heads), dtype=torch.uint8, device="cuda")
    got = fi.shared_prefix_attention(c["qn"], c["qp"], c["ckv"], c["kpe"], c["pages"], c["prefix"], c["table"], c["lens"],
                                     SCALE, token_request=c["request"], workspace=ws)
    plan = ws[256:256 + 8 * (blocks + 2)].view(torch.int64).tolist()
    assert ws[:4].view(torch.int32).item() == 0
    return got, [b - a for a, b in zip(plan[:blocks], plan[1:blocks + 1])], plan[-1]


@pytest.mark.parametrize("tokens,heads,per,prefix,own", [
    (256, 16, 2, 3000, 1500), (96, 16, 2, 1000, 900), (60, 48, 3, 700, 500), (30, 128, 1, 400, 3000)])
def test_even_cut_with_fewer_row_blocks_than_pairs(tokens, heads, per, prefix, own):
    """Ragged own parts: stretches begin inside row blocks, and most pairs work on two."""
    g = torch.Generator().manual_seed(tokens)
    lens = torch.randint(0, own, (tokens // per,), generator=g)[:, None] + 1 + torch.arange(per)
    lens[::7] = 0
    lens[-1] = own * 4  # one request far longer than the others: pairs of their own would wait for it
    c = P.make_case(tokens, tokens, heads, prefix, lens.flatten(), per)
    got, tiles, share = _planned(c)
    pairs = _pairs()
    assert share == 0 and len(tiles) < pairs
    each, starts, at = sum(tiles) / pairs, [], 0
    for n in tiles:
        starts.append(at)
        at += n
    # some row block begins inside a pair's stretch and reaches past it: the merge takes that pair's second partial
    assert any(s % each > 1 and n > each for s, n in zip(starts, tiles))
    P.check(c, got, SCALE)


@pytest.mark.parametrize("extra", [-8, -1, 0, 1, 5, 76])
def test_row_blocks_around_the_number_of_pairs(extra):
    """One row block a token (128 heads): a warp or the CTA plans, row blocks or cuts are merged, pairs have one or more."""
    blocks = _pairs() + extra
    for prefix, lens in ((300, [i * 37 % 400 for i in range(blocks)]), (129, [0] * blocks)):
        c = P.make_case(blocks, blocks, 128, prefix, lens)
        got, tiles, share = _planned(c)
        assert len(tiles) == blocks
        P.check(c, got, SCALE)


@pytest.mark.parametrize("blocks", [63, 64, 65])
def test_row_blocks_around_what_a_warp_plans_alone(blocks):
    c = P.make_case(blocks, blocks, 128, 500, [i * 11 % 150 for i in range(blocks)])
    got, tiles, _ = _planned(c)
    assert len(tiles) == blocks
    P.check(c, got, SCALE)
    c = P.make_case(blocks, blocks * 8 - 3, 16, 200, [i * 29 % 260 for i in range(blocks * 8 - 3)])
    got, tiles, _ = _planned(c)
    assert len(tiles) == blocks
    P.check(c, got, SCALE, range(0, blocks * 8 - 3, 3))


@pytest.mark.parametrize("tokens,heads,prefix", [(8, 16, 9000), (32, 16, 9000), (40, 16, 9000), (200, 16, 9000), (288, 16, 6000)])
def test_equal_row_blocks(tokens, heads, prefix):
    """From all pairs on one row block to two each: every variant of the merge.  Row blocks have pairs of their own
    unless too many pairs would stay idle (25 row blocks of 74 pairs: 24)."""
    c = P.make_case(tokens, tokens, heads, prefix, [i * 13 % 65 for i in range(tokens)])
    got, tiles, share = _planned(c)
    each, own = sum(tiles) / _pairs(), _pairs() // len(tiles)
    if max(tiles) <= each * own:
        assert share == own > 0
    elif max(tiles) > (math.ceil(each) + 3) * own:  # what a second row block costs a pair: three tiles
        assert share == 0
    P.check(c, got, SCALE, range(0, tokens, 1 + tokens // 40))


@pytest.mark.parametrize("prefix,own", [(64, 64), (130, 62), (320, 64), (321, 64), (385, 1)])
def test_around_what_one_pair_takes_whole(prefix, own):
    """Up to three tiles a row block: no partials and no merge grid; one more and the list is split."""
    for tokens in (1, 5, 64):
        c = P.make_case(tokens + prefix, tokens, 128, prefix, [own] * tokens)
        c["table"] = c["table"][:, :-(-own // 64)].contiguous()  # no room for more: the host's bound is the list itself
        got = _planned(c)[0]
        P.check(c, got, SCALE, range(0, tokens, 7))


def test_prompt_chunk_behind_a_prefix():
    """Hundreds of tokens of one request, each seeing the rows before it."""
    n, before = 500, 77
    c = P.make_case(9, 1, 16, 2000, [before + n])
    c["lens"] = torch.arange(before + 1, before + n + 1, device="cuda", dtype=torch.int32)
    c["request"] = torch.zeros(n, dtype=torch.int32, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(10)
    c["qn"] = torch.randn((n, 16, 512), generator=g, device="cuda").to(torch.bfloat16)
    c["qp"] = torch.randn((n, 16, 64), generator=g, device="cuda").to(torch.bfloat16)
    got, tiles, _ = _planned(c)
    # eight tokens a row block: the pages that all of them see, and a page or two more for each
    assert max(tiles) <= (2000 + before + n) // 128 + 2 + 8
    P.check(c, got, SCALE, range(0, n, 9))
