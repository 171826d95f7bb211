"""Refusals of the serving-step operators that need no GPU: argument errors of
the C ABI come back as status codes before anything is launched, the Python
wrappers raise, and the frequency helper's scalings follow their formulas."""
from __future__ import annotations

import ctypes
import math

import pytest
import torch

import flashinfer_repo_b200 as fi
from flashinfer_repo_b200 import _lib

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 3
X = 4096  # an aligned non-NULL address that is never read


def _rc(name, *args):
    return getattr(_lib.load(), name)(*args)


def _layout(seq=X, query=X, batch=2, table=X, stride=4, pages=4, free=X, nfree=8, prefix=None, rows=2, out=X,
            used=X):
    return _rc("dsa_step_layout", seq, query, batch, table, stride, pages, free, nfree, prefix, rows, out, out, out,
               out, used, None, None)


@pytest.mark.parametrize("kw", [dict(batch=-1), dict(pages=-1), dict(nfree=-1), dict(rows=-1), dict(seq=None),
                                dict(query=None), dict(table=None), dict(free=None), dict(out=None),
                                dict(used=None), dict(stride=3)])
def test_step_layout_refuses(kw):
    assert _layout(**kw) == INVALID


def test_step_layout_counts_in_32_bits():
    assert _layout(rows=1 << 31) == UNSUPPORTED and _layout(batch=1 << 31) == UNSUPPORTED


def _rope(x=X, out=X, dtype=0, tokens=1, heads=1, dim=64, offset=0, rot=64, pos=X, freq=X, layout=0):
    return _rc("dsa_apply_rope", x, dim, dim, out, dim, dim, dtype, tokens, heads, dim, offset, rot, pos, 0, freq,
               layout, 0, 1.0, None)


@pytest.mark.parametrize("kw", [dict(x=None), dict(out=None), dict(pos=None), dict(freq=None), dict(dtype=3),
                                dict(layout=2), dict(offset=1), dict(offset=-1), dict(tokens=-1), dict(dim=32)])
def test_rope_refuses(kw):
    assert _rope(**kw) == INVALID


@pytest.mark.parametrize("kw", [dict(rot=7, dim=8), dict(rot=0), dict(rot=514, dim=600), dict(heads=1 << 20)])
def test_rope_unsupported(kw):
    assert _rope(**kw) == UNSUPPORTED


def test_empty_calls_do_nothing():
    assert _rope(tokens=0, x=None, out=None, pos=None, freq=None) == 0
    assert _append(tokens=0, kv=None) == 0
    assert _prefix(tokens=0, q=None) == 0


def _append(kv=X, dtype=0, wdtype=0, tokens=1, slots=X, cache=X, layout=0, pages=4):
    return _rc("dsa_latent_cache_append", kv, 576, dtype, X, wdtype, tokens, X, 0, slots, X, cache, 64 * 512, 512,
               cache, 64 * 64, 64, pages, 1e-6, layout, 1.0, None, None)


@pytest.mark.parametrize("kw", [dict(kv=None), dict(slots=None), dict(cache=None), dict(dtype=9), dict(wdtype=-1),
                                dict(layout=5), dict(tokens=-1), dict(pages=-1)])
def test_append_refuses(kw):
    assert _append(**kw) == INVALID


def _prefix(q=X, q_st=16 * 512, cache=X, row=512, pages=X, max_prefix=64, table=X, batch=4, width=4, request=None,
            lens=X, tokens=1, heads=16, num_pages=8, out=X, ws=X, nws=1 << 40):
    return _rc("dsa_shared_prefix_attention", q, q_st, 512, q, 16 * 64, 64, cache, 64 * 512, row, cache, 64 * 64, 64,
               pages, max_prefix, None, table, 4, batch, width, request, lens, tokens, heads, num_pages, 0.1, out,
               16 * 512, 512, out, 16, 1, ws, nws, None)


@pytest.mark.parametrize("kw", [dict(q=None), dict(q=X + 8), dict(q_st=4, tokens=2), dict(cache=None), dict(cache=X + 2),
                                dict(row=516), dict(pages=None), dict(max_prefix=-1), dict(table=None),
                                dict(lens=None), dict(out=None), dict(ws=None), dict(batch=0, request=None),
                                dict(tokens=-1), dict(heads=24), dict(heads=0), dict(num_pages=-1)])
def test_prefix_refuses(kw):
    assert _prefix(**kw) == INVALID


def test_prefix_workspace_refusals():
    n = ctypes.c_size_t(0)
    assert _rc("dsa_shared_prefix_attention_workspace_size", 4, 20, ctypes.byref(n)) == INVALID
    assert b"multiple of 16" in _lib.load().dsa_last_error_message()
    assert _rc("dsa_shared_prefix_attention_workspace_size", 4, 16, None) == INVALID


def test_wrappers_raise_without_a_gpu():
    z = lambda *s, t=torch.int32: torch.zeros(s, dtype=t)  # noqa: E731
    inv = fi.rope_frequencies(64, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA"):
        fi.step_layout(z(2), z(2), z(2, 4), z(8), 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        fi.apply_rope(z(2, 1, 64, t=torch.bfloat16), z(2), inv)
    with pytest.raises(RuntimeError, match="CUDA"):
        fi.latent_cache_append(z(2, 576, t=torch.bfloat16), z(512, t=torch.bfloat16), z(2), z(2), inv,
                               z(4, 64, 512, t=torch.bfloat16), z(4, 64, 64, t=torch.bfloat16))
    with pytest.raises(RuntimeError, match="CUDA"):
        fi.shared_prefix_attention(z(2, 16, 512, t=torch.bfloat16), z(2, 16, 64, t=torch.bfloat16),
                                   z(4, 64, 512, t=torch.bfloat16), z(4, 64, 64, t=torch.bfloat16), z(1), 64, z(2, 2),
                                   z(2), 0.1)
    with pytest.raises(AssertionError):
        fi.step_layout(z(2), z(3), z(2, 4), z(8), 2)
    with pytest.raises(AssertionError):
        fi.apply_rope(z(2, 1, 64), z(2), inv)  # integer values


def test_frequency_scalings():
    plain = fi.rope_frequencies(64, 10000.0, device="cpu")
    i = torch.arange(32, dtype=torch.float64)
    assert torch.allclose(plain, 10000.0 ** (-2 * i / 64), rtol=1e-15, atol=0)
    assert torch.equal(fi.rope_frequencies(64, 10000.0, scaling="linear", factor=8.0, device="cpu"), plain / 8)
    # the lowest frequency of ntk scaling is the plain one divided by the factor, the highest stays
    ntk = fi.rope_frequencies(64, 10000.0, scaling="ntk", factor=8.0, device="cpu")
    assert ntk[0] == 1 and math.isclose(ntk[-1], plain[-1] / 8, rel_tol=1e-12)
    yarn = fi.rope_frequencies(64, 10000.0, scaling="yarn", factor=40.0, original_context=4096, device="cpu")
    turns = plain * 4096 / (2 * math.pi)
    assert torch.equal(yarn[turns > 48], plain[turns > 48])  # above beta_fast = 32, rounded down to a pair
    assert torch.allclose(yarn[turns < 0.66], plain[turns < 0.66] / 40, rtol=1e-15, atol=0)
    assert (yarn <= plain).all() and (yarn >= plain / 40 * (1 - 1e-15)).all()
    with pytest.raises(ValueError):
        fi.rope_frequencies(64, scaling="cubic", device="cpu")
    with pytest.raises(ValueError):
        fi.rope_frequencies(64, scaling="linear", factor=0.5, device="cpu")
    with pytest.raises(AssertionError):
        fi.rope_frequencies(63, device="cpu")
