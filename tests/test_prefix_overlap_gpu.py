"""Shared-prefix attention calls that run at the same time: on two streams, from two threads, out of two captured
graphs.  None is given a workspace."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import flashinfer_repo_b200 as fi

from . import prefix_oracle as P

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192.0)


def _attend(c):
    return fi.shared_prefix_attention(c["qn"], c["qp"], c["ckv"], c["kpe"], c["pages"], c["prefix"], c["table"], c["lens"],
                                      SCALE, token_request=c["request"])


def _cases():
    """Of different plans: one row block over all pairs, several blocks, more blocks than pairs."""
    return [P.make_case(1, 4, 16, 9000, [50] * 4), P.make_case(2, 40, 16, 3000, [i * 9 for i in range(40)]),
            P.make_case(3, 90, 128, 700, [i % 77 for i in range(90)])]


def _same(a, b):
    return torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_two_streams():
    cases = _cases()
    want = [_attend(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[] for _ in cases]
    for _ in range(10):
        for c, s, g in zip(cases, streams, got):
            with torch.cuda.stream(s):
                g.append(_attend(c))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(_same(w, x) for x in g)
    assert fi.read_prefix_error() == 0


def test_two_threads_on_one_stream():
    cases = _cases()
    want = [_attend(c) for c in cases]
    got = [[] for _ in cases]

    def work(i):
        for _ in range(20):
            got[i].append(_attend(cases[i]))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert len(g) == 20 and all(_same(w, x) for x in g)


def test_two_graphs_and_an_eager_call():
    cases = _cases()
    want = [_attend(c) for c in cases]
    torch.cuda.synchronize()
    graphs, got = [], []
    for c in cases[:2]:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(_attend(c))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(10):
        for w in got:
            w[0].zero_()
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        eager = _attend(cases[2])
        for s in streams:
            torch.cuda.current_stream().wait_stream(s)
        assert _same(want[0], got[0]) and _same(want[1], got[1]) and _same(want[2], eager)


def test_errors_reach_the_device_word_from_any_stream_and_graph():
    c = _cases()[0]
    _attend(c)
    assert fi.read_prefix_error() == 0
    c["table"][1, 0] = 10 ** 7
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _attend(c)
        assert fi.read_prefix_error() == 1
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _attend(c)
    assert fi.read_prefix_error() == 0
    graph.replay()
    assert fi.read_prefix_error() == 1 and out[0].isfinite().all()
