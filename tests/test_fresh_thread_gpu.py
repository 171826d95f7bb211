"""Calls from a host thread that has not touched CUDA before: the driver's tensor-map encoder needs a context there."""
from __future__ import annotations

import math
import threading

import pytest
import torch

import flashinfer_repo_b200 as fi

from . import prefix_oracle as P

pytestmark = pytest.mark.gpu
SCALE = 1 / math.sqrt(192.0)


def _in_thread(call):
    """The result of call() in a new thread, whose allocations are served from torch's cache."""
    box = []

    def work():
        try:
            box.append((call(), None))
        except Exception as e:  # noqa: BLE001
            box.append((None, e))

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    value, error = box[0]
    if error is not None:
        raise error
    return value


def test_shared_prefix_attention():
    c = P.make_case(1, 5, 16, 300, [0, 7, 64, 100, 1])

    def call():
        return fi.shared_prefix_attention(c["qn"], c["qp"], c["ckv"], c["kpe"], c["pages"], c["prefix"], c["table"],
                                          c["lens"], SCALE)
    call()
    got = _in_thread(call)
    P.check(c, got, SCALE)
    assert fi.read_prefix_error() == 0
