"""The status words of an engine whose projections have two scratch buffers: those of the bf16 head and of the 4-bit weights."""
from types import SimpleNamespace

import pytest
import torch

from conftest import load


def _engine(bits):
    cls, ops = load("model").Engine, load("ops")
    eng = cls.__new__(cls)
    eng.ws_linear, eng.ws_q4 = ops.new_workspace(4096, "cpu"), ops.new_workspace(4096, "cpu") if bits == 4 else None
    eng.kv, eng.m, eng.max_rows = None, SimpleNamespace(device="cpu", V=8), 64
    return eng


@pytest.mark.parametrize("head,q4,own", [(0, 2, 0), (1, 2, 0), (0, 2, 1), (4, 0, 0)])
def test_both_scratch_buffers_are_looked_at(head, q4, own):
    eng = _engine(4)
    assert eng.status_word() == 0
    eng.check_status()
    eng.ws_linear[:4].view(torch.int32)[0], eng.ws_q4[:4].view(torch.int32)[0] = head, q4
    eng._own_status_word()[0] = own
    eng.ws_q4[300] = 9  # an arrival counter that a late contributor has bumped
    assert eng.status_word() == head | q4
    with pytest.raises(RuntimeError, match=f"{head | q4:#x}") as told:
        eng.check_status()
    assert ("attention" in str(told.value)) == bool(own)
    assert not eng.ws_linear.any() and not eng.ws_q4.any()
    eng.check_status()
    assert eng.status_word() == 0


def test_without_4_bit_weights():
    eng = _engine(16)
    eng.ws_linear[:4].view(torch.int32)[0] = 3
    assert eng.status_word() == 3
    with pytest.raises(RuntimeError, match="0x3"):
        eng.check_status()
    assert eng.status_word() == 0
