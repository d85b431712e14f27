"""Calls of the label-distribution operators that are answered before any kernel (lib/losses.py, lib/_hip.py)."""
import pytest
import torch

from lib import _hip
from lib.losses import TopLogits, distill_loss

X = torch.zeros(4, 10)
REC = TopLogits(torch.zeros(4, 3), torch.zeros(4, 3, dtype=torch.int32), torch.zeros(4))


def test_a_row_weight_that_asks_for_a_gradient_is_refused():
    w = torch.ones(4, requires_grad=True)
    with pytest.raises(ValueError, match='row_weight gets no gradient'):
        distill_loss(X, REC, row_weight=w)
    for given in (w.detach(), torch.ones(4)):
        with pytest.raises(_hip.HipKernelError, match='no CPU fallback'):           # past the check
            distill_loss(X, REC, row_weight=given)
    with torch.no_grad(), pytest.raises(_hip.HipKernelError, match='no CPU fallback'):
        distill_loss(X, REC, row_weight=w)


def test_the_librarys_limit_of_a_record(so_path, monkeypatch):
    """one number on the Python side, and a library with another is not loaded"""
    import ctypes
    assert ctypes.CDLL(so_path).mh_top_logits_max_k() == _hip.MAX_TOP
    monkeypatch.setattr(_hip, '_lib', None)
    monkeypatch.setattr(_hip, 'MAX_TOP', 512)
    with pytest.raises(_hip.HipKernelError, match='up to 1024 entries'):
        _hip.lib()
    with pytest.raises(ValueError, match='1 to 512 entries'):
        distill_loss(X, REC._replace(values=torch.zeros(4, 513)))
