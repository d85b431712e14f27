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
