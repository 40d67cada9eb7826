"""Gradients of a head's loss in pieces of the vocabulary of which the last is short, and
by the kernels of the largest calls, against float64 (the bounds of test_gpu_head_loss)."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops
from tests.test_gpu_head_loss import check_loss, make, near, plain_grads

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("N,C,V", [(90112, 64, 4097), (33846, 320, 40970)])
def test_a_last_piece_with_fewer_steps_than_splits(N, C, V):
    """dx alone: five pieces of 1024 columns and one column more, two splits of a piece; 17 of
    2560, whose last has 10 columns."""
    x, W, t, w = make(N, C, V, 3)
    t[::1000] = V - 1                                 # some targets in the last piece
    _, lse = check_loss(x, W, t)
    dx, none = ops.head_loss_backward(x, W, t, lse, w, dW=False)
    assert none is None
    wx, _, ex, _ = plain_grads(x, W, t, w)
    near(dx, wx, ex)
    assert torch.equal(ops.head_loss_backward(x, W, t, lse, w, dW=False)[0], dx)
