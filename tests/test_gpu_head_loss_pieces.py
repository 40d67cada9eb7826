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


@pytest.mark.parametrize("N,C,V", [(4161, 832, 20011), (8200, 576, 20011), (5794, 2368, 2345), (700, 832, 60001)])
def test_large_tiles_in_the_products(N, C, V):
    """Tiles of 256 x 256 in both products, which calls of more than 512 channels and 100
    tiles of dW a piece take: rows, channels and columns that end inside a tile, two pieces,
    dx written at once (2345 columns) and from 4 to 64 splits."""
    x, W, t, w = make(N, C, V, 11)
    _, lse = check_loss(x, W, t)
    dx, dW = ops.head_loss_backward(x, W, t, lse, w)
    wx, wW, ex, eW = plain_grads(x, W, t, w)
    near(dx, wx, ex)
    near(dW, wW, eW)
    only, _ = ops.head_loss_backward(x, W, t, lse, w, dW=False)
    near(only, wx, ex)
    _, only = ops.head_loss_backward(x, W, t, lse, w, dx=False)
    near(only, wW, eW)


@pytest.mark.parametrize("N,C,V", [(1, 1536, 3000), (7, 1600, 3000), (16, 2048, 301), (70, 1600, 3000), (300, 4160, 1000),
                                   (33, 16384, 513)])
def test_wide_rows(N, C, V):
    """Past 1024 channels, and past 1536, where a few rows take the tiles, too."""
    x, W, t, w = make(N, C, V, C)
    _, lse = check_loss(x, W, t)
    wx, wW, ex, eW = plain_grads(x, W, t, w)
    for dtype in (torch.float16, torch.float32):
        dx, dW = ops.head_loss_backward(x, W, t, lse, w, dtype)
        near(dx, wx, ex)
        near(dW, wW, eW)


@pytest.mark.parametrize("N", [8, 9, 16, 17, 128, 129])
def test_rows_at_the_kernels_limits(N):
    x, W, t, w = make(N, 768, 2000, N)
    _, lse = check_loss(x, W, t)
    dx, dW = ops.head_loss_backward(x, W, t, lse, w)
    wx, wW, ex, eW = plain_grads(x, W, t, w)
    near(dx, wx, ex)
    near(dW, wW, eW)
