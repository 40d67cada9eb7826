"""Sizes past what the kernels of a head's loss gradients can be launched for are refused
before anything runs, without a device."""
import pytest
import torch

from krunch_amd import _lib

L = _lib.lib()
BUF = torch.zeros(1 << 10, dtype=torch.uint8)
PTR = (BUF.data_ptr() + 255) // 256 * 256
MOST = 1 << 33


@pytest.mark.parametrize("N,C,V", [(MOST // 16384 + 1, 16384, 64), (1 << 24, 576, 64), (64, 16384, MOST // 16384 + 1)])
def test_gradients_of_too_many_values(N, C, V):
    for dx, dW in ((PTR, PTR), (PTR, None), (None, PTR)):
        rc = L.kr_head_loss_backward(PTR, C, N, C, PTR, C, V, PTR, PTR, PTR, 0, dx, dW, PTR, 1 << 60, None)
        assert rc < 0 and "2^33" in L.kr_last_error().decode()
    assert L.kr_head_loss_backward_workspace_bytes(N, C, V, 1, 1) == 0


def test_the_largest_are_not():
    for N, C, V in ((MOST // 16384, 16384, 64), (1 << 24, 512, 64), (64, 16384, MOST // 16384)):
        assert L.kr_head_loss_backward_workspace_bytes(N, C, V, 1, 1) > 0
    assert L.kr_head_loss_workspace_bytes(1 << 24, 576, 64) > 0      # the loss has no such limit
