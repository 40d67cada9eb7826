"""float32 gradients of a head's loss (kr_head_loss_backward with out_f32): dz enters the
products in two fp16 parts, 22 bits, against float64. Sizes around the tiles, short last
pieces, the kernels of large and small calls, one gradient only, weights far apart."""
import pytest
import torch

from krunch_amd import _lib, krunch_ac_hip as ops
from tests.test_gpu_head_loss import DEV, make, plain_loss, rows

pytestmark = pytest.mark.gpu


def plain(x, W, t, w):
    """dx, dW in float64 and the bounds of their errors: those of test_gpu_head_loss, but for
    dz, of which two parts keep 2^-22 (2^-39 of the largest |w| where the second is
    subnormal) and a target's difference in fp32 as much of w; chains have twice the terms."""
    N, V = x.shape[0], W.shape[0]
    lse, _, zerr, err, _ = plain_loss(x, W, t)
    x, W = x.double(), W.double()
    w = torch.where(t >= 0, w.double(), 0.0)
    top = w.abs().max()
    dx, ex = torch.zeros_like(x), torch.zeros_like(x)
    dW, eW = torch.zeros_like(W), torch.zeros_like(W)
    for i in rows(N, V):
        dz = torch.softmax(x[i] @ W.t(), 1) * w[i, None]
        e = dz.abs() * (2 * (zerr + err)[i, None] + 2.0 ** -21)
        at = t[i].long().clamp_min(0)[:, None]
        dz.scatter_add_(1, at, -w[i, None])
        e.scatter_add_(1, at, 2.0 ** -22 * w[i, None].abs())
        e = (e + 2.0 ** -39 * top) * (w[i, None] != 0)
        dx[i] = dz @ W
        dW += dz.t() @ x[i]
        a = dz.abs()
        ex[i] = (e + (V / 4 + 64) * 2.0 ** -24 * a) @ W.abs()
        eW += (e + (N / 4 + 64) * 2.0 ** -24 * a).t() @ x[i].abs()
    return dx, dW, ex + 2.0 ** -23 * dx.abs(), eW + 2.0 ** -23 * dW.abs()


def check(x, W, t, w, tight=True):
    lse = ops.head_loss(x, W, t)[1]
    dx, dW = ops.head_loss_backward(x, W, t, lse, w, torch.float32)
    wx, wW, ex, eW = plain(x, W, t, w)
    for got, want, err in ((dx, wx, ex), (dW, wW, eW)):
        assert got.dtype == torch.float32
        off = (got.double() - want).abs()
        assert (off <= err).all(), (off / err).max()
        # of either sign: far below the 2^-12 that one part would leave in 2-norm. An
        # lse of up to 16 and its sum are fp32 within 2^-20, which all of a row has
        if tight:
            assert off.norm() <= 2.0 ** -18 * want.norm()
    return lse, dx, dW


@pytest.mark.parametrize("N,C,V", [(1, 64, 1), (1, 768, 50277), (3, 128, 127), (65, 768, 256), (129, 128, 1000),
                                   (513, 192, 257), (97, 1024, 5000), (700, 64, 3001)])
def test_sizes(N, C, V):
    # one column is all of the softmax: its gradient is what roundings leave of 0
    check(*make(N, C, V, N + C), tight=V > 1)


@pytest.mark.parametrize("N,C,V", [(4161, 832, 20011), (8192, 64, 11000), (45056, 64, 2049), (20000, 256, 256)])
def test_pieces_and_tiles(N, C, V):
    """Large tiles in the products; several pieces; a last one a column longer than its tiles."""
    x, W, t, w = make(N, C, V, 7)
    lse, dx, dW = check(x, W, t, w)
    again = ops.head_loss_backward(x, W, t, lse, w, torch.float32)
    assert torch.equal(again[0], dx) and torch.equal(again[1], dW)


def test_one_gradient_only():
    x, W, t, w = make(45056, 64, 2049, 2)
    lse = ops.head_loss(x, W, t)[1]
    wx, wW, ex, eW = plain(x, W, t, w)
    dx, none = ops.head_loss_backward(x, W, t, lse, w, torch.float32, dW=False)
    assert none is None and ((dx.double() - wx).abs() <= ex).all()
    none, dW = ops.head_loss_backward(x, W, t, lse, w, torch.float32, dx=False)
    assert none is None and ((dW.double() - wW).abs() <= eW).all()


def test_rows_without_gradient_and_weights_far_apart():
    x, W, t, w = make(190, 128, 600, 4, none=False)
    w = torch.logspace(-5, 1, 190).to(DEV) * torch.where(torch.arange(190) % 2 == 0, 1.0, -1.0).to(DEV)
    check(x, W, t, w)
    t[5], w[6] = -1, 0.0
    x[5], x[6] = float("nan"), float("inf")
    lse = ops.head_loss(x, W, t)[1]
    dx, dW = ops.head_loss_backward(x, W, t, lse, w, torch.float32)
    live = torch.ones(190, dtype=torch.bool, device=DEV)
    live[5:7] = False
    wx, wW, ex, eW = plain(x[live], W, t[live], w[live])
    assert (dx[~live] == 0).all()
    assert ((dx[live].double() - wx).abs() <= ex).all() and ((dW.double() - wW).abs() <= eW).all()


def test_graph():
    x, W, t, w = make(400, 128, 3000, 14)
    lse = ops.head_loss(x, W, t)[1]
    graph, ws = torch.cuda.CUDAGraph(), w.clone()
    with torch.cuda.graph(graph):
        out = ops.head_loss_backward(x, W, t, lse, ws, torch.float32)
    for k in range(4):
        ws.copy_(w if k % 2 == 0 else -3 * w)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, ops.head_loss_backward(x, W, t, lse, ws, torch.float32)))


def test_workspace_holds_both_outputs_plans():
    """The query knows no output type: what it says is enough for both."""
    L = _lib.lib()
    for N, C, V in ((45056, 64, 2049), (8192, 768, 50277), (300, 64, 100)):
        x, W, t, w = make(N, C, V, 1)
        lse = ops.head_loss(x, W, t)[1]
        nbytes = L.kr_head_loss_backward_workspace_bytes(N, C, V, 1, 1)
        ws = torch.full((nbytes + 4096,), 255, dtype=torch.uint8, device=DEV)
        for f32, dtype in ((0, torch.float16), (1, torch.float32)):
            dx, dW = torch.empty(N, C, dtype=dtype, device=DEV), torch.empty(V, C, dtype=dtype, device=DEV)
            _lib.call("kr_head_loss_backward", x.data_ptr(), C, N, C, W.data_ptr(), C, V, t.data_ptr(), lse.data_ptr(),
                      w.data_ptr(), f32, dx.data_ptr(), dW.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_ptr())
            assert (ws[nbytes:] == 255).all()
            want = ops.head_loss_backward(x, W, t, lse, w, dtype)
            assert torch.equal(dx, want[0]) and torch.equal(dW, want[1])
