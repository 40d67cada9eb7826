"""dW of the rows that are targets (kr_head_loss_backward, fp16 outputs): what fp16 leaves of
a target's dz, of most of such a row, is added back, so that the output's own rounding, at
most half a step of it, is nearly all of the error. Against float64: one row of x for a
row of W, many for one, lists longer than a workgroup holds, byte vocabularies, several
column tiles, pieces."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops
from tests.test_gpu_head_loss import DEV, make, plain_loss, rows

pytestmark = pytest.mark.gpu


def plain(x, W, t, w):
    """dW in float64 and the bound of its error: that of test_gpu_head_loss.plain_grads, but
    for a target's dz = w (p - 1), which has the errors of p, a difference in fp32 and two
    fp16 parts, 2^-22 of it (2^-39 of the largest |w| where the second is subnormal)."""
    N, V = x.shape[0], W.shape[0]
    lse, _, zerr, err, _ = plain_loss(x, W, t)
    x, W = x.double(), W.double()
    w = torch.where(t >= 0, w.double(), 0.0)
    top = w.abs().max()
    dW, eW = torch.zeros_like(W), torch.zeros_like(W)
    for i in rows(N, V):
        dz = torch.softmax(x[i] @ W.t(), 1) * w[i, None]
        e = dz.abs() * (2 * (zerr + err)[i, None] + 2.0 ** -22)
        at = t[i].long().clamp_min(0)[:, None]
        own = e.gather(1, at) + 2.0 ** -22 * w[i, None].abs() + 2.0 ** -39 * top
        e = e + 2.0 ** -11 * dz.abs() + 2.0 ** -39 * top
        e.scatter_(1, at, own)
        dz.scatter_add_(1, at, -w[i, None])
        e = e * (w[i, None] != 0)
        dW += dz.t() @ x[i]
        eW += (e + (N / 8 + 64) * 2.0 ** -24 * dz.abs()).t() @ x[i].abs()
    return dW, eW + 2.0 ** -23 * dW.abs()


def check(x, W, t, w):
    lse = ops.head_loss(x, W, t)[1]
    _, dW = ops.head_loss_backward(x, W, t, lse, w)
    want, err = plain(x, W, t, w)
    off = (dW.double() - want).abs()
    # half a step of fp16 where the value before its rounding may be
    half_step = torch.exp2(torch.floor(torch.log2(want.abs() + err)).clamp_min(-14) - 11)
    assert (off <= half_step + err).all(), (off / (half_step + err)).max()
    return dW


@pytest.mark.parametrize("N,C,V", [(1, 64, 300), (2, 768, 50277), (97, 256, 5000), (300, 1024, 3001),
                                   (1000, 128, 50277), (4161, 64, 20011), (20000, 256, 256), (9000, 64, 20000)])
def test_a_targets_row(N, C, V):
    check(*make(N, C, V, N + V))


@pytest.mark.parametrize("N", [200, 3001, 7000])
def test_one_target_for_all_rows(N):
    """Every row has the same target, or one of two in a tile: lists of N rows."""
    x, W, t, w = make(N, 192, 1000, N)
    t.fill_(999)
    check(x, W, t, w)
    t[1::2] = 900
    t[::7] = -1
    check(x, W, t, w)


def test_a_mean_of_a_thousand_rows():
    """dloss 1 / 1000, 1.02 times a power of two, puts every target's dz where fp16 is
    coarsest. In fp16 the outputs' rounding is to be all that shows: 2^-12 of a value on
    average over a binade's rounding errors, 2.1e-4 in 2-norm, and dz's of 1e-5 beside it."""
    x, W, t, w = make(1000, 768, 50277, 1, none=False)
    w.fill_(1e-3)
    lse = ops.head_loss(x, W, t)[1]
    _, dW = ops.head_loss_backward(x, W, t, lse, w)
    want = plain(x, W, t, w)[0]
    least = (want.half().double() - want).norm()
    assert (dW.double() - want).norm() <= 1.05 * least


def test_rows_that_hold_anything_reach_no_target():
    x, W, t, w = make(700, 128, 300, 4, none=False)
    want = check(x, W, t, torch.where(torch.arange(700, device=DEV) % 3 == 0, 0.0, w))
    x[::3] = float("nan")
    lse = ops.head_loss(x, W, t)[1]
    w[::3] = 0
    assert torch.equal(ops.head_loss_backward(x, W, t, lse, w)[1], want)
