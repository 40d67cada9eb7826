"""Cross entropy of a head without its logits (kr_head_loss) and its gradients
(kr_head_loss_backward), against float64: sizes around the tiles' edges, pieces of the
vocabulary, strides, rows without a token, NaN and infinities, types, graphs, streams."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(N, C, V, seed, amp=1.0, none=True):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(N, C, generator=g).half().to(DEV)
    W = (amp * torch.randn(V, C, generator=g) / C ** 0.5).half().to(DEV)
    t = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    if none and N > 2:
        t[torch.randint(0, N, (1 + N // 16,), generator=g)] = -1
    return x, W, t.to(DEV), (0.1 + torch.rand(N, generator=g)).to(DEV)


def rows(N, V):
    """Row blocks whose [rows, V] float64 matrices take at most 1 GB."""
    step = max(1, (1 << 27) // V)
    return [slice(i, min(N, i + step)) for i in range(0, N, step)]


def plain_loss(x, W, t):
    """lse and loss in float64 and the error of z (fp32 sums of C exact products), of a
    row's logsumexp and of its loss."""
    N, C, V = x.shape[0], x.shape[1], W.shape[0]
    x, W = x.double(), W.double()
    lse, loss, zerr, spread = (torch.zeros(N, dtype=torch.float64, device=DEV) for _ in range(4))
    for i in rows(N, V):
        z = x[i] @ W.t()
        lse[i] = torch.logsumexp(z, 1)
        at = z.gather(1, t[i].long().clamp(0, V - 1)[:, None])[:, 0]
        loss[i] = torch.where(t[i] >= 0, lse[i] - at, 0.0)
        zerr[i] = (C + 8) * 2.0 ** -24 * (x[i].abs() @ W.abs().t()).amax(1)
        spread[i] = z.amax(1) - z.amin(1)
    # a sum of at most 64 + V / 128 positive terms in a chain, each with the roundings
    # of a difference, a product with log2 e and an exp2 of up to `spread`
    err = zerr + (72 + V / 128 + 3 * spread) * 2.0 ** -24 + 4 * 2.0 ** -24 * lse.abs()
    return lse, loss, zerr, err, err + zerr + 2.0 ** -22 * (lse.abs() + loss.abs())


def check_loss(x, W, t):
    lse, loss, _, err, loss_err = plain_loss(x, W, t)
    got, got_lse = ops.head_loss(x, W, t)
    assert ((got_lse.double() - lse).abs() <= err).all(), ((got_lse - lse).abs() / err).max()
    assert ((got.double() - loss).abs() <= loss_err).all(), ((got - loss).abs() / loss_err).max()
    return got, got_lse


def plain_grads(x, W, t, w):
    """dx, dW in float64 and the bound of their errors for an fp32 output."""
    N, C, V = x.shape[0], x.shape[1], W.shape[0]
    lse, _, zerr, err, _ = plain_loss(x, W, t)
    x, W = x.double(), W.double()
    w = torch.where(t >= 0, w.double(), 0.0)
    top = w.abs().max()
    dx, ex = torch.zeros_like(x), torch.zeros_like(x)
    dW, eW = torch.zeros_like(W), torch.zeros_like(W)
    for i in rows(N, V):
        p = torch.softmax(x[i] @ W.t(), 1)
        dz = p * w[i, None]
        # a probability: its exponent's error, 2^-22 of roundings; a dz: fp16's half
        # step, or half a subnormal one at the largest |dloss| = 2^14
        e = dz.abs() * (2 * (zerr + err)[i, None] + 2.0 ** -22)
        at = t[i].long().clamp_min(0)[:, None]
        dz.scatter_add_(1, at, -w[i, None])
        e = (e + 2.0 ** -11 * dz.abs() + 2.0 ** -39 * top) * (w[i, None] != 0)
        dx[i] = dz @ W
        dW += dz.t() @ x[i]
        # and fp32 sums: chains of an eighth of the terms
        a = dz.abs()
        ex[i] = (e + (V / 8 + 64) * 2.0 ** -24 * a) @ W.abs()
        eW += (e + (N / 8 + 64) * 2.0 ** -24 * a).t() @ x[i].abs()
    return dx, dW, ex, eW


def near(got, want, err):
    half = got.dtype == torch.float16
    err = err + (2.0 ** -11 * want.abs() + 2.0 ** -25 if half else 2.0 ** -23 * want.abs())
    assert torch.isfinite(got).all()
    off = (got.double() - want).abs()
    assert (off <= err).all(), (off / err).max()


def check_grads(x, W, t, w, dtype=None):
    _, lse = ops.head_loss(x, W, t)
    dx, dW = ops.head_loss_backward(x, W, t, lse, w, dtype)
    wx, wW, ex, eW = plain_grads(x, W, t, w)
    near(dx, wx, ex)
    near(dW, wW, eW)
    return lse, dx, dW


SIZES = [(1, 64, 1), (1, 768, 50277), (2, 64, 5), (3, 128, 127), (17, 64, 128), (64, 320, 129), (65, 768, 256),
         (128, 64, 1000), (129, 128, 1000), (257, 512, 255), (300, 1024, 3001), (513, 192, 257), (1000, 256, 256)]


@pytest.mark.parametrize("N,C,V", SIZES)
def test_sizes(N, C, V):
    x, W, t, w = make(N, C, V, N + C + V)
    check_loss(x, W, t)
    check_grads(x, W, t, w)


@pytest.mark.parametrize("N,C,V", [(8192, 64, 20000), (5000, 128, 50277), (70000, 64, 300), (65541, 64, 130),
                                   (300, 64, 200001)])
def test_pieces_and_splits(N, C, V):
    x, W, t, w = make(N, C, V, 5)
    check_loss(x, W, t)
    check_grads(x, W, t, w)


@pytest.mark.parametrize("N", [5, 200])
def test_float_outputs_and_one_gradient_only(N):
    x, W, t, w = make(N, 256, 1500, N)
    lse, dx, dW = check_grads(x, W, t, w, torch.float32)
    assert dx.dtype == dW.dtype == torch.float32
    only, none = ops.head_loss_backward(x, W, t, lse, w, torch.float32, dW=False)
    assert none is None
    near(only, dx.double(), plain_grads(x, W, t, w)[2])
    none, only = ops.head_loss_backward(x, W, t, lse, w, torch.float32, dx=False)
    assert none is None and torch.equal(only, dW)
    assert ops.head_loss_backward(x, W, t, lse, w, dx=False, dW=False) == (None, None)


@pytest.mark.parametrize("N", [6, 150])
def test_strided_rows(N):
    x, W, t, w = make(N, 128, 700, 3)
    wide_x = torch.full((N, 3 * 128), float("nan"), dtype=torch.float16, device=DEV)
    wide_W = torch.full((700, 136), float("nan"), dtype=torch.float16, device=DEV)
    wide_x[:, 128:256] = x
    wide_W[:, :128] = W
    xs, Ws = wide_x[:, 128:256], wide_W[:, :128]
    loss, lse = ops.head_loss(x, W, t)
    assert all(torch.equal(a, b) for a, b in zip(ops.head_loss(xs, Ws, t), (loss, lse)))
    for a, b in zip(ops.head_loss_backward(xs, Ws, t, lse, w), ops.head_loss_backward(x, W, t, lse, w)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("amp", [0.0, 30.0, 300.0])
def test_flat_and_peaked_rows(amp):
    """Equal logits; probabilities from 1 down to far below what fp16 holds."""
    x, W, t, w = make(140, 128, 900, 8, amp)
    check_loss(x, W, t)
    check_grads(x, W, t, w)


@pytest.mark.parametrize("N", [40, 190])
def test_rows_without_gradient_may_hold_anything(N):
    x, W, t, w = make(N, 128, 600, 4, none=False)
    t[5], t[6], w[7] = -1, -1, 0.0
    x[5], w[6] = float("nan"), float("inf")
    x[6], x[7] = float("inf"), float("-inf")
    loss, lse = ops.head_loss(x, W, t)
    assert loss[5] == 0 and loss[6] == 0 and torch.isnan(lse[5])
    dx, dW = ops.head_loss_backward(x, W, t, lse, w)
    live = torch.ones(N, dtype=torch.bool, device=DEV)
    live[5:8] = False
    assert (dx[~live] == 0).all()
    wx, wW, ex, eW = plain_grads(x[live], W, t[live], w[live])
    near(dx[live], wx, ex)
    near(dW, wW, eW)
    none = torch.full_like(t, -1)
    dx, dW = ops.head_loss_backward(x, W, none, lse, w)
    assert (dx == 0).all() and (dW == 0).all()
    assert (ops.head_loss(x, W, none)[0] == 0).all()


@pytest.mark.parametrize("N", [40, 190])
def test_nan_infinities_and_foreign_ids(N):
    x, W, t, w = make(N, 128, 600, 6, none=False)
    clean, clean_lse = ops.head_loss(x, W, t)
    x[3] = float("nan")
    x[4, 0] = float("inf")
    t[8], t[9] = 600, -2
    loss, lse = ops.head_loss(x, W, t)
    bad = torch.zeros(N, dtype=torch.bool, device=DEV)
    bad[3:5] = True
    assert torch.isnan(lse[bad]).all() and torch.equal(lse[~bad], clean_lse[~bad])
    bad[8:10] = True
    assert torch.isnan(loss[bad]).all() and torch.equal(loss[~bad], clean[~bad])
    x, W, t, w = make(N, 128, 600, 6, none=False)
    t[8] = 600
    dx, dW = ops.head_loss_backward(x, W, t, clean_lse, w)
    assert torch.isnan(dx[8]).all() and torch.isfinite(dx[:8]).all() and torch.isfinite(dx[9:]).all()
    assert torch.isnan(dW).all()


def test_weights_far_apart():
    """dloss over seven powers of ten, and below fp32's normal range."""
    x, W, t, w = make(200, 128, 500, 9, none=False)
    w = torch.logspace(-6, 1, 200).to(DEV) * torch.where(torch.arange(200) % 2 == 0, 1.0, -1.0).to(DEV)
    check_grads(x, W, t, w, torch.float32)
    lse = ops.head_loss(x, W, t)[1]
    tiny = ops.head_loss_backward(x, W, t, lse, torch.full_like(w, 1e-41), torch.float32)
    assert all(torch.isfinite(g).all() and (g.abs() < 1e-38).all() for g in tiny)


def test_differences():
    """The gradients along random directions against differences of the float64 loss."""
    x, W, t, w = make(37, 64, 130, 2)
    lse = ops.head_loss(x, W, t)[1]
    dx, dW = ops.head_loss_backward(x, W, t, lse, w, torch.float32)
    _, _, ex, eW = plain_grads(x, W, t, w)
    g = torch.Generator().manual_seed(1)
    h = 1e-4

    def total(x, W):
        return (plain_loss(x, W, t)[1] * w.double()).sum()

    for grad, err, on_x in ((dx, ex, True), (dW, eW, False)):
        for _ in range(3):
            d = torch.randn(grad.shape, generator=g).double().to(DEV)
            diff = ((total(x.double() + h * d, W.double()) - total(x.double() - h * d, W.double())) if on_x else
                    (total(x.double(), W.double() + h * d) - total(x.double(), W.double() - h * d))) / (2 * h)
            # the third derivative along d: cumulants of z's change of up to a few
            # units a row, h^2 / 6 of their cubes
            change = (d @ W.double().t()) if on_x else (x.double() @ d.t())
            cut = (h * h * change.abs().amax(1) ** 3 * w.double()).sum() + 1e-9
            got = (grad.double() * d).sum()
            assert (got - diff).abs() <= ((err + 2.0 ** -23 * grad.abs()) * d.abs()).sum() + cut


def test_same_bits_again_and_no_rows():
    x, W, t, w = make(700, 192, 5000, 12)
    first = ops.head_loss(x, W, t)
    grads = ops.head_loss_backward(x, W, t, first[1], w)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(ops.head_loss(x, W, t), first))
        assert all(torch.equal(a, b) for a, b in zip(ops.head_loss_backward(x, W, t, first[1], w), grads))
    loss, lse = ops.head_loss(x[:0], W, t[:0])
    assert loss.shape == lse.shape == (0,)
    dx, dW = ops.head_loss_backward(x[:0], W, t[:0], lse, w[:0])
    assert dx.shape == (0, 192) and dW.shape == W.shape and (dW == 0).all()


@pytest.mark.parametrize("N", [3, 400])
def test_graph_and_streams(N):
    x, W, t, w = make(N, 128, 3000, 14)
    want = ops.head_loss(x, W, t)
    grads = ops.head_loss_backward(x, W, t, want[1], w)
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for s in (a, b, a, b):
        with torch.cuda.stream(s):
            loss, lse = ops.head_loss(x, W, t)
            got.append((loss, lse, *ops.head_loss_backward(x, W, t, lse, w)))
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(p, q) for p, q in zip(one, (*want, *grads)))
    graph = torch.cuda.CUDAGraph()
    xs = x.clone()
    with torch.cuda.graph(graph):
        loss, lse = ops.head_loss(xs, W, t)
        dx, dW = ops.head_loss_backward(xs, W, t, lse, w)
    for k in range(4):
        xs.copy_(x if k % 2 == 0 else -x)
        graph.replay()
        torch.cuda.synchronize()
        eager = ops.head_loss(xs, W, t)
        eager += ops.head_loss_backward(xs, W, t, eager[1], w)
        assert all(torch.equal(p, q) for p, q in zip(eager, (loss, lse, dx, dW)))
