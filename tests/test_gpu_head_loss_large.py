"""A head's loss and its gradients where logits are large: up to 2^33, and of thousands with
a gradient that is a small difference from lse. All z are whole numbers that fp32 sums
hold exactly in any order, so that float64 has the same z."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
SIZES = [(5, 300), (40, 300), (300, 300), (300, 50000)]       # few rows, small and large tiles


@pytest.mark.parametrize("N,V", SIZES)
@pytest.mark.parametrize("sign,least", [(1.0, 0), (-1.0, 1), (1.0, 8)])
def test_losses_of_huge_logits(N, V, sign, least):
    """z = sign a k 2^27, k of least..8 and a of 1..8 by row: finite, so lse and losses are."""
    g = torch.Generator().manual_seed(N + V)
    k = torch.randint(least, 9, (V,), generator=g)
    x = torch.zeros(N, 64)
    x[:, :8] = sign * 4096 * torch.randint(1, 9, (N, 1), generator=g)
    W = torch.zeros(V, 64)
    W[:, :8] = 32768.0 * (torch.arange(8)[None] < k[:, None])
    t = torch.randint(0, V, (N,), generator=g, dtype=torch.int32)
    x, W, t = x.half().to(DEV), W.half().to(DEV), t.to(DEV)
    loss, lse = ops.head_loss(x, W, t)
    z = x.double() @ W.double().t()
    want = torch.logsumexp(z, 1)
    top = z.amax(1)
    # max - z_t is exact, and ln of a sum of V / 9 equal terms has a few steps of 16
    want_loss = (top - z.gather(1, t.long()[:, None])[:, 0]) + torch.log(torch.exp(z - top[:, None]).sum(1))
    assert ((lse.double() - want).abs() <= 2.0 ** -23 * want.abs() + 2.0 ** -19).all(), (lse, want)
    assert ((loss.double() - want_loss).abs() <= 2.0 ** -23 * want_loss + 2.0 ** -19).all(), (loss, want_loss)


@pytest.mark.parametrize("N,V", SIZES)
def test_gradients_beside_a_large_lse(N, V):
    """z of thousands, half of the targets the largest: dz is dloss (e^(z - lse) - 1) with z - lse
    of some 2^-12 or none, for the lse that the call is given."""
    g = torch.Generator().manual_seed(3 * N + V)
    x = torch.randint(-32, 33, (N, 64), generator=g).half().to(DEV)
    W = torch.randint(-8, 9, (V, 64), generator=g).half().to(DEV)
    z = x.double() @ W.double().t()
    t = z.argmax(1).int()
    t[::2] = torch.randint(0, V, t[::2].shape, generator=g, dtype=torch.int32).to(DEV)
    w = (0.5 + torch.rand(N, generator=g)).to(DEV)
    lse = torch.logsumexp(z, 1).float()
    assert lse.min() > 200
    dx, dW = ops.head_loss_backward(x, W, t, lse, w, torch.float32)
    p = torch.exp(z - lse.double()[:, None]) * w.double()[:, None]
    dz = p.clone()
    dz.scatter_add_(1, t.long()[:, None], -w.double()[:, None])
    # z - lse and its product with log2 e, exp2: 2^-20 of a p down to e^-16 (far smaller ones
    # are below the absolute part); a target's difference, two parts; fp32 sums
    e = 2.0 ** -20 * p + 2.0 ** -22 * dz.abs() + 2.0 ** -38 * w.max().double()
    e.scatter_add_(1, t.long()[:, None], 2.0 ** -23 * w.double()[:, None])
    a = dz.abs()
    for got, want, err in ((dx, dz @ W.double(), (e + (V / 4 + 64) * 2.0 ** -24 * a) @ W.double().abs()),
                           (dW, dz.t() @ x.double(), (e + (N / 4 + 64) * 2.0 ** -24 * a).t() @ x.double().abs())):
        off = (got.double() - want).abs()
        assert (off <= err + 2.0 ** -23 * want.abs()).all(), (off / err).max()
