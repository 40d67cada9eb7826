"""A head's loss where logits are large, up to 2^33. All z are whole numbers that fp32 sums
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
