"""Scores of tokens: widths on both sides of the lines between its kernels, sums
over very wide rows, and signs (no probability above 1, no entropy below 0)."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops
from tests.test_gpu_scores import check, rand

pytestmark = pytest.mark.gpu
DEV = "cuda"


# chunks are of 8 fp16 or 4 fp32 logits: 256 and 512 logits, and 128, 256, 1024 and
# 4096 chunks, are the last widths of a kernel
@pytest.mark.parametrize("dtype,V", [(torch.float16, v + d) for v in (1024, 8192, 32768) for d in (-1, 0, 1)] +
                         [(torch.float32, v + d) for v in (4096, 16384) for d in (-1, 0, 1)])
@pytest.mark.parametrize("k", [0, 8, 32])
def test_widths_of_the_dispatch(dtype, V, k):
    check(*rand(4, V, dtype, V + k), k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [(1 << 20) + 3, (1 << 24) + 5])
def test_sums_of_very_wide_rows(dtype, V):
    """Equal and nearly equal logits: every addition of a chain rounds to one side.
    Within the tolerances of the other tests, which allow 128 roundings of 2^-24 in ln
    s: a block of at most 32 terms is summed by itself, blocks are added with their
    rounding errors carried along, then come 6 + 8 additions."""
    x, tok = rand(3, V, dtype, 5, 1e-3)
    x[0] = 0.0
    x += 1.7
    x[2, ::3] -= 4.0
    check(x, tok, 0)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_a_rising_row(dtype):
    """Sorted logits: the running maximum rises in most blocks. fp16 has few steps to
    rise by; the fp32 row has V / 8192 = 64 blocks a thread, each with an exp2 and a
    product, 3 roundings of 2^-24: 192, beside the 128 of the check: 2^-15 in all."""
    V = 1 << 19
    x, tok = rand(2, V, dtype, 7)
    x = torch.sort(x, dim=1).values
    lp, h = (a.double().cpu() for a in ops.token_scores(x, tok)[:2])
    logp = torch.log_softmax(x.double().cpu(), 1)
    want = logp.gather(1, tok.long().cpu()[:, None])[:, 0]
    assert ((lp - want).abs() <= 2.0 ** -15 + 2.0 ** -22 * want.abs()).all()
    assert ((h + (logp.exp() * logp).sum(1)).abs() <= 2.0 ** -14 + 2.0 ** -18 * h).all()

@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [1, 100, 300, 700, 2000, 6000, 50277])
def test_no_probability_above_one_and_no_entropy_below_zero(dtype, V):
    """Rows of one token of probability 1, by masks or by distance, at many values."""
    N = 400
    g = torch.Generator().manual_seed(V)
    top = (40 * torch.randn(N, generator=g)).to(dtype).to(DEV)
    x = torch.full((N, V), -float("inf"), dtype=dtype, device=DEV)
    at = torch.randint(0, V, (N,), generator=g).to(DEV)
    rows = torch.arange(N, device=DEV)
    x[N // 2:] = -30000.0
    x[rows, at] = top
    lp, h, tl, tt = ops.token_scores(x, at.to(torch.int32), min(V, 3))
    assert (lp <= 0).all() and (tl <= 0).all() and (h >= 0).all()
    assert (lp >= -2.0 ** -17).all() and (h <= 2.0 ** -16).all() and torch.equal(tt[:, 0], at.to(torch.int32))
    check(x, at.to(torch.int32), min(V, 3))
