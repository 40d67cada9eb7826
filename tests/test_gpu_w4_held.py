"""Products with 4-bit weights in the kernels that hold rows in LDS (up to 16 rows
with 1536 tiles of 16 outputs or more; 32 and 64 rows where 256 workgroups of 12
waves get a unit of 32 outputs each): every group, output and epilogue, the same
bits as calls of few rows, inputs that end inside a group and a block."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops
from tests.test_gpu_w4 import check, make

pytestmark = pytest.mark.gpu
DEV = "cuda"

# (M, K, N): 16 rows held; 32 held by units, and by K; 64 held. N / 32 is no integer,
# K = 416 and 1440 are 32 past a block, 1248 is 96 past one
HELD = [(9, 416, 24601), (16, 768, 24576), (250, 416, 12333), (520, 1440, 12333), (520, 416, 12333),
        (600, 1248, 11001)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", HELD)
def test_bits_of_a_call_of_few_rows(M, K, N, group):
    w = ops.quantize_w4(make(K, N, K + N).to(DEV), group)
    x = make(M, K, M + K, 1.0).to(DEV)
    for dtype in (torch.float16, torch.float32):
        full = ops.det_matmul_w4(x, w, dtype)
        for rows in (slice(0, 1), slice(M // 2, M // 2 + 16), slice(M - 3, M), slice(0, 48), slice(M - 20, M)):
            assert torch.equal(ops.det_matmul_w4(x[rows], w, dtype), full[rows])
        pick = torch.arange(0, M, max(1, M // 40), device=DEV)[:40]
        assert torch.equal(check(x[pick].contiguous(), w, dtype), full[pick])


@pytest.mark.parametrize("group", [32, 64, 128])
def test_head_sized_products(group):
    w = ops.quantize_w4(make(768, 50277, 3).to(DEV), group)
    x = make(512, 768, 4, 1.0).to(DEV)
    for dtype in (torch.float16, torch.float32):
        full = ops.det_matmul_w4(x, w, dtype)
        for M in (1, 5, 16, 17, 40, 100):
            assert torch.equal(ops.det_matmul_w4(x[:M], w, dtype), full[:M]), M
        check(x[:5], w, dtype)
        del full


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [HELD[0], HELD[2], HELD[4]])
def test_epilogues(M, K, N, group):
    w = ops.quantize_w4(make(K, N, 9).to(DEV), group)
    x, res, gate = make(M, K, 1, 1.0).to(DEV), make(M, N, 2, 1.0).to(DEV), make(M, N, 3, 1.0).to(DEV)
    h16 = ops.det_matmul_w4(x, w)
    assert torch.equal(ops.det_matmul_w4(x, w, torch.float32).half(), h16)
    h = h16.float()
    assert torch.equal(ops.det_matmul_w4(x, w, epilogue="relu2"), (torch.relu(h) ** 2).half())
    assert torch.equal(ops.det_matmul_w4(x, w, epilogue="residual", res=res), (res.float() + h).half())
    assert torch.equal(ops.det_matmul_w4(x, w, epilogue="gated", res=res, gate=gate),
                       (res.float() + (gate.float() * h).half().float()).half())
    # exp and two operations, a few ulp of fp32, before the rounding to fp16
    got = ops.det_matmul_w4(x, w, epilogue="sigmoid").double()
    ref = torch.sigmoid(h.double())
    assert ((got - ref).abs() <= 2.0 ** -11 * ref * (1 + 2.0 ** -8) + 2.0 ** -25).all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [HELD[0], HELD[2], HELD[4]])
def test_non_finite_inputs_stay_in_their_row_and_output(M, K, N, group):
    W = make(K, N, 5)
    W[K - 1, 7] = float("nan")
    W[3, N - 1] = float("inf")
    w = ops.quantize_w4(W.to(DEV), group)
    x = make(M, K, 6, 1.0).to(DEV)
    x[3, 5] = float("nan")
    x[M - 1, K - 1] = float("inf")
    good = torch.isfinite(ops.det_matmul_w4(x, w))
    want = torch.ones_like(good)
    want[:, [7, N - 1]] = False
    want[[3, M - 1]] = False
    assert not good[3].any() and not good[:, [7, N - 1]].any() and good[want].all()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,N", [(3, 100), (40, 100), (9, 24601), (250, 12333), (520, 12333)])
def test_subnormal_inputs_and_scales(M, N, group):
    """fp16 below 2^-14 is not flushed, in x nor in a scale."""
    K = 160
    w = ops.quantize_w4(make(K, N, 2, 2.0 ** -16).to(DEV), group)
    assert (w.scales.abs() < 2.0 ** -14).all() and w.scales.any()
    x = make(M, K, 3, 2.0 ** -16).to(DEV)
    y = ops.det_matmul_w4(x, w, torch.float32)
    assert y.any()
    assert torch.equal(check(x[:40].contiguous(), w, torch.float32), y[:40])
