"""Products with 4-bit weights (kr_quantize_w4, kr_det_matmul_w4): the packed
form against a plain quantiser, the products against float64 on the values that
q and scales stand for, every epilogue, and each row's independence of M."""
import numpy as np
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain_quantize(W, group):
    """W [K, N] float16 (numpy) -> q [K, N] int, s [groups, N] float16."""
    K, N = W.shape
    groups = -(-K // group)
    q = np.zeros((K, N), np.int64)
    s = np.zeros((groups, N), np.float16)
    for g in range(groups):
        w = W[g * group:(g + 1) * group].astype(np.float32)
        ok = np.isfinite(w).all(0)
        with np.errstate(all="ignore"):
            sg = (np.abs(w).max(0) / np.float32(7)).astype(np.float16)
            sg[~ok] = np.nan
            v = np.rint(w.astype(np.float64) / sg.astype(np.float64))
        live = ok & (sg > 0)
        q[g * group:(g + 1) * group] = np.where(live, np.clip(np.nan_to_num(v), -7, 7), 0)
        s[g] = sg
    return q, s


def unpacked(w):
    """q [K, N] of a W4, from the documented layout; padding must be q = 0."""
    K, N = w.K, w.N
    words = w.q.cpu().numpy().view(np.uint32).reshape(-(-N // 16), -(-K // 128), 64, 4)
    full = np.zeros((words.shape[1] * 128, words.shape[0] * 16), np.int64)
    for place, e in enumerate((0, 2, 4, 6, 1, 3, 5, 7)):
        nib = (words >> np.uint32(4 * place) & np.uint32(15)).astype(np.int64) - 8
        for l in range(64):
            for c in range(4):
                k = 32 * c + 8 * (l // 16) + e
                full[k::128, l % 16::16] = nib[:, :, l, c].T
    assert not full[K:].any() and not full[:, N:].any()
    return full[:K, :N]


def values(w):
    s = w.scales.cpu().numpy().astype(np.float64)[:, :w.N]
    return unpacked(w) * np.repeat(s, w.group, axis=0)[:w.K]


def make(K, N, seed, scale=None):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(K, N, generator=g) * (scale or K ** -0.5)).half()


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("K,N", [(32, 1), (96, 15), (128, 16), (160, 17), (768, 300), (1056, 257)])
def test_quantize(K, N, group):
    W = make(K, N, K + N)
    W[:, 0] = 0.0                                 # groups of zeros
    W[0, N - 1] = 65504.0                         # a group's other values vanish beside it
    if N > 2:
        W[:, 1] = torch.arange(K) % 15 - 7.0      # every quotient an integer
        W[:, 2] = (torch.arange(K) % 29 - 14.0) / 2 * 2.0 ** -20    # ties, subnormal scale
    if N > 20:
        W[5, 3] = float("nan"); W[40, 4] = float("inf"); W[7, 5] = -float("inf")
        W[:, 6] = 2.0 ** -24                      # scale rounds to zero
    q, s = plain_quantize(W.numpy(), group)
    for view in (W.to(DEV), W.t().contiguous().to(DEV).t()):
        w = ops.quantize_w4(view, group)
        assert np.array_equal(unpacked(w), q)
        got = w.scales.cpu().numpy()
        assert np.array_equal(got[:, :N], s, equal_nan=True) and not got[:, N:].any()


def check(x, w, out_dtype=torch.float16):
    y = ops.det_matmul_w4(x, w, out_dtype)
    xs, V = x.cpu().numpy().astype(np.float64), values(w)
    ref, size = xs @ V, np.abs(xs) @ np.abs(V)
    # fp32: at most K additions and one scaling, each within 2^-24 of a partial
    # sum no larger than `size`; fp16: half a step of the result, or of the
    # smallest subnormal, on top
    tol = (w.K + 2) * 2.0 ** -24 * size
    if out_dtype == torch.float16:
        tol = tol + 2.0 ** -11 * np.abs(ref) * (1 + 1e-3) + 2.0 ** -25
    got = y.double().cpu().numpy()
    assert (np.abs(got - ref) <= tol).all(), np.abs(got - ref).max()
    return y


# one group and less than a block; partial blocks and groups; slices of 512 and
# a last one of 32; outputs around 16; rows around every tile height
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("M,K,N", [(1, 32, 1), (3, 96, 15), (1, 160, 17), (16, 512, 48), (17, 544, 33),
                                   (1, 768, 768), (32, 768, 100), (33, 1056, 64), (65, 768, 2100),
                                   (7, 4096, 70), (130, 1024, 1000), (257, 288, 523), (16, 1984, 48),
                                   (15, 2080, 100), (16, 8192, 20), (3, 5152, 25000)])
def test_products(M, K, N, group):
    w = ops.quantize_w4(make(K, N, M + K + N).to(DEV), group)
    x = make(M, K, 7 * M + K, 1.0).to(DEV)
    check(x, w)
    check(x, w, torch.float32)


def test_head_sized_product():
    w = ops.quantize_w4(make(768, 50277, 3).to(DEV), 64)
    for M in (1, 5, 40):
        check(make(M, 768, M, 1.0).to(DEV), w)


@pytest.mark.parametrize("K,N,group", [(768, 777, 64), (1536, 64, 32), (512, 4100, 128)])
def test_a_row_does_not_depend_on_the_others(K, N, group):
    w = ops.quantize_w4(make(K, N, 5).to(DEV), group)
    x = make(600, K, 6, 1.0).to(DEV)
    for dtype in (torch.float16, torch.float32):
        full = ops.det_matmul_w4(x, w, dtype)
        for M in (1, 2, 16, 17, 40, 64, 65, 128, 129, 300, 512):
            assert torch.equal(ops.det_matmul_w4(x[:M], w, dtype), full[:M]), M
            assert torch.equal(ops.det_matmul_w4(x[600 - M:], w, dtype), full[600 - M:]), M


@pytest.mark.parametrize("M,N", [(1, 64), (20, 101), (70, 768), (300, 770)])
def test_epilogues(M, N):
    K = 768
    w = ops.quantize_w4(make(K, N, 9).to(DEV), 64)
    x, res, gate = make(M, K, 1, 1.0).to(DEV), make(M, N, 2, 1.0).to(DEV), make(M, N, 3, 1.0).to(DEV)
    h = ops.det_matmul_w4(x, w).float()
    f16 = lambda t: t.half().float()
    exact = lambda got, ref: torch.equal(got, ref.half())
    assert exact(ops.det_matmul_w4(x, w, epilogue="relu2"), torch.relu(h) ** 2)
    assert exact(ops.det_matmul_w4(x, w, epilogue="residual", res=res), res.float() + h)
    assert exact(ops.det_matmul_w4(x, w, epilogue="gated", res=res, gate=gate),
                 res.float() + f16(gate.float() * h))
    # exp and two operations, a few ulp of fp32, before the rounding to fp16
    got = ops.det_matmul_w4(x, w, epilogue="sigmoid").double()
    ref = torch.sigmoid(h.double())
    assert ((got - ref).abs() <= 2.0 ** -11 * ref * (1 + 2.0 ** -8) + 2.0 ** -25).all()


@pytest.mark.parametrize("M,K,N", [(200, 768, 16400), (800, 256, 12333), (1000, 1280, 8200), (333, 1312, 16384),
                                   (700, 2560, 8192), (5000, 128, 9000), (20000, 96, 1030)])
def test_many_rows(M, K, N):
    """Around the lines between tiles and held rows: the rows of a call of 48."""
    w = ops.quantize_w4(make(K, N, 5).to(DEV), 64)
    x = make(M, K, 6, 1.0).to(DEV)
    full = ops.det_matmul_w4(x, w)
    for m in (0, M // 2, M - 48):
        assert torch.equal(ops.det_matmul_w4(x[m:m + 48], w), full[m:m + 48]), m
    check(x[:48], w)


def test_all_values_of_a_nibble():
    """q = -8 is in the format, though the quantiser does not use it."""
    K, N = 128, 16
    q = torch.randint(-2 ** 31, 2 ** 31, (N * 16,), dtype=torch.int64).to(torch.int32).to(DEV)
    scales = torch.rand(2, 16).half().to(DEV)
    check(make(9, K, 4, 1.0).to(DEV), ops.W4(q, scales, K, N, 64), torch.float32)


def test_strided_rows_and_out_of_range_rows_untouched():
    from krunch_amd import _lib
    K, N, M = 768, 301, 21
    w = ops.quantize_w4(make(K, N, 5).to(DEV), 64)
    wide = make(M, K + 24, 8, 1.0).to(DEV)
    x = wide[:, 16:16 + K]
    ref = ops.det_matmul_w4(x.contiguous(), w)
    assert torch.equal(ops.det_matmul_w4(x, w), ref)
    out = torch.full((M + 40, N + 7), 3.5, dtype=torch.float16, device=DEV)
    _lib.call("kr_det_matmul_w4", x.data_ptr(), K + 24, M, K, w.q.data_ptr(), w.scales.data_ptr(), 64,
              N, out.data_ptr(), N + 7, 1, None, None, _lib.stream_ptr())
    assert torch.equal(out[:M, :N], ref)
    assert (out[M:] == 3.5).all() and (out[:, N:] == 3.5).all()


def test_non_finite_inputs_stay_in_their_row_and_output():
    K, N = 768, 40
    W = make(K, N, 5)
    W[100, 7] = float("nan")
    w = ops.quantize_w4(W.to(DEV), 64)
    x = make(18, K, 6, 1.0).to(DEV)
    x[3, 5] = float("nan")
    x[17, 767] = float("inf")
    y = ops.det_matmul_w4(x, w)
    bad = ~torch.isfinite(y)
    assert bad[:, 7].all() and bad[3].all() and bad[17].all()
    rows = [i for i in range(18) if i not in (3, 17)]
    cols = [i for i in range(N) if i != 7]
    assert not bad[rows][:, cols].any()


def test_no_rows_another_stream_and_a_graph():
    K, N = 768, 768
    w = ops.quantize_w4(make(K, N, 5).to(DEV), 64)
    assert ops.det_matmul_w4(torch.empty(0, K, dtype=torch.float16, device=DEV), w).shape == (0, N)
    x = make(3, K, 6, 1.0).to(DEV)
    ref = ops.det_matmul_w4(x, w)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.det_matmul_w4(x, w)
    side.synchronize()
    assert torch.equal(got, ref)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.det_matmul_w4(x, w)
    for seed in (1, 2, 3):
        y = make(3, K, seed, 1.0).to(DEV)
        x.copy_(y)
        graph.replay()
        eager = ops.det_matmul_w4(y, w)
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


def test_refusals():
    W = make(768, 40, 1).to(DEV)
    w = ops.quantize_w4(W)
    x = make(3, 768, 2, 1.0).to(DEV)
    res = torch.zeros(3, 40, dtype=torch.float16, device=DEV)
    for args in ((W[:40],), (W.float(),), (W[0],), (W, 16), (W[:, :0],), (W[:, :1].expand(768, 5),)):
        with pytest.raises(RuntimeError):
            ops.quantize_w4(*args)
    W4 = ops.W4
    for args in ((x.float(), w), (x[0], w), (x[:, :736], w), (x[:, 1:], w), (x[:1].expand(3, 768), w),
                 (make(3, 1536, 2).to(DEV)[:, ::2], w), (x, w, torch.bfloat16), (x, w, None, "tanh"),
                 (x, w, torch.float32, "relu2"), (x, w, None, "residual"), (x, w, None, "none", res),
                 (x, w, None, "gated", res), (x, w, None, "residual", res[:2]), (x, w, None, "residual", res.float()),
                 (x, W4(w.q[:-1], w.scales, 768, 40, 64)), (x, W4(w.q, w.scales[1:], 768, 40, 64)),
                 (x, W4(w.q, w.scales, 768, 56, 64)), (x, W4(w.q, w.scales, 768, 40, 32)),
                 (x, W4(w.q.cpu(), w.scales, 768, 40, 64)), (x, W4(w.q.float(), w.scales, 768, 40, 64))):
        with pytest.raises(RuntimeError):
            ops.det_matmul_w4(*args)


def test_offsets_past_32_bits():
    """x rows and out rows that start more than 2^31 elements after the first."""
    from krunch_amd import _lib
    K, N, ld = 64, 48, 2 ** 30 + 8
    w = ops.quantize_w4(make(K, N, 1).to(DEV), 32)
    x = make(3, K, 2, 1.0).to(DEV)
    wide = torch.empty(2 * ld + K, dtype=torch.float16, device=DEV).as_strided((3, K), (ld, 1))
    wide.copy_(x)
    out = torch.empty(2 * ld + N, dtype=torch.float16, device=DEV).as_strided((3, N), (ld, 1))
    _lib.call("kr_det_matmul_w4", wide.data_ptr(), ld, 3, K, w.q.data_ptr(), w.scales.data_ptr(), 32, N,
              out.data_ptr(), ld, 1, None, None, _lib.stream_ptr())
    assert torch.equal(out.contiguous(), ops.det_matmul_w4(x, w))
