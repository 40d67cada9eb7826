"""Scores of tokens (kr_token_scores) against a plain log-softmax in 64 bits:
widths around every kernel's and segment's edge, both types, strided and
misaligned rows, masks up to whole rows, ties, NaN and infinities."""
import numpy as np
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(x, tokens, k):
    """The definition in float64 on the CPU: logprob, entropy, top by (value, lower id)."""
    z = x.double().cpu().numpy()
    t = tokens.cpu().numpy()
    N, V = z.shape
    lp, h = np.full(N, np.nan), np.full(N, np.nan)
    tl, tt = np.full((N, k), np.nan), np.full((N, k), -1, np.int32)
    for i in range(N):
        r = z[i]
        if not (np.isnan(r).any() or np.isposinf(r).any()):
            live = r > -np.inf
            if live.any():
                m = r.max()
                s = np.exp(r[live] - m).sum()
                logp = r - m - np.log(s)
                p = np.exp(logp[live])
                h[i] = -(p * logp[live]).sum()
                order = np.argsort(-r, kind="stable")[:k]
                order = order[r[order] > -np.inf]
                tl[i] = -np.inf
                tl[i, :len(order)] = logp[order]
                tt[i, :len(order)] = order
                lp[i] = logp[t[i]] if 0 <= t[i] < V else np.nan
            else:
                h[i], tl[i] = 0.0, -np.inf
                lp[i] = -np.inf if 0 <= t[i] < V else np.nan
        if t[i] == -1:
            lp[i] = 0.0
    return lp, h, tl, tt


def check(x, tokens, k):
    lp, h, tl, tt = (a.cpu().numpy() for a in ops.token_scores(x, tokens, k))
    rlp, rh, rtl, rtt = plain(x, tokens, k)
    # fp32 throughout. ln s: a thread's chain of V / 512 additions (V / 64 below
    # 2049, at most 64 otherwise up to V = 32768), 6 levels in the wave, 8 waves,
    # and the exponents' last bits, under 128 * 2^-24 in all; at V = 151937, where
    # the chain has 297, that takes the additions' errors to differ in sign. x - m
    # and the difference are rounded at their own size, at most 2^-22 of it together.
    tol = lambda r: 2.0 ** -17 + 2.0 ** -22 * np.abs(np.where(np.isfinite(r), r, 0))
    for got, ref in ((lp, rlp), (tl, rtl)):
        assert np.array_equal(np.isnan(got), np.isnan(ref))
        fin = np.isfinite(ref)
        assert np.array_equal(got[~fin & ~np.isnan(ref)], ref[~fin & ~np.isnan(ref)])
        assert (np.abs(got[fin] - ref[fin]) <= tol(ref)[fin]).all(), np.abs(got[fin] - ref[fin]).max()
    assert np.array_equal(np.isnan(h), np.isnan(rh))
    fin = ~np.isnan(rh)
    # sum of e * a: each factor as above, |a| e^a <= 1/e per term
    assert (np.abs(h[fin] - rh[fin]) <= 2.0 ** -16 + 2.0 ** -18 * rh[fin]).all()
    assert np.array_equal(tt, rtt)
    return lp, h, tl, tt


def rand(N, V, dtype, seed, scale=3.0):
    g = torch.Generator().manual_seed(seed)
    x = (scale * torch.randn(N, V, generator=g)).to(dtype).to(DEV)
    tok = torch.randint(0, V, (N,), generator=g, dtype=torch.int32).to(DEV)
    return x, tok


# one element; around a chunk, a wave's row, four waves' row, sixteen waves' row
# and one segment of it, by type; the codec's vocabulary; several segments
@pytest.mark.parametrize("dtype,V", [(torch.float16, v) for v in (
    1, 2, 7, 8, 9, 127, 255, 256, 257, 511, 512, 513, 2047, 2048, 2049, 8191, 8192, 8193, 50277, 65535, 65536,
    65537, 131080, 151937)] + [(torch.float32, v) for v in (
    1, 3, 4, 5, 63, 255, 256, 257, 511, 512, 513, 1023, 1024, 1025, 4096, 4097, 32768, 32769, 50277, 65543)])
def test_widths(dtype, V):
    x, tok = rand(5, V, dtype, V)
    check(x, tok, min(V, 9))
    check(x, tok, min(V, 8))      # (short rows have a kernel up to 8)
    check(x, tok, 0)


@pytest.mark.parametrize("k", [0, 1, 2, 8, 9, 20, 31, 32])
@pytest.mark.parametrize("V", [256, 1500, 5000, 50277, 70001])
def test_top_counts(V, k):
    x, tok = rand(3, V, torch.float16, V + k)
    check(x, tok, k)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [200, 300, 600, 3000, 9000, 66000])
def test_ties_clusters_and_long_candidate_lists(dtype, V):
    """All equal, many equal maxima, sorted up and down, all mass in one chunk,
    zeros of both signs: lists that overflow and ranks by id."""
    x, tok = rand(8, V, dtype, V)
    x[0] = 1.5
    x[1] = -65504.0
    x[2] = torch.round(x[2])
    x[3] = torch.sort(x[3]).values
    x[4] = torch.sort(x[4], descending=True).values
    x[5, 100:140] += 30
    x[6] = 0.0
    x[6, ::2] = -0.0
    x[7] = torch.clamp(x[7], max=1.0)
    check(x, tok, 5)
    check(x, tok, 17)
    check(x, tok, 32)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("V", [200, 2000, 8000, 50277, 140000])
def test_masks_nan_and_infinities(dtype, V):
    x, tok = rand(12, V, dtype, 7 * V)
    inf = float("inf")
    x[0] = -inf                                   # nothing left
    x[1] = -inf; x[1, V - 1] = -3.0               # one token, the last
    x[2] = -inf; x[2, 0] = 7.0; tok[2] = 0        # one token, the first
    x[3, ::3] = -inf; tok[3] = 0                  # a masked token asked for
    x[4, 17] = float("nan")
    x[5, V - 1] = inf
    x[6, 5] = inf; x[6, 6] = -inf
    x[7] = float("nan")
    x[8] = torch.finfo(dtype).min                 # the type's lowest value everywhere
    x[9] = torch.finfo(dtype).min; x[9, 9] = 2.0
    x[10] = -inf; x[10, 50:54] = 1.0              # fewer than asked for
    x[11, :] = -inf; x[11, 3] = float("nan")      # NaN among masked ones
    tok[6] = -1
    check(x, tok, 10)
    check(x, tok, 6)
    check(x, tok, 0)


def test_large_values():
    x, tok = rand(4, 1000, torch.float16, 3)
    x[0, 5] = 65504.0; tok[0] = 5
    x[1] = 65504.0
    x[2] = -65504.0; x[2, 1] = 65504.0; tok[2] = 0
    check(x, tok, 5)
    y, tok = rand(4, 1000, torch.float32, 4)
    y[0] = -3.4e38
    y[1] = 3.4e38
    y[2] = -1e38; y[2, 7] = 1e38; tok[2] = 7
    check(y, tok, 5)


def test_rows_without_a_token_and_ids_out_of_range():
    x, tok = rand(6, 777, torch.float16, 5)
    tok[:] = torch.tensor([-1, 776, 777, -2, 0, 2 ** 31 - 1], dtype=torch.int32)
    lp, h, tl, tt = check(x, tok, 3)
    assert lp[0] == 0 and np.isnan(lp[[2, 3, 5]]).all() and (tt >= 0).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strided_and_misaligned_rows(dtype):
    """Rows of a wider buffer at every offset: same bits as the row alone."""
    V = 4999
    x, tok = rand(9, V, dtype, 11)
    ref = [a.cpu() for a in ops.token_scores(x, tok, 8)]
    for off in range(1, 9):
        wide = torch.full((9, V + 13 + off), float("nan"), dtype=dtype, device=DEV)
        wide[:, off:off + V] = x
        got = ops.token_scores(wide[:, off:off + V], tok, 8)
        assert all(torch.equal(a, b.cpu()) for a, b in zip(ref, got)), off


@pytest.mark.parametrize("V", [256, 2000, 50277])
def test_a_row_does_not_depend_on_the_others(V):
    x, tok = rand(700, V, torch.float16, 13)
    all_rows = ops.token_scores(x, tok, 4)
    for i in (0, 1, 350, 699):
        one = ops.token_scores(x[i:i + 1], tok[i:i + 1], 4)
        assert all(torch.equal(a[i:i + 1], b) for a, b in zip(all_rows, one))


def test_offsets_past_32_bits():
    """Rows that start more than 2^31 elements after the first."""
    V, ld = 1000, 2 ** 30 + 8
    buf = torch.empty(3 * ld, dtype=torch.float16, device=DEV)
    view = buf.as_strided((3, V), (ld, 1))
    x, tok = rand(3, V, torch.float16, 17)
    view.copy_(x)
    ref, got = ops.token_scores(x, tok, 5), ops.token_scores(view, tok, 5)
    assert all(torch.equal(a, b) for a, b in zip(ref, got))


def test_no_rows_another_stream_and_a_graph():
    x, tok = rand(0, 50, torch.float16, 1)
    assert [tuple(a.shape) for a in ops.token_scores(x, tok, 2)] == [(0,), (0,), (0, 2), (0, 2)]
    x, tok = rand(33, 9000, torch.float16, 19)
    ref = ops.token_scores(x, tok, 6)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.token_scores(x, tok, 6)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(ref, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.token_scores(x, tok, 6)
    for seed in (23, 29, 31):
        y, _ = rand(33, 9000, torch.float16, seed)
        x.copy_(y)
        graph.replay()
        eager = ops.token_scores(y, tok, 6)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, out))


def test_refusals():
    x, tok = rand(4, 100, torch.float16, 1)
    bad = [(x.bfloat16(), tok, 0), (x.t(), tok, 0), (x.reshape(-1), tok, 0), (x[:1].expand(4, 100), tok, 0),
           (x, tok[:3], 0), (x, tok.long(), 0), (x, tok.cpu(), 0), (x, tok[None], 0), (x, tok, 33), (x, tok, -1),
           (x[:, :3], tok, 4), (x[:, :0], tok, 0), (x.repeat(2, 1)[::2, ::2], tok, 0)]
    for args in bad:
        with pytest.raises(RuntimeError):
            ops.token_scores(*args)
