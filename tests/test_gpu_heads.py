"""WKV with heads (kr_wkv_heads): both forms against the recurrence in float64,
token-by-token calls bit for bit, ragged and padded streams, strides, decays at
both ends, ranges that fp16 parts have to be scaled for."""
import numpy as np
import pytest
import torch

from krunch_amd import _lib, krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def plain(r, k, v, w, u, S, lens=None):
    """y, state in float64 on the CPU, and the same sums over absolute values."""
    r, k, v, S = (t.double().cpu() for t in (r, k, v, S))
    w = w.double().cpu()
    g, u = torch.exp(torch.where(w > 0, torch.zeros_like(w), w))[None, :, None, None], u.double().cpu()
    u = u[None, :, None, None]
    B, T, H, D = r.shape
    n = torch.full((B,), T) if lens is None else lens.cpu().long().clamp(0, T)
    A = S.abs()
    y, size = torch.zeros_like(r), torch.zeros_like(r)
    for t in range(T):
        live = (t < n)[:, None, None, None]
        kv = k[:, t, :, :, None] * v[:, t, :, None, :]
        at = r[:, t, :, :, None]
        y[:, t] = torch.where(live[..., 0], (at * (S + u * kv)).sum(2), 0.0)
        size[:, t] = torch.where(live[..., 0], (at.abs() * (A + (u * kv).abs())).sum(2), 0.0)
        S, A = torch.where(live, g * S + kv, S), torch.where(live, g * A + kv.abs(), A)
    return y, S, size, A


def make(B, T, H, D, seed, amp=0.5):
    g = torch.Generator().manual_seed(seed)
    r, k, v = ((a * torch.randn(B, T, H, D, generator=g)).half().to(DEV) for a in (amp, amp, 1.0))
    w = -torch.exp(torch.linspace(-6.0, 1.0, H)).to(DEV)
    u = (0.2 + torch.rand(H, generator=g)).to(DEV)
    return r, k, v, w, u, torch.randn(B, H, D, D, generator=g).to(DEV)


def check(r, k, v, w, u, S, lens=None, chunked=True):
    ref_y, ref_S, size, size_S = plain(r, k, v, w, u, S, lens)
    y = ops.wkv_heads(r, k, v, w, u, S, lens, chunked)
    # recurrent: one fp32 rounding of each state element a token, which later
    # decays shrink with it, and the decay's own (2 of 2^-24 a token): T + 2 and
    # at most 3 T of 2^-24 together, 2 D more in y. chunked: parts carry 2^-22 of a
    # value, products of 3 factors of a few 2^-24, and 2^-38 of the largest
    # value of the row or columns it is scaled with: 2^-20 covers them for the
    # inputs here, beside the recurrent part of T / 64 chunks.
    T, D = r.shape[1], r.shape[3]
    eps = (4 * T + 2 * D + 8) * 2.0 ** -24
    if chunked:
        eps += 2.0 ** -20
    err = (y.double().cpu() - ref_y).abs()
    tol = eps * size + 2.0 ** -11 * ref_y.abs() + 2.0 ** -25 + eps * size.amax(3, keepdim=True) * 2.0 ** -14
    assert (err <= tol).all(), (err / tol).max()
    err = (S.double().cpu() - ref_S).abs()
    tol = eps * size_S + eps * 2.0 ** -14 * size_S.amax((2, 3), keepdim=True)
    assert (err <= tol).all(), (err / tol).max()
    return y


@pytest.mark.parametrize("B,T,H,D", [(1, 1, 1, 64), (3, 1, 4, 128), (2, 2, 3, 64), (2, 16, 12, 64),
                                     (1, 40, 2, 128), (2, 100, 3, 64)])
def test_recurrent(B, T, H, D):
    check(*make(B, T, H, D, B + T + H), chunked=False)


# the last length of the recurrent form, around one and two chunks, and around the
# lengths where the time axis splits; many heads (no split) and few
@pytest.mark.parametrize("B,T,H,D", [(2, 8, 3, 64), (2, 9, 3, 64), (1, 17, 1, 64), (2, 63, 2, 64), (1, 64, 3, 64), (3, 65, 4, 64),
                                     (1, 127, 2, 128), (2, 128, 1, 128), (1, 129, 2, 64), (1, 257, 2, 128),
                                     (1, 640, 1, 64), (50, 200, 12, 64), (40, 130, 16, 64), (70, 70, 8, 128),
                                     (1, 1000, 12, 64), (1, 1000, 4, 128)])
def test_chunked(B, T, H, D):
    check(*make(B, T, H, D, B + T + H))


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("B,T,H,D", [(7, 150, 2, 64), (9, 400, 1, 128), (130, 90, 4, 64), (6, 3, 2, 64),
                                     (300, 70, 1, 64), (257, 40, 2, 128)])
def test_ragged_streams(B, T, H, D, chunked):
    """Lengths of none, one, a chunk, all and out of range; NaN in the padding."""
    args = make(B, T, H, D, B + T)
    g = torch.Generator().manual_seed(1)
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32)
    lens[:6] = torch.tensor([0, 1, min(64, T), T, T + 9, -4], dtype=torch.int32)
    for b in range(B):
        for x in args[:3]:
            x[b, max(0, int(lens[b])):] = float("nan")
    clean = [torch.nan_to_num(x) for x in args[:3]]
    S = args[5].clone()
    ref = check(*clean, *args[3:5], S, lens.to(DEV), chunked)
    got = ops.wkv_heads(*args, lens.to(DEV), chunked)
    assert torch.equal(got, ref) and torch.equal(args[5], S)
    for b in range(B):
        assert not got[b, max(0, int(lens[b])):].any()


@pytest.mark.parametrize("D", [64, 128])
def test_tokens_in_one_call_equal_tokens_one_by_one(D):
    B, T, H = 3, 37, 4
    r, k, v, w, u, S = make(B, T, H, D, 5)
    S1, S2 = S.clone(), S.clone()
    y = ops.wkv_heads(r, k, v, w, u, S, chunked=False)
    one = [ops.wkv_heads(*(x[:, t:t + 1].contiguous() for x in (r, k, v)), w, u, S1) for t in range(T)]
    assert torch.equal(torch.cat(one, 1), y) and torch.equal(S1, S)
    # and a stream does not depend on the others
    yb = ops.wkv_heads(r[1:2], k[1:2], v[1:2], w, u, S2[1:2].contiguous(), chunked=False)
    assert torch.equal(yb, y[1:2])


def test_a_prompt_then_tokens():
    r, k, v, w, u, S = make(2, 140, 4, 64, 6)
    S1 = S.clone()
    ref, _, size, _ = plain(r, k, v, w, u, S)
    y = torch.cat([ops.wkv_heads(*(x[:, a:b] for x in (r[:1], k[:1], v[:1])), w, u, S1[:1])
                   for a, b in ((0, 100), (100, 120), (120, 121), (121, 140))], 1)
    err = (y.double().cpu() - ref[:1]).abs()
    assert (err <= 2.0 ** -11 * ref[:1].abs() + 2.0 ** -15 * size[:1]).all()


@pytest.mark.parametrize("chunked", [False, True])
def test_decays_at_both_ends(chunked):
    """No decay, above 0 (counts as 0), no memory, almost none, subnormal powers."""
    r, k, v, w, u, S = make(2, 150, 6, 64, 8)
    w[:] = torch.tensor([0.0, 0.7, -float("inf"), -90.0, -1.0, -1e-9])
    check(r, k, v, w, u, S, chunked=chunked)
    r, k, v, w, u, S = make(1, 70, 2, 64, 9)
    w[0] = float("nan")
    y = ops.wkv_heads(r, k, v, w, u, S, chunked=chunked)
    assert torch.isnan(y[:, 2:, 0]).all() and torch.isfinite(y[:, :, 1]).all()


@pytest.mark.parametrize("chunked", [False, True])
@pytest.mark.parametrize("a,b,c", [(200.0, 200.0, 1e-4), (1e-4, 1e-4, 1e3), (1e-3, 300.0, 300.0),
                                   (300.0, 1e-3, 1e-3)])
def test_ranges(a, b, c, chunked):
    """r k, v and the state past fp16's largest and below its smallest numbers,
    and columns of v of very different sizes."""
    r, k, v, w, u, S = make(1, 200, 2, 64, 11, 1.0)
    r, k, v = r * a, k * b, v * c
    v[..., ::3] *= 2.0 ** -6
    S = S * (b * c)
    check(r.half(), k.half(), v.half(), w, u, S, chunked=chunked)
    zero = torch.zeros_like(r)
    S = torch.zeros_like(S)
    y = ops.wkv_heads(zero, zero, zero, w, u, S, chunked=chunked)
    assert not y.any() and not S.any()


def test_slices_of_one_projection():
    B, T, H, D = 3, 130, 4, 64
    big = torch.randn(B, T, 3 * H * D + 8, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    r, k, v = (big[..., 8 + i * H * D:8 + (i + 1) * H * D].unflatten(2, (H, D)) for i in range(3))
    _, _, _, w, u, S = make(B, T, H, D, 3)
    S1, S2 = S.clone(), S.clone()
    a = ops.wkv_heads(r, k, v, w, u, S1)
    b = ops.wkv_heads(r.contiguous(), k.contiguous(), v.contiguous(), w, u, S2)
    assert torch.equal(a, b) and torch.equal(S1, S2)


@pytest.mark.parametrize("T", [1, 90, 300])
def test_rows_past_the_call_stay(T):
    """y by a wider stride: nothing between its rows or behind the last is written."""
    B, H, D = 2, 2, 64
    r, k, v, w, u, S = make(B, T, H, D, 4)
    S1 = S.clone()
    ref = ops.wkv_heads(r, k, v, w, u, S1)
    ld = H * D + 16
    y = torch.full((B * T + 30, ld), 2.5, dtype=torch.float16, device=DEV)
    nbytes = _lib.lib().kr_wkv_heads_workspace_bytes(B, T, H, D)
    ws = torch.empty(nbytes + 64, dtype=torch.uint8, device=DEV)
    _lib.call("kr_wkv_heads", B, T, H, D, r.data_ptr(), H * D, k.data_ptr(), H * D, v.data_ptr(), H * D,
              w.data_ptr(), u.data_ptr(), None, S.data_ptr(), y.data_ptr(), ld, 1, ws.data_ptr(), nbytes,
              _lib.stream_ptr())
    assert torch.equal(y[:B * T, :H * D].reshape(B, T, H, D), ref) and torch.equal(S, S1)
    assert (y[B * T:] == 2.5).all() and (y[:, H * D:] == 2.5).all()


@pytest.mark.parametrize("B,T,H", [(2, 1, 4), (1, 300, 2)])
def test_nothing_to_do_another_stream_and_a_graph(B, T, H):
    D = 64
    r, k, v, w, u, S = make(B, T, H, D, 6)
    before = S.clone()
    empty = torch.empty(B, 0, H, D, dtype=torch.float16, device=DEV)
    assert ops.wkv_heads(empty, empty, empty, w, u, S).shape == (B, 0, H, D)
    none = torch.empty(0, T, H, D, dtype=torch.float16, device=DEV)
    ops.wkv_heads(none, none, none, w, u, torch.empty(0, H, D, D, device=DEV))
    assert torch.equal(S, before)
    ref = ops.wkv_heads(r, k, v, w, u, S)
    S2 = before.clone()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = ops.wkv_heads(r, k, v, w, u, S2)
    side.synchronize()
    assert torch.equal(got, ref) and torch.equal(S, S2)
    # two graphs captured one after the other and replayed in turn
    Sg = [before.clone(), before.clone()]
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(ops.wkv_heads(r, k, v, w, u, Sg[i]))
    Se = before.clone()
    for seed in (21, 22, 23):
        x = make(B, T, H, D, seed)
        for a, b in zip((r, k, v), x):
            a.copy_(b)
        eager = ops.wkv_heads(r, k, v, w, u, Se)
        for i in range(2):
            graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(outs[i], eager) and torch.equal(Sg[i], Se)


def test_refusals():
    B, T, H, D = 2, 5, 2, 64
    r, k, v, w, u, S = make(B, T, H, D, 1)
    before = S.clone()
    lens = torch.tensor([1, 2], dtype=torch.int32, device=DEV)
    wide = torch.zeros(B, T + 1, H, D, dtype=torch.float16, device=DEV)[:, :T]
    for args in ((r.float(), k, v, w, u, S), (r, k[:1], v, w, u, S), (r, k, v.cpu(), w, u, S), (r[0], k, v, w, u, S),
                 (r[..., :32], k[..., :32], v[..., :32], w, u, S), (wide, k, v, w, u, S),
                 (r.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2), w, u, S), (r, k, v, w[:1], u, S),
                 (r, k, v, w, u.double(), S), (r, k, v, w, u, S[:1]), (r, k, v, w, u, S.half()),
                 (r, k, v, w, u, S.transpose(2, 3)), (r, k, v, w, u, S, lens[:1]), (r, k, v, w, u, S, lens.long()),
                 (r[:, :1].expand(B, T, H, D), k, v, w, u, S)):
        with pytest.raises(RuntimeError):
            ops.wkv_heads(*args)
    assert torch.equal(S, before)


def test_a_long_prompt():
    """Many segments of the time axis, sums over thousands of tokens."""
    r, k, v, w, u, S = make(1, 5000, 2, 64, 14)
    check(r, k, v, w, u, S)


@pytest.mark.parametrize("chunked", [False, True])
def test_offsets_past_32_bits(chunked):
    """Token strides of 2^27 elements, and states of more than 2^31."""
    B, T, H, D, ld = 1, 20, 2, 64, 1 << 27
    r, k, v, w, u, S = make(B, T, H, D, 9)
    wide = torch.empty(T * ld, dtype=torch.float16, device=DEV)
    views = []
    for i, x in enumerate((r, k, v)):
        views.append(wide.as_strided((B, T, H, D), (T * ld, ld, D, 1), ld - (3 - i) * H * D))
        views[-1].copy_(x)
    S2 = S.clone()
    assert torch.equal(ops.wkv_heads(*views, w, u, S2, chunked=chunked), ops.wkv_heads(r, k, v, w, u, S, chunked=chunked))
    assert torch.equal(S, S2)
    del wide, views
    B, T, H, D = 8200, 9, 16, 128
    r, k, v, w, u, S = make(2, T, H, D, 10)
    big = torch.zeros(B, H, D, D, device=DEV)
    assert big.numel() > 2 ** 31
    big[-2:] = S
    many = [torch.zeros(B, T, H, D, dtype=torch.float16, device=DEV) for _ in range(3)]
    for m, x in zip(many, (r, k, v)):
        m[-2:] = x
    y = ops.wkv_heads(*many, w, u, big, chunked=chunked)
    assert torch.equal(y[-2:], ops.wkv_heads(r, k, v, w, u, S, chunked=chunked))
    assert torch.equal(big[-2:], S) and not y[:-2].any() and not big[:-2].any()
