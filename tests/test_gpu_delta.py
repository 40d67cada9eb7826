"""The gated delta rule (kr_gated_delta) and its gradients (kr_gated_delta_backward)
against the recurrence in float64: chunk edges, ragged streams, strides, decays at both
ends, repeated keys, values far apart, infinities, token-by-token bits, graphs."""
import pytest
import torch

from krunch_amd import _lib, krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(B, T, H, D, seed, ragged=False, rate=(-6.0, 0.7)):
    g = torch.Generator().manual_seed(seed)
    q, k, v = (torch.randn(B, T, H, D, generator=g) for _ in range(3))
    k = k / k.norm(dim=3, keepdim=True)
    decay = -torch.exp(torch.linspace(*rate, H)) * (0.5 + torch.rand(B, T, H, generator=g))
    beta = torch.sigmoid(torch.randn(B, T, H, generator=g))
    S = 0.5 * torch.randn(B, H, D, D, generator=g)
    lens = torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32) if ragged else None
    f = lambda t: t.to(DEV)  # noqa: E731
    return [f((q / D ** 0.5).half()), f(k.half()), f(v.half()), f(decay), f(beta), f(S),
            None if lens is None else f(lens)]


def lengths(q, lens):
    B, T = q.shape[:2]
    return torch.full((B,), T, device=q.device) if lens is None else lens.long().clamp(0, T)


def plain(q, k, v, a, b, S, lens=None, chunked=True):
    """y, state in float64, and bounds of their errors: E of a state column's 2-norm.
    I - beta k'k shrinks (beta |k|^2 <= 2), so a token adds its own roundings to E.
    Token by token: the state's scaling (2^-24, and 3 of the decay), a sum of D/16
    terms and 4 lanes, u's 3, the update's. Chunked: 2^-22 of what enters the matrix
    units (parts) and as much for their fp32 sums, of k S0, of all that the chunk's other
    tokens write, and in N and A of it again: 2^-20 of both."""
    q, k, v, a, b, S = (t.double() for t in (q, k, v, a, b, S))
    B, T, H, D = q.shape
    n = lengths(q, lens)
    y, ey = torch.zeros_like(q), torch.zeros_like(q)
    E = torch.zeros_like(S[:, :, 0])
    wrote = torch.zeros_like(E)
    start = S.norm(dim=2)
    for t in range(T):
        live = (t < n)[:, None, None]
        f = torch.exp(a[:, t].clamp_max(0))[..., None]
        if t % 64 == 0:
            wrote, start = torch.zeros_like(E), S.norm(dim=2)
        kk = k[:, t].norm(dim=2)[..., None]
        old = f[..., None] * S
        u = b[:, t, :, None] * (v[:, t] - (old * k[:, t, :, :, None]).sum(2))
        new = old + k[:, t, :, :, None] * u[:, :, None, :]
        bk = (b[:, t, :, None] * kk * kk).abs()
        add = 2.0 ** -24 * ((4 + bk * (D / 16 + 5)) * old.norm(dim=2) + 3 * u.abs() * kk + new.norm(dim=2))
        wrote = wrote + u.abs() * kk
        if chunked:
            add = add + 2.0 ** -20 * ((1 + bk) * (start + wrote) + b[:, t, :, None].abs() * kk * v[:, t].abs())
        grow = torch.clamp((1 - bk).abs(), min=1.0)
        S = torch.where(live[..., None], new, S)
        E = torch.where(live, f * grow * E + add, E)
        y[:, t] = torch.where(live, (S * q[:, t, :, :, None]).sum(2), 0.0)
        ey[:, t] = q[:, t].norm(dim=2)[..., None] * (E + 2.0 ** -20 * (new.norm(dim=2) + start + wrote))
    return y, S, ey, E


def check(q, k, v, a, b, S, lens=None, chunked=True, tight=1.0):
    want_y, want_S, ey, E = plain(q, k, v, a, b, S, lens, chunked)
    S = S.clone()
    y = ops.gated_delta(q, k, v, a, b, S, lens, chunked)
    off = (y.double() - want_y).abs()
    tol = ey + 2.0 ** -11 * want_y.abs() + 2.0 ** -25
    held = want_y.abs() + tol < 65504                  # by fp16; half a step further it is infinite
    assert (off[held] <= tol[held]).all(), (off[held] / tol[held]).max()
    assert torch.isinf(y[want_y.abs() - tol > 65520]).all()
    off = (S.double() - want_S).norm(dim=2)
    assert (off <= E + 1e-30).all(), (off / (E + 1e-30)).max()
    if tight and want_S.norm() > 0:
        # roundings of either sign, a few of 2^-22 a chunk that shrink with the state:
        # in 2-norm over all of it 8 of them, `tight` times where N enlarges them
        assert (S.double() - want_S).norm() <= tight * 2.0 ** -19 * want_S.norm()
    return y, S


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 2, 8, 9, 31, 33, 63, 64, 65, 127, 128, 129, 200])
def test_lengths(T, D):
    for chunked in (False, True):
        check(*make(2, T, 3, D, T + D), chunked=chunked)


@pytest.mark.parametrize("B,T,H,D", [(1, 1500, 2, 64), (70, 130, 1, 64), (300, 70, 1, 64), (3, 700, 4, 128),
                                     (513, 9, 2, 64)])
def test_ragged(B, T, H, D):
    args = make(B, T, H, D, B + T, ragged=True)
    args[6][0], args[6][-1] = T, 0
    if B > 2:
        args[6][1], args[6][2] = 2000000, -3          # clamped
    for t in range(3):                                # rows past a stream's end hold anything
        for i in range(B):
            args[t][i, min(T, max(0, int(args[6][i]))):] = float("nan")
    clean = [torch.nan_to_num(t) if i < 3 else t for i, t in enumerate(args)]
    want = [plain(*clean[:6], lens=args[6])]
    S = args[5].clone()
    y = ops.gated_delta(*args[:5], S, args[6])
    assert ((y.double() - want[0][0]).abs() <= want[0][2] + 2.0 ** -11 * want[0][0].abs() + 2.0 ** -25).all()
    assert ((S.double() - want[0][1]).norm(dim=2) <= want[0][3] + 1e-30).all()
    n = lengths(y, args[6])
    past = torch.arange(T, device=DEV)[None] >= n[:, None]
    assert (y[past] == 0).all()
    assert torch.equal(S[n == 0], args[5][n == 0])


@pytest.mark.parametrize("D", [64, 128])
def test_token_by_token_bits(D):
    q, k, v, a, b, S, _ = make(3, 21, 2, D, 5)
    all_at_once, S1 = S.clone(), S.clone()
    y = ops.gated_delta(q, k, v, a, b, all_at_once, chunked=False)
    for t in range(21):
        one = ops.gated_delta(*(x[:, t:t + 1].contiguous() for x in (q, k, v, a, b)), S1)
        assert torch.equal(one, y[:, t:t + 1])
    assert torch.equal(all_at_once, S1)
    few = S.clone()
    assert torch.equal(ops.gated_delta(q[:, :8].contiguous(), k[:, :8].contiguous(), v[:, :8].contiguous(),
                                       a[:, :8].contiguous(), b[:, :8].contiguous(), few), y[:, :8])


@pytest.mark.parametrize("T", [5, 100])
def test_slices_of_one_projection(T):
    q, k, v, a, b, S, lens = make(2, T, 3, 64, 1, ragged=True)
    wide = torch.full((2, T, 5, 3, 64), float("nan"), dtype=torch.float16, device=DEV)
    wide[:, :, 0], wide[:, :, 2], wide[:, :, 3] = q, k, v
    gates = torch.full((2, T, 2, 3), float("nan"), device=DEV)
    gates[:, :, 0], gates[:, :, 1] = a, b
    S1, S2 = S.clone(), S.clone()
    y = ops.gated_delta(q, k, v, a, b, S1, lens)
    args = (wide[:, :, 0], wide[:, :, 2], wide[:, :, 3], gates[:, :, 0], gates[:, :, 1])
    assert torch.equal(ops.gated_delta(*args, S2, lens), y) and torch.equal(S1, S2)
    dy = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    wide[:, :, 4] = dy
    one = ops.gated_delta_backward(q, k, v, a, b, S, dy, None, lens)
    two = ops.gated_delta_backward(*args, S, wide[:, :, 4], None, lens)
    assert all(torch.equal(x, y) for x, y in zip(one, two))


@pytest.mark.parametrize("D", [64, 128])
def test_decays_at_both_ends(D):
    q, k, v, a, b, S, _ = make(2, 150, 3, D, 9)
    a[:, :, 0] = 0.0
    a[:, :, 1] = -90.0
    a[0, 70, 2], a[0, 71, 2], a[1, 100, 2] = float("-inf"), -2e4, -800.0
    for chunked in (False, True):
        check(q, k, v, a, b, S, chunked=chunked)
    a[0, 3, 0] = 5.0                                   # counts as 0
    for chunked in (False, True):
        check(q, k, v, a, b, S, chunked=chunked)


@pytest.mark.parametrize("beta", [0.0, 0.5, 0.999, 1.0, 1.9])
def test_repeated_keys(beta):
    """One key for all tokens, no decay: a chunk's triangular system has entries beta
    everywhere, and its powers cancel."""
    q, k, v, a, b, S, _ = make(2, 200, 2, 64, 11)
    k[:] = k[:1, :1, :1]
    a.zero_()
    b.fill_(beta)
    # N_ij = (1 - beta)^(i - j - 1): a row of beta N sums to at most beta / (1 - |1 - beta|)
    # in absolute values, 1 up to beta 1 and 19 at 1.9, and so much larger are the
    # roundings of the X that it is applied to
    grow = max(1.0, beta / (1 - abs(1 - beta))) if beta else 1.0
    for chunked in (False, True):
        check(q, k, v, a, b, S, chunked=chunked, tight=grow)


def test_values_far_apart():
    """A value channel 2^14 times the others, keys of lengths 2^-7..2^3, states of 2^40."""
    q, k, v, a, b, S, _ = make(2, 130, 2, 64, 13)
    v[..., 3] *= 16384
    check(q, k, v, a, b, S)
    S *= 2.0 ** 40
    S[..., 5] = 0
    check(q, k, v, a, b, S)
    check(q, k / 128, v, a, b, S)
    check(q, 8 * k, v, a, b / 64, S)
    check(q, k, 0 * v, a, b, 0 * S, tight=0.0)


@pytest.mark.parametrize("T", [6, 100])
def test_an_infinite_value_channel_changes_no_other(T):
    q, k, v, a, b, S, _ = make(1, T, 2, 64, 17)
    S1 = S.clone()
    y = ops.gated_delta(q, k, v, a, b, S1)
    v[0, T // 2, 0, 7] = float("inf")
    S2 = S.clone()
    S2[0, 1, 4, 9] = float("nan")
    z = ops.gated_delta(q, k, v, a, b, S2)
    keep = torch.ones(2, 64, dtype=torch.bool, device=DEV)
    keep[0, 7] = keep[1, 9] = False
    assert torch.equal(z[:, :, keep], y[:, :, keep])
    assert torch.equal(S2.transpose(2, 3)[:, keep], S1.transpose(2, 3)[:, keep])
    assert not torch.isfinite(S2[0, 0, :, 7]).any() and torch.isnan(S2[0, 1, :, 9]).all()


@pytest.mark.parametrize("T", [1, 9])
def test_states_past_32_bits(T):
    """Heads whose states lie past 2^31 elements."""
    H = 131072 // 8 + 2
    q, k, v, a, b, S, _ = make(1, T, 2, 128, 3)
    many = [torch.zeros(8, T, H, 128, dtype=torch.float16, device=DEV) for _ in range(3)]
    gates = [torch.zeros(8, T, H, device=DEV) for _ in range(2)]
    for big, small in zip(many + gates, (q, k, v, a, b)):
        big[7, :, -2:] = small[0]
    states = torch.zeros(8, H, 128, 128, device=DEV)
    states[7, -2:] = S[0]
    y = ops.gated_delta(*many, *gates, states)
    want = ops.gated_delta(q, k, v, a, b, S)
    assert torch.equal(y[7, :, -2:], want[0]) and torch.equal(states[7, -2:], S[0])
    assert (y[:7] == 0).all()


# ------------------------------------------------------------------ gradients
def plain_grads(q, k, v, a, b, S, dy, dS, lens=None):
    q, k, v, a, b, S, dy = (t.double() for t in (q, k, v, a, b, S, dy))
    G = torch.zeros_like(S) if dS is None else dS.double()
    B, T, H, D = q.shape
    n = lengths(q, lens)
    keep = []
    for t in range(T):
        live = (t < n)[:, None, None, None]
        old = torch.exp(a[:, t].clamp_max(0))[..., None, None] * S
        d = v[:, t] - (old * k[:, t, :, :, None]).sum(2)
        u = b[:, t, :, None] * d
        S = torch.where(live, old + k[:, t, :, :, None] * u[:, :, None, :], S)
        keep.append((old, d, u, S))
    out = [torch.zeros_like(x) for x in (q, k, v, a, b)]
    for t in range(T - 1, -1, -1):
        live = (t < n)[:, None, None, None]
        old, d, u, S = keep[t]
        E = G + q[:, t, :, :, None] * dy[:, t, :, None, :]
        du = (E * k[:, t, :, :, None]).sum(2)
        dd = b[:, t, :, None] * du
        F = E - k[:, t, :, :, None] * dd[:, :, None, :]
        on = ((a[:, t] <= 0) & (a[:, t] >= -10000)).double()
        one = ((S * dy[:, t, :, None, :]).sum(3), (E * u[:, :, None, :]).sum(3) - (old * dd[:, :, None, :]).sum(3), dd,
               on * (F * old).sum((2, 3)), (d * du).sum(2))
        for o, x in zip(out, one):
            o[:, t] = torch.where(live.reshape((B,) + (1,) * (x.dim() - 1)), x, 0.0)
        G = torch.where(live, torch.exp(a[:, t].clamp_max(0))[..., None, None] * F, G)
    return (*out, G)


NAMES = ("dq", "dk", "dv", "dlog_decay", "dbeta", "dstate")


def check_grads(got, want, eps=2.0 ** -18):
    """fp32 gradients are sums of some D^2 terms of parts of 2^-22, which pass a few
    products: 16 of them in 2-norm over a tensor; fp16 ones those and half a step."""
    for name, x, y in zip(NAMES, got, want):
        assert torch.isfinite(x).all(), name
        off = x.double() - y
        if x.dtype == torch.float16:
            rows = y.norm(dim=3, keepdim=True).amax((1, 2), keepdim=True)
            tol = 2.0 ** -11 * y.abs() + 2.0 ** -25 + eps * rows
            assert (off.abs() <= tol).all(), (name, (off.abs() / tol).max())
        else:
            assert off.norm() <= eps * y.norm() + 1e-30, (name, off.norm() / y.norm())
            assert off.abs().max() <= 4 * eps * y.abs().max() + 1e-30, (name, off.abs().max() / y.abs().max())


def random_grads(args, seed):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(args[0].shape, generator=g).half().to(DEV),
            torch.randn(args[5].shape, generator=g).to(DEV))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T", [1, 3, 32, 63, 64, 65, 129, 200])
def test_gradients(T, D):
    args = make(2, T, 3, D, 7 * T + D)
    dy, dS = random_grads(args, T)
    for g in (dS, None):
        check_grads(ops.gated_delta_backward(*args[:6], dy, g), plain_grads(*args[:6], dy, g))


@pytest.mark.parametrize("B,T,H,D", [(1, 900, 2, 64), (40, 150, 2, 64), (5, 300, 2, 128), (300, 20, 1, 64)])
def test_ragged_gradients(B, T, H, D):
    args = make(B, T, H, D, B + T, ragged=True)
    if B > 1:
        args[6][0], args[6][-1] = T, 0
    dy, dS = random_grads(args, B)
    want = plain_grads(*args[:6], dy, dS, args[6])
    for t in (*args[:5], dy):                         # rows past a stream's end hold anything
        for i in range(B):
            t[i, int(args[6][i]):] = float("nan")
    got = ops.gated_delta_backward(*args[:6], dy, dS, args[6])
    check_grads(got, want)
    past = torch.arange(T, device=DEV)[None] >= lengths(args[0], args[6])[:, None]
    assert all((g[past] == 0).all() for g in got[:5])


def test_gradients_at_the_ends_of_gates():
    args = make(2, 150, 3, 64, 19)
    a, b = args[3], args[4]
    a[:, :, 0] = 0.0
    a[:, :, 1] = -90.0
    a[0, 70, 2], a[0, 71, 2], a[1, 100, 2], a[1, 3, 2] = -float("inf"), -2e4, -800.0, 5.0
    b[:, ::3, 0], b[:, 1::7, 2] = 0.0, 1.0
    b[0, :, 1] = 0.0
    dy, dS = random_grads(args, 3)
    want = plain_grads(*args[:6], dy, dS)
    got = ops.gated_delta_backward(*args[:6], dy, dS)
    # beside decays of 0 a head's sums of thousands of tokens' terms cancel to what a
    # decay of e^-90 leaves: its gradient is compared with the others' size
    check_grads(got, want)
    assert got[3][0, 70, 2] == 0 and got[3][0, 71, 2] == 0 and got[3][1, 3, 2] == 0


def test_gradients_against_differences():
    """Along random directions, with central differences of the float64 recurrence."""
    args = make(2, 70, 2, 64, 23)
    dy, dS = random_grads(args, 5)
    got = ops.gated_delta_backward(*args[:6], dy, dS)
    x = [t.double() for t in args[:6]]
    g = torch.Generator().manual_seed(4)

    def value(parts):
        y, S, _, _ = plain(*parts)
        return (y * dy.double()).sum() + (S * dS.double()).sum()

    for i in range(6):
        d = torch.randn(x[i].shape, generator=g).double().to(DEV)
        d *= 0.05 * x[i].norm() / d.norm()
        if i == 3:
            d = -d.abs().clamp_max(0.5 * x[i].abs().min())     # stays below 0
        plus, minus, wide = ([t + c * d if j == i else t for j, t in enumerate(x)] for c in (1e-3, -1e-3, 2e-3))
        low = [t - 2e-3 * d if j == i else t for j, t in enumerate(x)]
        diff = (value(plus) - value(minus)) / 2e-3
        # of order h^2: a third of the difference to twice the step
        cut = (diff - (value(wide) - value(low)) / 4e-3).abs() / 3 + 1e-9 * diff.abs() + 1e-8
        slack = (2.0 ** -11 if i < 3 else 0) * (got[i].double() * d).abs().sum() + 2.0 ** -18 * got[i].double().norm() * d.norm()
        assert ((got[i].double() * d).sum() - diff).abs() <= 2 * cut + slack, NAMES[i]


def test_bits_graph_and_streams():
    args = make(3, 200, 2, 64, 29, ragged=True)
    dy, dS = random_grads(args, 7)

    def both():
        S = args[5].clone()
        return (ops.gated_delta(*args[:5], S, args[6]), S, *ops.gated_delta_backward(*args[:6], dy, dS, args[6]))

    want = both()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    got = []
    for s in (a, b, a, b):
        with torch.cuda.stream(s):
            got.append(both())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for one in got for x, y in zip(one, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = both()
    v = args[2].clone()
    for i in range(4):
        args[2].copy_(v if i % 2 == 0 else -v)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(out, both()))


def test_empty_calls():
    q, k, v, a, b, S, _ = make(2, 4, 2, 64, 1)
    before = S.clone()
    none = [t[:, :0] for t in (q, k, v, a, b)]
    assert ops.gated_delta(*none, S).shape == (2, 0, 2, 64) and torch.equal(S, before)
    got = ops.gated_delta_backward(*none, S, q[:, :0], before)
    assert got[0].shape == (2, 0, 2, 64) and torch.equal(got[5], before)
    assert (ops.gated_delta_backward(*none, S, q[:, :0])[5] == 0).all()
    assert ops.gated_delta(*(t[:0] for t in (q, k, v, a, b, S))).shape == (0, 4, 2, 64)
    lens = torch.zeros(2, dtype=torch.int32, device=DEV)
    got = ops.gated_delta_backward(q, k, v, a, b, S, q, before, lens)
    assert all((g == 0).all() for g in got[:5]) and torch.equal(got[5], before)
    assert _lib.lib().kr_gated_delta_backward_workspace_bytes(0, 4, 2, 64) == 0
