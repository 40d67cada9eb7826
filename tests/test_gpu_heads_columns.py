"""WKV with heads, chunked: a value channel's results do not depend on what the
other channels' columns of the state hold, be it infinite or far larger."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def make(B, T, H, D, seed):
    g = torch.Generator().manual_seed(seed)
    r, k, v = ((a * torch.randn(B, T, H, D, generator=g)).half().to(DEV) for a in (0.5, 0.5, 1.0))
    w = -torch.exp(torch.linspace(-6.0, -2.0, H)).to(DEV)
    u = (0.2 + torch.rand(H, generator=g)).to(DEV)
    return r, k, v, w, u, torch.randn(B, H, D, D, generator=g).to(DEV)


def walk(r, k, v, w, u, S):
    """In float64 on the CPU: y, state, the sums over absolute values of y and the
    state, and per token and column sum |r| times the column's largest state."""
    r, k, v, S = (t.double().cpu() for t in (r, k, v, S))
    g, u = torch.exp(w.double().cpu())[None, :, None, None], u.double().cpu()[None, :, None, None]
    A = S.abs()
    y, size, top = (torch.zeros_like(r) for _ in range(3))
    for t in range(r.shape[1]):
        kv = k[:, t, :, :, None] * v[:, t, :, None, :]
        at = r[:, t, :, :, None]
        y[:, t] = (at * (S + u * kv)).sum(2)
        size[:, t] = (at.abs() * (A + (u * kv).abs())).sum(2)
        top[:, t] = at.abs().sum(2) * A.amax(2)
        S, A = g * S + kv, g * A + kv.abs()
    return y, S, size, A, top


def check(y, S, ref, inside, live):
    """On the channels `live`. fp32 sums and the decays: (4 T + 2 D + 8) 2^-24 of the
    absolute sums. Two fp16 parts: 2^-22 of a value (products of up to three such
    factors: 2^-20) and 2^-38 of the largest one of its scale: a column of the
    state (sum |r| times it), a row of r k' and a column of v (of which a chunk
    has 64: 2^-32, under the 2^-20 for channels whose v are alike, as here, with
    2^-34 of the largest beside). y is rounded to fp16."""
    ref_y, ref_S, size, size_S, top = ref
    T, D = y.shape[1], y.shape[3]
    eps = (4 * T + 2 * D + 8) * 2.0 ** -24 + 2.0 ** -20
    tol = (eps * size + 2.0 ** -11 * ref_y.abs() + 2.0 ** -25 + 2.0 ** -25 * top +
           2.0 ** -34 * inside[2].amax(3, keepdim=True))
    err = (y.double().cpu() - ref_y).abs()
    assert (err <= tol)[..., live].all(), (err / tol)[..., live].max()
    tol = eps * size_S + 2.0 ** -34 * size_S.amax(2, keepdim=True)
    err = (S.double().cpu() - ref_S).abs()
    assert (err <= tol)[..., live].all(), (err / tol)[..., live].max()


# one chunk, several, a split time axis; both widths
SHAPES = [(1, 64, 2, 64), (40, 70, 8, 64), (1, 300, 2, 64), (1, 200, 2, 128), (130, 70, 2, 128)]


@pytest.mark.parametrize("B,T,H,D", SHAPES)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")])
def test_an_infinite_element_stays_in_its_column(B, T, H, D, bad):
    r, k, v, w, u, S = make(B, T, H, D, B + T)
    col = D - 11
    clean = S.clone()
    clean[:, :, :, col] = 0.0
    ref, inside = walk(r, k, v, w, u, clean), walk(r, k, v, w, u, torch.zeros_like(S))
    S[0, 0, 5, col] = bad
    y = ops.wkv_heads(r, k, v, w, u, S)
    live = [c for c in range(D) if c != col]
    check(y, S, ref, inside, live)
    assert torch.isfinite(y[..., live]).all() and torch.isfinite(S[..., live]).all()
    assert not torch.isfinite(y[0, :, 0, col]).any()
    assert torch.equal(~torch.isfinite(S[0, 0, :, col]).cpu(), torch.arange(D) == 5)


def test_after_an_infinite_value_token_by_token():
    """What the recurrent form leaves of an infinite v: inf in that channel's column."""
    r, k, v, w, u, S = make(2, 100, 3, 64, 3)
    v[0, 2, 1, 20] = float("inf")
    S1 = S.clone()
    for f in (S, S1):
        ops.wkv_heads(*(x[:, :5].contiguous() for x in (r, k, v)), w, u, f, chunked=False)
    assert torch.equal(S, S1) and not torch.isfinite(S[0, 1, :, 20]).any()
    clean = torch.where(torch.isfinite(S), S, torch.zeros_like(S))
    rest = [x[:, 5:].contiguous() for x in (r, k, v)]
    ref, inside = walk(*rest, w, u, clean), walk(*rest, w, u, torch.zeros_like(S))
    live = [c for c in range(64) if c != 20]
    y = ops.wkv_heads(*rest, w, u, S)
    check(y, S, ref, inside, live)
    assert torch.isfinite(y[..., live]).all() and torch.isfinite(y[1]).all()
    assert not torch.isfinite(y[0, :, 1, 20]).any()
    one = ops.wkv_heads(*rest, w, u, S1, chunked=False)
    assert torch.equal(torch.isfinite(one), torch.isfinite(y))


@pytest.mark.parametrize("B,T,H,D", SHAPES)
@pytest.mark.parametrize("power", [20, 40, 100, -60])
def test_columns_of_very_different_sizes(B, T, H, D, power):
    """A column 2^power times the others, in y as precise as its neighbours."""
    r, k, v, w, u, S = make(B, T, H, D, B + T + 1)
    S[..., 3] *= 2.0 ** power
    ref, inside = walk(r, k, v, w, u, S), walk(r, k, v, w, u, torch.zeros_like(S))
    y = ops.wkv_heads(r, k, v, w, u, S)
    live = [c for c in range(D) if c != 3 or power < 0]
    check(y, S, ref, inside, live)
    if power >= 40:       # the large column itself: past fp16's range, or nearly
        big = ref[0][..., 3].abs() > 66000
        assert torch.isinf(y[..., 3].cpu()[big]).all()
