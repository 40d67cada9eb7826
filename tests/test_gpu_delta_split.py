"""The gated delta rule and its gradients where the time axis is split over workgroups:
streams that end in the first, a middle and the last segment, at a segment's edge, or
have no token, against the recurrence in float64. The tolerances are test_gpu_delta's: a
join adds a segment's map in two parts, 2^-22 of what it is applied to, where the bounds
count 2^-20 a token."""
import pytest
import torch

from krunch_amd import _lib, krunch_ac_hip as ops
from tests.test_gpu_delta import check, check_grads, lengths, make, plain_grads, random_grads

pytestmark = pytest.mark.gpu
DEV = "cuda"


def segment_tokens(B, T, H, D, back=False):
    """Tokens of a segment, from what a call's workspace holds: three or five states a
    segment, and the backward pass's of every chunk."""
    state, chunks = 4 * B * H * D * D, -(-T // 64)
    if back:
        need = _lib.lib().kr_gated_delta_backward_workspace_bytes(B, T, H, D)
        need -= (2 * chunks + 1) * state + 2 * chunks * 4 * B * H * 64 * D
        segments = need // (5 * state)
    else:
        segments = _lib.lib().kr_gated_delta_workspace_bytes(B, T, H, D) // (3 * state)
    assert segments >= 4, "the rule splits these calls"
    return 64 * -(-chunks // segments)


def ends(T, seg):
    """Lengths: whole, none, one token, at and around a segment's edge, in the middle of
    one, in the last."""
    last = (T - 1) // seg * seg
    return torch.tensor([T, 0, 1, seg - 1, seg, seg + 1, 2 * seg + 37, last, last + 5, T - 1], dtype=torch.int32)


@pytest.mark.parametrize("D,T", [(64, 1999), (64, 1280), (128, 1400)])
def test_streams_that_end_in_any_segment(D, T):
    B, H = 10, 1
    args = make(B, T, H, D, T + D)
    args[6] = ends(T, segment_tokens(B, T, H, D)).to(DEV)
    y, S = check(*args)
    past = torch.arange(T, device=DEV)[None] >= lengths(y, args[6])[:, None]
    assert (y[past] == 0).all()
    assert torch.equal(S[1], args[5][1])
    # the same bits in every call
    for _ in range(10):
        again = args[5].clone()
        assert torch.equal(ops.gated_delta(*args[:5], again, args[6]), y) and torch.equal(again, S)


@pytest.mark.parametrize("D", [64, 128])
def test_streams_without_an_end(D):
    """No lens, and decays that leave what the first segments wrote in the last."""
    B, T, H = 2, 1500, 2
    segment_tokens(B, T, H, D)
    check(*make(B, T, H, D, D, rate=(-9.0, -7.0)))


@pytest.mark.parametrize("D,T", [(64, 1999), (128, 1400)])
def test_gradients_of_streams_that_end_in_any_segment(D, T):
    B, H = 10, 1
    args = make(B, T, H, D, T - D)
    args[6] = ends(T, segment_tokens(B, T, H, D, True)).to(DEV)
    dy, dS = random_grads(args, D)
    want = plain_grads(*args[:6], dy, dS, args[6])
    got = ops.gated_delta_backward(*args[:6], dy, dS, args[6])
    check_grads(got, want)
    past = torch.arange(T, device=DEV)[None] >= lengths(args[0], args[6])[:, None]
    assert all((g[past] == 0).all() for g in got[:5])
    assert torch.equal(got[5][1], dS[1])
    for _ in range(10):
        again = ops.gated_delta_backward(*args[:6], dy, dS, args[6])
        assert all(torch.equal(x, y) for x, y in zip(again, got))


@pytest.mark.parametrize("D", [64, 128])
def test_gradients_through_all_segments(D):
    """Decays that carry the last state's gradient to the first tokens, and no gradient of it."""
    B, T, H = 2, 1500, 2
    segment_tokens(B, T, H, D, True)
    args = make(B, T, H, D, 3 * D, rate=(-9.0, -7.0))
    dy, dS = random_grads(args, 1)
    for g in (dS, None):
        check_grads(ops.gated_delta_backward(*args[:6], dy, g), plain_grads(*args[:6], dy, g))
