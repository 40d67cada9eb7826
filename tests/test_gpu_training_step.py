"""The gated delta rule and the head's cross entropy together, as a training step runs
them: a one-layer model's loss and the gradients of all its weights against autograd in
float64, and a prompt followed by single tokens against the whole text at once."""
import pytest
import torch

from krunch_amd import krunch_ac_hip as ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def model(V, H, D, seed):
    g = torch.Generator().manual_seed(seed)
    C = H * D
    emb = torch.randn(V, C, generator=g)
    proj = torch.randn(C, 3 * C, generator=g) / C ** 0.5
    gates = torch.randn(C, 2 * H, generator=g) / C ** 0.5
    head = 2 * torch.randn(V, C, generator=g) / C ** 0.5
    return [w.to(DEV) for w in (emb.half(), proj.half(), gates.half(), head.half())]


def in_64_bits(weights, ids, targets, H, D):
    emb, proj, gates, head = (w.double().requires_grad_() for w in weights)
    B, T = ids.shape
    x = emb[ids.long()]
    q, k, v = (x @ proj).view(B, T, 3, H, D).unbind(2)
    a, b = (x @ gates).view(B, T, 2, H).unbind(2)
    a, b = -torch.nn.functional.softplus(a), torch.sigmoid(b)
    k = k / k.norm(dim=3, keepdim=True)
    S, ys = torch.zeros(B, H, D, D, dtype=torch.float64, device=DEV), []
    for t in range(T):
        S = torch.exp(a[:, t])[..., None, None] * S
        u = b[:, t, :, None] * (v[:, t] - (S * k[:, t, :, :, None]).sum(2))
        S = S + k[:, t, :, :, None] * u[:, :, None, :]
        ys.append((S * q[:, t, :, :, None]).sum(2) / D ** 0.5)
    z = x + torch.stack(ys, 1).reshape(B, T, H * D)
    logp = torch.log_softmax(z @ head.t(), 2)
    loss = -logp.gather(2, targets.long().clamp_min(0)[..., None])[..., 0] * (targets >= 0)
    loss.sum().backward()
    return loss.detach(), [w.grad for w in (emb, proj, gates, head)]


@pytest.mark.parametrize("B,T,H,D,V", [(3, 100, 2, 64, 300), (2, 70, 1, 128, 1000)])
def test_training_step(B, T, H, D, V):
    weights = model(V, H, D, B + T)
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (B, T), generator=g).to(DEV)
    targets = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32)
    targets[0, 5] = targets[1, -3:] = -1
    targets = targets.to(DEV)
    want, grads = in_64_bits(weights, ids, targets, H, D)

    # the step: fp32 between the operators, fp16 where they take it
    emb, proj, gates, head = (w.float().requires_grad_() for w in weights)
    x = emb[ids]
    q, k, v = (x @ proj).view(B, T, 3, H, D).unbind(2)
    ab = (x @ gates).view(B, T, 2, H)
    a, b = -torch.nn.functional.softplus(ab[:, :, 0]), torch.sigmoid(ab[:, :, 1])
    k, q = k / k.norm(dim=3, keepdim=True), q / D ** 0.5
    ins = [t.detach().half() for t in (q, k, v)] + [a.detach().contiguous(), b.detach().contiguous()]
    S = torch.zeros(B, H, D, D, device=DEV)
    y = ops.gated_delta(*ins, S.clone())
    z = (x.detach() + y.reshape(B, T, H * D).float()).half().reshape(B * T, H * D)
    loss, lse = ops.head_loss(z, head.detach().half(), targets.reshape(-1))
    dz, dhead = ops.head_loss_backward(z, head.detach().half(), targets.reshape(-1), lse,
                                       torch.ones_like(loss), torch.float32)
    dy = dz.half().reshape(y.shape)
    dq, dk, dv, da, db, _ = ops.gated_delta_backward(*ins, S, dy)
    torch.autograd.backward([q, k, v, a, b, x], [dq.float(), dk.float(), dv.float(), da, db,
                                                 dz.reshape(B, T, H * D)])
    # inputs rounded to fp16 at 4 places of a row: some 2^-11 of each value, so 2^-8 in
    # 2-norm after the products behind them
    assert ((loss.double() - want.reshape(-1)).norm() / want.norm()) < 2.0 ** -8
    for got, ref in zip((emb.grad, proj.grad, gates.grad, dhead), grads):
        assert (got.double() - ref).norm() < 2.0 ** -8 * ref.norm()


def test_prompt_then_tokens():
    """A prompt in chunks, then token by token: the state is carried, and the losses are
    those of the text in one call, up to the forms' rounding (2^-20 of the state, which
    fp16 y and its row hide but for a rounding's flip, 2^-11)."""
    B, T, H, D, V = 2, 90, 2, 64, 500
    g = torch.Generator().manual_seed(2)
    q, k, v = (torch.randn(B, T, H, D, generator=g) for _ in range(3))
    k = k / k.norm(dim=3, keepdim=True)
    ins = [t.half().to(DEV) for t in (q / 8, k, v)] + [
        (-0.1 * torch.rand(B, T, H, generator=g)).to(DEV), torch.rand(B, T, H, generator=g).to(DEV)]
    head = (torch.randn(V, H * D, generator=g) / 8).half().to(DEV)
    targets = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32).to(DEV)
    S, P = torch.zeros(B, H, D, D, device=DEV), torch.zeros(B, H, D, D, device=DEV)
    y = ops.gated_delta(*ins, S)
    whole = ops.head_loss(y.reshape(B * T, H * D), head, targets.reshape(-1))[0].view(B, T)
    parts = [ops.gated_delta(*(t[:, :80].contiguous() for t in ins), P)]
    parts += [ops.gated_delta(*(t[:, i:i + 1].contiguous() for t in ins), P) for i in range(80, T)]
    joined = torch.cat(parts, 1)
    assert (S - P).norm() <= 2.0 ** -18 * S.norm()
    assert (y.float() - joined.float()).norm() <= 2.0 ** -12 * y.float().norm()
    for i in range(80, T):
        one = ops.head_loss(parts[i - 79].reshape(B, H * D), head, targets[:, i].contiguous())[0]
        size = parts[i - 79].float().abs().reshape(B, -1) @ head.float().abs().t()
        assert ((one - whole[:, i]).abs() <= 2.0 ** -9 * size.amax(1)).all()
