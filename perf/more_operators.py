"""What the speed of the training-side operators is measured on: the cross
entropy of a head over a large vocabulary, in pieces of it and without its
logits, with its gradients; and the gated delta rule, chunked and token by token,
with its gradients; each through its public entry point.

They are what adapts a model to the texts that it is to compress. A text's cost
in bits is the cross entropy of its next tokens, whose gradient moves the head
and, through the last rows, the layers. The delta rule is a recurrence with a
matrix state per head, as the WKV with heads is one, which replaces what a key
had stored instead of adding to it.

Sizes are the 169M configuration's (width 768, vocabulary 50277, heads of 64),
its neighbours' (width 256..1024, heads of 128) and the byte tokenizer's (256).
"""
from __future__ import annotations

import math

import torch

own = False          # True: run() calls the framework; False: the plain form

DEV = "cuda"
CHUNK = 64           # tokens that the plain form of the delta rule takes at a time


def listed():
    return [
        # What one next token costs: latency against the whole head.
        {"name": "loss_1x768x50277", "kind": "loss", "N": 1, "C": 768, "V": 50277},
        # A byte-level model's losses over a long text, an odd row count.
        {"name": "loss_30001x512x256", "kind": "loss", "N": 30001, "C": 512, "V": 256},
        # Eight windows of 1024 tokens.
        {"name": "loss_8192x768x50277", "kind": "loss", "N": 8192, "C": 768, "V": 50277},
        # Gradients of one short text through a wider head.
        {"name": "grad_97x1024x50277", "kind": "grad", "N": 97, "C": 1024, "V": 50277},
        # Gradients of a byte-level head.
        {"name": "grad_20000x256x256", "kind": "grad", "N": 20000, "C": 256, "V": 256},
        # Gradients of eight windows of 1024 tokens (the largest).
        {"name": "grad_8192x768x50277", "kind": "grad", "N": 8192, "C": 768, "V": 50277},
        # One stream's next token.
        {"name": "delta_step_1", "kind": "delta", "B": 1, "T": 1, "H": 12, "D": 64, "ragged": False},
        # The engine's default batch, one token each.
        {"name": "delta_step_512", "kind": "delta", "B": 512, "T": 1, "H": 12, "D": 64, "ragged": False},
        # One prompt of odd length, wide heads.
        {"name": "delta_1x1777_wide", "kind": "delta", "B": 1, "T": 1777, "H": 8, "D": 128, "ragged": False},
        # A scoring window of prompts of different lengths.
        {"name": "delta_128x1024_ragged", "kind": "delta", "B": 128, "T": 1024, "H": 12, "D": 64, "ragged": True},
        # Gradients of one long text.
        {"name": "delta_grad_1x2000", "kind": "delta_grad", "B": 1, "T": 2000, "H": 12, "D": 64, "ragged": False},
        # Gradients of a training batch of texts of different lengths.
        {"name": "delta_grad_48x1024_ragged", "kind": "delta_grad", "B": 48, "T": 1024, "H": 12, "D": 64,
         "ragged": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["loss", "grad", "delta", "delta_grad"])
    if kind in ("loss", "grad"):
        V = rng.choice([50277, 256, _log(rng, 100, 150000)])
        C = rng.choice([256, 512, 768, 1024, 64 * rng.randint(1, 20)])
        most = 8192 * 50277 * 768 // (V * C)
        return {"kind": kind, "N": _log(rng, 1, max(2, min(60000, most // 2))), "C": C, "V": V}
    D = rng.choice([64, 64, 128])
    H = rng.choice([4, 8, 12, 16]) * 64 // D
    if kind == "delta" and rng.random() < 0.35:
        T, B = 1, _log(rng, 1, 512)
    else:
        T = _log(rng, 2, 4096)
        B = _log(rng, 1, max(1, min(256, (70000 if kind == "delta" else 30000) * 12 * 64 // (T * H * D))))
    return {"kind": kind, "B": B, "T": T, "H": H, "D": D, "ragged": T > 1 and rng.random() < 0.4}


# ------------------------------------------------------------------ inputs
def _gen(seed, what):
    return torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + what)


def _head_inputs(case, seed):
    """Normalised rows before a head, the head [V, C], and the tokens that follow,
    one row in 64 without. A head whose first column answers a constant in every
    row with the tokens' frequencies: a row's entropy is some nats. For the
    gradients: each row's weight, and the logsumexp that the forward pass left."""
    g = _gen(seed, 1)
    N, C, V = case["N"], case["C"], case["V"]
    x = torch.randn((N, C), generator=g, device=DEV)
    W = torch.randn((V, C), generator=g, device=DEV).mul_(2 / math.sqrt(C))
    x[:, 0] = 1
    rank = torch.randperm(V, generator=g, device=DEV)
    W[:, 0] = -1.1 * torch.log1p(rank.float())
    x, W = x.half(), W.half()
    targets = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    if N > 1:
        targets[torch.rand(N, generator=g, device=DEV) < 1 / 64] = -1
    state = {"x": x, "W": W, "targets": targets}
    if case["kind"] == "grad":
        state["dloss"] = 0.5 + torch.rand(N, generator=g, device=DEV)
        lse = torch.empty(N, device=DEV)
        for i in range(0, N, 2048):
            lse[i:i + 2048] = torch.logsumexp(x[i:i + 2048].float() @ W.float().t(), 1)
        state["lse"] = lse
    return state


def _delta_inputs(case, seed):
    """Queries, keys of length 1 and values of B streams, decays from near 1 to a
    token or two that vary from token to token, write strengths in 0..1, the
    state that earlier tokens left, and the lengths of ragged streams. For the
    gradients: those of y and of the last state."""
    g = _gen(seed, 2)
    B, T, H, D = case["B"], case["T"], case["H"], case["D"]
    q, k, v = (torch.randn((B, T, H, D), generator=g, device=DEV) for _ in range(3))
    k = k / k.square().sum(3, keepdim=True).sqrt()
    rate = torch.exp(torch.linspace(-6.0, 0.7, H, device=DEV))
    log_decay = -rate * (0.5 + torch.rand((B, T, H), generator=g, device=DEV))
    beta = torch.sigmoid(torch.randn((B, T, H), generator=g, device=DEV))
    s = {"q": (q / math.sqrt(D)).half(), "k": k.half(), "v": v.half(), "log_decay": log_decay, "beta": beta,
         "state": 0.5 * torch.randn((B, H, D, D), generator=g, device=DEV), "lens": None}
    if case["ragged"]:
        s["lens"] = torch.randint(max(1, T // 4), T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    if case["kind"] == "delta_grad":
        s["dy"] = torch.randn((B, T, H, D), generator=g, device=DEV).half()
        s["dstate"] = torch.randn((B, H, D, D), generator=g, device=DEV)
    return s


def prepare(case, seed):
    state = (_head_inputs if case["kind"] in ("loss", "grad") else _delta_inputs)(case, seed)
    state["kind"] = case["kind"]
    return state


# -------------------------------------------------------------- plain forms
def _loss_plain(s):
    z = s["x"].float() @ s["W"].float().t()
    m = z.amax(1, keepdim=True)
    lse = m[:, 0] + torch.log(torch.exp(z - m).sum(1))
    t = s["targets"].long()
    loss = lse - z.gather(1, t.clamp_min(0)[:, None])[:, 0]
    return {"loss": torch.where(t < 0, torch.zeros_like(loss), loss), "lse": lse}


def _grad_plain(s):
    """dz = dloss (softmax - the target's 1), rows without a target 0."""
    x, W, t = s["x"].float(), s["W"].float(), s["targets"].long()
    weight = torch.where(t < 0, torch.zeros_like(s["dloss"]), s["dloss"])
    dz = torch.exp(x @ W.t() - s["lse"][:, None])
    dz[torch.arange(len(t), device=DEV), t.clamp_min(0)] -= 1
    dz.mul_(weight[:, None])
    return {"dx": (dz @ W).half(), "dW": (dz.t() @ x).half()}


def _delta_step_plain(s):
    """One token: S <- e^g S; S <- S + beta k'(v - k S); y = q S."""
    q, k, v = (s[n][:, 0].float() for n in ("q", "k", "v"))
    S = s["state"]
    old = S * torch.exp(s["log_decay"][:, 0])[..., None, None]
    u = s["beta"][:, 0, :, None] * (v - (k[..., None] * old).sum(2))
    S.copy_(old + k[..., None] * u[..., None, :])
    return {"y": (q[..., None] * S).sum(2).half()[:, None], "state": S}


class _Chunks:
    """A call's tokens by chunks, [B, H, chunks, 64, ...] in fp32, and what of a
    chunk does not depend on the state. With a_i the sum of the log decays to i:
      A_ij = e^(a_i - a_j) k_i k_j' (j < i), P_ij = e^(a_i - a_j) q_i k_j' (j <= i),
      N = A (1 + beta A)^-1, by rows: N_i = A_i - sum_j A_ij beta_j N_j.
    Then r = X - N (beta X) with X = v - e^a k S are the differences that the
    tokens write, u = beta r, and y = e^a q S + P u."""

    def __init__(self, s):
        B, T, H, D = s["q"].shape
        self.T, self.shape = T, (B, H, D)
        self.n = s["lens"].long() if s["lens"] is not None else torch.full((B,), T, device=DEV)
        live = torch.arange(T, device=DEV)[None, :] < self.n[:, None]
        self.live = live
        self.q, self.k, self.v = (self.split(s[m]) for m in ("q", "k", "v"))
        self.b, a = self.split(s["beta"]), self.split(s["log_decay"]).double().cumsum(3)
        i = torch.arange(CHUNK, device=DEV)
        self.low = (i[:, None] >= i[None, :])
        far = torch.where(self.low, a[..., :, None] - a[..., None, :], -math.inf)
        self.decay = torch.exp(far).float()                       # [i, j], 0 above the diagonal
        self.e0 = torch.exp(a).float()[..., None]                 # from the chunk's start
        self.e1 = torch.exp(a[..., -1:] - a).float()[..., None]   # to its end
        self.all = torch.exp(a[..., -1]).float()[..., None, None]
        kt = self.k.transpose(3, 4).contiguous()
        self.P = (self.q @ kt) * self.decay
        self.A = (self.k @ kt) * torch.where(i[:, None] > i[None, :], self.decay, torch.zeros_like(self.decay))
        N = self.A.clone()
        Ab = self.A * self.b[..., None, :]
        for t in range(1, CHUNK):
            N[..., t, :] -= (Ab[..., t, None, :t] @ N[..., :t, :])[..., 0, :]
        self.N = N

    def split(self, t):
        """[B, T, H, ...] -> [B, H, chunks, 64, ...], tokens past a stream's 0."""
        t = torch.where(self.live.reshape(self.live.shape + (1,) * (t.dim() - 2)), t.float(), 0.0)
        pad = -(-self.T // CHUNK) * CHUNK - self.T
        t = torch.cat((t, t.new_zeros((t.shape[0], pad) + t.shape[2:])), 1)
        t = t.reshape((t.shape[0], -1, CHUNK) + t.shape[2:])
        return t.permute((0, 3, 1, 2) + tuple(range(4, t.dim()))).contiguous()

    def join(self, t):
        """Back to [B, T, H, ...], tokens past a stream's 0."""
        t = t.permute((0, 2, 3, 1) + tuple(range(4, t.dim())))
        t = t.reshape((t.shape[0], -1) + t.shape[3:])[:, :self.T]
        return torch.where(self.live.reshape(self.live.shape + (1,) * (t.dim() - 2)), t, 0.0).contiguous()

    def forward(self, S):
        """The state before each chunk, what its tokens write, and the last state."""
        kt = (self.k * self.e1).transpose(3, 4).contiguous()
        before, u = [], []
        for c in range(self.q.shape[2]):
            before.append(S)
            X = self.v[:, :, c] - self.e0[:, :, c] * (self.k[:, :, c] @ S)
            r = X - self.N[:, :, c] @ (self.b[:, :, c, :, None] * X)
            u.append(self.b[:, :, c, :, None] * r)
            S = self.all[:, :, c] * S + kt[:, :, c] @ u[-1]
        return torch.stack(before, 2), torch.stack(u, 2), S


def _delta_plain(s):
    if s["q"].shape[1] == 1 and s["lens"] is None:
        return _delta_step_plain(s)
    c = _Chunks(s)
    before, u, S = c.forward(s["state"])
    y = c.e0 * (c.q @ before) + c.P @ u
    s["state"].copy_(S)
    return {"y": c.join(y.half()), "state": s["state"]}


def _delta_grad_plain(s):
    """From the last chunk to the first, with D the gradient of the state behind a
    chunk: du = P'dy + e^(end - a) k D, w = du - N'(beta du), dX = beta w and
    the state's e^end D + (e^a q)'dy - (e^a k)'dX; the rest for all chunks at once."""
    c = _Chunks(s)
    before, u, _ = c.forward(s["state"])
    dy, b = c.split(s["dy"]), c.b[..., None]
    qt, kt = ((t * c.e0).transpose(3, 4).contiguous() for t in (c.q, c.k))
    Pt, Nt = c.P.transpose(3, 4).contiguous(), c.N.transpose(3, 4).contiguous()
    D = s["dstate"]
    behind, w = [], []
    for i in range(c.q.shape[2] - 1, -1, -1):
        behind.append(D)
        du = Pt[:, :, i] @ dy[:, :, i] + c.e1[:, :, i] * (c.k[:, :, i] @ D)
        w.append(du - Nt[:, :, i] @ (b[:, :, i] * du))
        D = c.all[:, :, i] * D + qt[:, :, i] @ dy[:, :, i] - kt[:, :, i] @ (b[:, :, i] * w[-1])
    behind, w = torch.stack(behind[::-1], 2), torch.stack(w[::-1], 2)
    X = c.v - c.e0 * (c.k @ before)
    r = X - c.N @ (b * X)
    dX, ut, St = b * w, u.transpose(3, 4).contiguous(), before.transpose(3, 4).contiguous()
    strict = c.decay - torch.diag_embed(torch.diagonal(c.decay, dim1=3, dim2=4))
    MP = (dy @ ut) * c.decay
    MA = -(dX @ ut) * strict
    dq = c.e0 * (dy @ St) + MP @ c.k
    dk_read = MA @ c.k - c.e0 * (dX @ St)
    dk_write = (MP.transpose(3, 4).contiguous() @ c.q + MA.transpose(3, 4).contiguous() @ c.k
                + c.e1 * (u @ behind.transpose(3, 4).contiguous()))
    # a_i is in e^(a_i) of q_i and of the key that reads, e^(-a_i) of the key that
    # writes; the end's in all of the state behind
    da = ((c.q * dq).double() + (c.k * dk_read).double() - (c.k * dk_write).double()).sum(4)
    after = c.all * before + (c.k * c.e1).transpose(3, 4).contiguous() @ u
    da[..., -1] += (behind.double() * after.double()).sum((3, 4))
    dg = da.flip(3).cumsum(3).flip(3).float()
    return {"dq": c.join(dq.half()), "dk": c.join((dk_read + dk_write).half()), "dv": c.join(dX.half()),
            "dlog_decay": c.join(dg), "dbeta": c.join((w * r).sum(4)), "dstate": D}


def run(state):
    s, kind = state, state["kind"]
    if own:
        from krunch_amd import krunch_ac_hip
        if kind == "loss":
            loss, lse = krunch_ac_hip.head_loss(s["x"], s["W"], s["targets"])
            return {"loss": loss, "lse": lse}
        if kind == "grad":
            dx, dW = krunch_ac_hip.head_loss_backward(s["x"], s["W"], s["targets"], s["lse"], s["dloss"])
            return {"dx": dx, "dW": dW}
        if kind == "delta":
            y = krunch_ac_hip.gated_delta(s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"],
                                          s["lens"])
            return {"y": y, "state": s["state"]}
        names = ("dq", "dk", "dv", "dlog_decay", "dbeta", "dstate")
        return dict(zip(names, krunch_ac_hip.gated_delta_backward(
            s["q"], s["k"], s["v"], s["log_decay"], s["beta"], s["state"], s["dy"], s["dstate"], s["lens"])))
    return {"loss": _loss_plain, "grad": _grad_plain, "delta": _delta_plain, "delta_grad": _delta_grad_plain}[kind](s)


# -------------------------------------------------------------------- work
def work(case):
    if case["kind"] in ("loss", "grad"):
        N, C, V = case["N"], case["C"], case["V"]
        if case["kind"] == "loss":
            return {"bytes": 2 * C * (N + V) + 12 * N, "flops": 2 * N * C * V}
        # the logits again (none were kept), and the two gradients' products
        return {"bytes": 4 * C * (N + V) + 12 * N, "flops": 6 * N * C * V}
    B, T, H, D = (case[n] for n in "BTHD")
    live = T * 5 / 8 if case["ragged"] else T   # mean length; past it outputs are only written
    if case["kind"] == "delta":
        # a token reads the state with its key, writes to it, reads it with its query
        return {"bytes": B * H * (live * (6 * D + 8) + T * 2 * D + 8 * D * D),
                "flops": 6 * B * live * H * D * D}
    # the states again, and two products for each of the forward pass's
    return {"bytes": B * H * (live * (8 * D + 8) + T * (6 * D + 8) + 12 * D * D),
            "flops": 16 * B * live * H * D * D}


# ------------------------------------------------------------------- exact
def _head_exact(s):
    x, W, tok = s["x"].double(), s["W"].double(), s["targets"].tolist()
    N = len(tok)
    if s["kind"] == "loss":
        loss, lse = (torch.zeros(N, dtype=torch.float64, device=DEV) for _ in range(2))
        for i in range(0, N, 4096):
            z = x[i:i + 4096] @ W.t()
            lse[i:i + 4096] = torch.logsumexp(z, 1)
            rows = [j for j in range(i, min(N, i + 4096)) if tok[j] >= 0]
            if rows:
                at = torch.tensor(rows, device=DEV)
                loss[at] = lse[at] - z[at - i, torch.tensor([tok[j] for j in rows], device=DEV)]
        return {"loss": loss, "lse": lse}
    dx, dW = torch.zeros_like(x), torch.zeros_like(W)
    for i in range(0, N, 4096):
        xi, t = x[i:i + 4096], s["targets"][i:i + 4096].long()
        p = torch.softmax(xi @ W.t(), 1)
        hit = torch.nn.functional.one_hot(t.clamp_min(0), p.shape[1])
        dz = (p - hit) * (s["dloss"][i:i + 4096].double() * (t >= 0))[:, None]
        dx[i:i + 4096] = dz @ W
        dW += dz.t() @ xi
    return {"dx": dx, "dW": dW}


def _delta_exact(s):
    """Token by token, and back."""
    q, k, v, a, b, S = (s[n].double() for n in ("q", "k", "v", "log_decay", "beta", "state"))
    B, T, H, D = q.shape
    n = s["lens"].long() if s["lens"] is not None else torch.full((B,), T, device=DEV)
    back = s["kind"] == "delta_grad"
    y, states = torch.zeros_like(q), []
    for t in range(T):
        live = (t < n)[:, None, None, None]
        old = torch.exp(a[:, t])[..., None, None] * S
        u = b[:, t, :, None] * (v[:, t] - (old * k[:, t, :, :, None]).sum(2))
        S = torch.where(live, old + k[:, t, :, :, None] * u[:, :, None, :], S)
        if back:
            states.append((old, u, S))
        y[:, t] = (S * q[:, t, :, :, None]).sum(2) * live[..., 0]
    if not back:
        return {"y": y, "state": S}
    dy, G = s["dy"].double(), s["dstate"].double()
    out = {m: torch.zeros_like(q) for m in ("dq", "dk", "dv")}
    out |= {m: torch.zeros_like(a) for m in ("dlog_decay", "dbeta")}
    for t in range(T - 1, -1, -1):
        live = (t < n)[:, None, None, None]
        old, u, S = states.pop()
        E = G + q[:, t, :, :, None] * dy[:, t, :, None, :]
        du = (E * k[:, t, :, :, None]).sum(2)
        left = -b[:, t, :, None] * du
        full = E + k[:, t, :, :, None] * left[:, :, None, :]
        one = {"dq": (S * dy[:, t, :, None, :]).sum(3), "dv": -left,
               "dk": (E * u[:, :, None, :]).sum(3) + (old * left[:, :, None, :]).sum(3),
               "dbeta": (du * (v[:, t] - (old * k[:, t, :, :, None]).sum(2))).sum(2),
               "dlog_decay": (full * old).sum((2, 3))}
        for m, x in one.items():
            out[m][:, t] = torch.where(live.reshape((B,) + (1,) * (x.dim() - 1)), x, 0.0)
        G = torch.where(live, torch.exp(a[:, t])[..., None, None] * full, G)
    out["dstate"] = G
    return out


def exact(case, seed):
    if case["kind"] == "delta_grad" and case["B"] * case["T"] * case["H"] * case["D"] ** 2 > 3.5e9:
        return None                             # three states a token in 64 bits: 84 GB
    s = prepare(case, seed)
    return (_head_exact if case["kind"] in ("loss", "grad") else _delta_exact)(s)
