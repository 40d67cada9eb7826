"""What the speed of the scoring and small-model operators is measured on:
scores of tokens from logits, products with 4-bit weights, and the WKV
recurrence with one decay per head, each through its public entry point.

They are what a scorer or a stepped decoder runs beside the codec. A text's
cost in bits is the sum of its tokens' log probabilities, read from the same
[rows, vocabulary] logits that the coder's CDF stage reads. A model whose
weights are kept in 4 bits steps a few streams at a time, so its products read
more weights than activations. A recurrence with a matrix state per head runs
over whole prompts, and token by token after them.

Sizes are the 169M configuration's (width 768, vocabulary 50277, heads of 64),
its neighbours' (width 256..1024, heads of 128) and the byte tokenizer's (256).
"""
from __future__ import annotations

import math

import torch

own = False          # True: run() calls the framework; False: the plain form

DEV = "cuda"
W4_K = 128           # a packed block of 4-bit weights: 16 outputs x 128 inputs


def listed():
    return [
        # Next-token scores and five alternatives of one stream: latency.
        {"name": "scores_1x50277_top5", "kind": "scores", "N": 1, "V": 50277, "f32": False, "top": 5, "masked": False},
        # A text's log probabilities and entropies only, over an alphabet part
        # of which a caller has masked with -inf; an odd row count.
        {"name": "scores_301x50277_masked", "kind": "scores", "N": 301, "V": 50277, "f32": False, "top": 0, "masked": True},
        # Byte-level model, many short rows, fp32 logits.
        {"name": "scores_30000x256_f32", "kind": "scores", "N": 30000, "V": 256, "f32": True, "top": 3, "masked": False},
        # One head block of a scoring window with alternatives (the largest).
        {"name": "scores_8192x50277_top8", "kind": "scores", "N": 8192, "V": 50277, "f32": False, "top": 8, "masked": False},
        # One stream's square projection.
        {"name": "w4_1x768x768", "kind": "w4", "M": 1, "K": 768, "N": 768, "group": 64, "f32": False},
        # One stream's head: the largest matrix against one row.
        {"name": "w4_1x768x50277", "kind": "w4", "M": 1, "K": 768, "N": 50277, "group": 64, "f32": False},
        # A few tens of streams through a channel-mix of width 1024, fine groups.
        {"name": "w4_40x1024x4096_g32", "kind": "w4", "M": 40, "K": 1024, "N": 4096, "group": 32, "f32": True},
        # The engine's default decode batch through the head.
        {"name": "w4_512x768x50277", "kind": "w4", "M": 512, "K": 768, "N": 50277, "group": 128, "f32": False},
        # One stream's next token.
        {"name": "heads_step_1", "kind": "heads", "B": 1, "T": 1, "H": 12, "D": 64, "ragged": False},
        # The engine's default batch, one token each.
        {"name": "heads_step_512", "kind": "heads", "B": 512, "T": 1, "H": 12, "D": 64, "ragged": False},
        # One prompt of odd length, wide heads.
        {"name": "heads_1x1777_wide", "kind": "heads", "B": 1, "T": 1777, "H": 8, "D": 128, "ragged": False},
        # A scoring window of prompts of different lengths.
        {"name": "heads_128x1024_ragged", "kind": "heads", "B": 128, "T": 1024, "H": 12, "D": 64, "ragged": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["scores", "w4", "heads"])
    if kind == "scores":
        V = rng.choice([50277, 256, _log(rng, 200, 160000)])
        return {"kind": kind, "N": _log(rng, 1, min(50000, 8192 * 50277 // V // 2)), "V": V,
                "f32": rng.random() < 0.3, "top": rng.choice([0, 1, 5, 20, rng.randint(2, 32)]),
                "masked": rng.random() < 0.3}
    if kind == "w4":
        K, N = rng.choice([(768, 768), (768, 50277), (1024, 1024), (1024, 4096), (512, 2048),
                           (32 * rng.randint(8, 64), _log(rng, 100, 20000))])
        return {"kind": kind, "M": _log(rng, 1, 512), "K": K, "N": N,
                "group": rng.choice([32, 64, 64, 128]), "f32": rng.random() < 0.3}
    D = rng.choice([64, 64, 128])
    H = rng.choice([4, 8, 12, 16]) * 64 // D
    if rng.random() < 0.35:
        T, B = 1, _log(rng, 1, 512)
    else:
        T = _log(rng, 2, 4096)
        B = _log(rng, 1, max(1, min(256, 2 ** 30 // (H * T * T) + 1, 100000 // T)))
    return {"kind": kind, "B": B, "T": T, "H": H, "D": D, "ragged": T > 1 and rng.random() < 0.4}


# ------------------------------------------------------------------ inputs
def _gen(seed, what):
    return torch.Generator(device=DEV).manual_seed(1000003 * int(seed) + what)


def _scores_inputs(case, seed):
    """Logits as a head gives them: a falling unigram part and a per-row part,
    so a row's entropy is a few nats; a text's tokens, one row in 64 without."""
    g = _gen(seed, 1)
    N, V = case["N"], case["V"]
    rank = torch.randperm(V, generator=g, device=DEV)
    prior = -1.1 * torch.log1p(rank.float())
    x = torch.empty((N, V), dtype=torch.float32 if case["f32"] else torch.float16, device=DEV)
    for i in range(0, N, 2048):
        rows = x[i:i + 2048]
        rows.copy_(2.0 * torch.randn(rows.shape, generator=g, device=DEV) + prior)
        if case["masked"]:
            rows.masked_fill_(torch.rand(rows.shape, generator=g, device=DEV) < 0.3, -math.inf)
    tokens = torch.randint(0, V, (N,), generator=g, device=DEV, dtype=torch.int32)
    if N > 1:
        tokens[torch.rand(N, generator=g, device=DEV) < 1 / 64] = -1
    return {"logits": x, "tokens": tokens}


def _w4_inputs(case, seed):
    """x [M, K] fp16, and a [K, N] weight in 4 bits: values q in -7..7 with one
    fp16 scale per output and group of inputs. The scales are [groups, N16]; the
    nibbles q + 8 are packed in blocks of 16 outputs x 128 inputs, 64 x 4 words:
    word c of lane l holds output l % 16, inputs 32c + 8(l / 16) + e, with
    e = 0, 2, 4, 6, 1, 3, 5, 7 from the low nibble up. Padding is q = 0, scale 0."""
    g = _gen(seed, 2)
    M, K, N, G = case["M"], case["K"], case["N"], case["group"]
    N16, KP = -(-N // 16) * 16, -(-K // W4_K) * W4_K
    W = torch.zeros((N16, KP), device=DEV)
    W[:N, :K] = torch.randn((N, K), generator=g, device=DEV).mul_(1 / math.sqrt(K)).half().float()
    scale = (W.reshape(N16, KP // G, G).abs().amax(2) / 7).half()
    s = scale.float().repeat_interleave(G, 1)
    q = torch.where(s > 0, torch.round(W / s.clamp_min(1e-30)), torch.zeros_like(W)).clamp_(-7, 7)
    nib = (q + 8).to(torch.int32)
    # [nb, 16, kb, 4 (c), 4 (l / 16), 4 (p % 4), 2 (p / 4)] -> words by (nb, kb, l / 16, l % 16, c)
    nib = nib.reshape(N16 // 16, 16, KP // W4_K, 4, 4, 4, 2).permute(0, 2, 4, 1, 3, 6, 5)
    shift = 4 * torch.arange(8, device=DEV, dtype=torch.int32).reshape(2, 4)
    words = (nib.to(torch.int64) << shift).sum((5, 6))
    words = torch.where(words >= 2 ** 31, words - 2 ** 32, words).to(torch.int32).contiguous()
    x = torch.randn((M, K), generator=g, device=DEV).half()
    return {"x": x, "q": words.reshape(-1), "scales": scale[:, :-(-K // G)].t().contiguous(), "K": K, "N": N,
            "group": G, "f32": case["f32"]}


def _heads_inputs(case, seed):
    """Receptance, key and value of B streams, decays from near 1 to a token or
    two, the state that earlier tokens left, and the lengths of ragged streams."""
    g = _gen(seed, 3)
    B, T, H, D = case["B"], case["T"], case["H"], case["D"]
    r, k, v = (torch.randn((B, T, H, D), generator=g, device=DEV).half() for _ in range(3))
    decay = -torch.exp(torch.linspace(-6.0, 0.7, H, device=DEV))
    first = 0.3 + torch.rand(H, generator=g, device=DEV)
    state = torch.randn((B, H, D, D), generator=g, device=DEV)
    lens = None
    if case["ragged"]:
        lens = torch.randint(max(1, T // 4), T + 1, (B,), generator=g, device=DEV, dtype=torch.int32)
    return {"r": r * 0.5, "k": k * 0.5, "v": v, "decay": decay, "first": first, "state": state,
            "lens": lens}


def prepare(case, seed):
    make = {"scores": _scores_inputs, "w4": _w4_inputs, "heads": _heads_inputs}[case["kind"]]
    state = make(case, seed)
    state["kind"] = case["kind"]
    state["top"] = case.get("top", 0)
    return state


# -------------------------------------------------------------- plain forms
def _scores_plain(s):
    x = s["logits"].float()
    N, V = x.shape
    m = x.amax(1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    d = x - m
    e = torch.exp(d)
    total = e.sum(1)
    log_total = torch.log(total)
    entropy = log_total - (e * d.clamp_min(-200.0)).sum(1) / total
    tok = s["tokens"].long()
    logprob = d.gather(1, tok.clamp_min(0)[:, None])[:, 0] - log_total
    out = {"logprob": torch.where(tok < 0, torch.zeros_like(logprob), logprob), "entropy": entropy}
    if s["top"]:
        # keys that order by value, then by lower index
        bits = (x + 0.0).view(torch.int32)
        bits = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).to(torch.int64)
        key = (bits << 32) | (V - 1 - torch.arange(V, device=x.device))
        best = torch.topk(key, s["top"], dim=1, sorted=True).values
        at = V - 1 - (best & 0xFFFFFFFF)
        out["top_token"] = at.to(torch.int32)
        out["top_logprob"] = d.gather(1, at) - log_total[:, None]
    return out


def _w4_plain(s):
    K, N, G = s["K"], s["N"], s["group"]
    N16, KP = -(-N // 16) * 16, -(-K // W4_K) * W4_K
    words = s["q"].reshape(N16 // 16, KP // W4_K, 4, 16, 4, 1, 1)
    shift = 4 * torch.arange(8, device=words.device, dtype=torch.int32).reshape(2, 4)
    nib = (words >> shift) & 15
    W = (nib - 8).permute(0, 3, 1, 4, 2, 6, 5).reshape(N16, KP)[:N, :K].float()
    scale = s["scales"].float().t().repeat_interleave(G, 1)[:N, :K]
    y = s["x"].float() @ (W * scale).t().contiguous()
    return y if s["f32"] else y.half()


def _heads_plain(s):
    """y_t = r_t (S + u k_t' v_t) and S <- e^w S + k_t' v_t, all t at once:
    y = (r k' weighted by e^(w (t - j - 1)), u on the diagonal) v + e^(w t) r S."""
    r, k, v = (s[n].permute(0, 2, 1, 3).float().contiguous() for n in ("r", "k", "v"))
    w, u, S = s["decay"], s["first"], s["state"]
    B, H, T, D = r.shape
    t = torch.arange(T, device=r.device)
    back = t[:, None] - t[None, :] - 1
    G = torch.exp(w[:, None, None] * back.clamp_min(0))
    G = torch.where(back >= 0, G, torch.where(back == -1, u[:, None, None], torch.zeros_like(G)))
    n = s["lens"].long() if s["lens"] is not None else torch.full((B,), T, device=r.device)
    live = (t[None, :] < n[:, None])[:, None, :, None]
    y = ((r @ k.transpose(2, 3).contiguous()) * G) @ v
    y = y + torch.exp(w[:, None] * t)[None, :, :, None] * (r @ S)
    y = torch.where(live, y, torch.zeros_like(y)).half().permute(0, 2, 1, 3).contiguous()
    left = (n[:, None, None] - 1 - t[None, None, :]).clamp_min(0)
    kd = torch.where(live, k * torch.exp(w[None, :, None] * left)[..., None], torch.zeros_like(k))
    S.mul_(torch.exp(w[None, :] * n[:, None])[..., None, None])
    S.add_(kd.transpose(2, 3).contiguous() @ v)
    return {"y": y, "state": S}


def run(state):
    kind = state["kind"]
    if own:
        from krunch_amd import krunch_ac_hip
        if kind == "scores":
            logprob, entropy, top_logprob, top_token = krunch_ac_hip.token_scores(
                state["logits"], state["tokens"], state["top"])
            out = {"logprob": logprob, "entropy": entropy}
            if state["top"]:
                out |= {"top_token": top_token, "top_logprob": top_logprob}
            return out
        if kind == "w4":
            w = krunch_ac_hip.W4(state["q"], state["scales"], state["K"], state["N"], state["group"])
            return krunch_ac_hip.det_matmul_w4(state["x"], w,
                                               torch.float32 if state["f32"] else torch.float16)
        y = krunch_ac_hip.wkv_heads(state["r"], state["k"], state["v"], state["decay"],
                                    state["first"], state["state"], state["lens"])
        return {"y": y, "state": state["state"]}
    return {"scores": _scores_plain, "w4": _w4_plain, "heads": _heads_plain}[kind](state)


# -------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "scores":
        # per logit: maximum, difference, exp, two sums and a product
        N, V = case["N"], case["V"]
        return {"bytes": N * V * (4 if case["f32"] else 2) + N * (12 + 8 * case["top"]),
                "flops": 6 * N * V}
    if case["kind"] == "w4":
        M, K, N, G = case["M"], case["K"], case["N"], case["group"]
        return {"bytes": K * N // 2 + 2 * N * -(-K // G) + 2 * M * K + M * N * (4 if case["f32"] else 2),
                "flops": 2 * M * K * N}
    B, T, H, D = (case[n] for n in "BTHD")
    T = T * 5 / 8 if case["ragged"] else T      # mean length; past it y is only written
    return {"bytes": B * H * D * (6 * T + 2 * case["T"]) + 8 * B * H * D * D + 8 * H,
            "flops": 4 * B * T * H * D * D}


# ------------------------------------------------------------------- exact
def _scores_exact(s):
    x, tok = s["logits"], s["tokens"].tolist()
    N, V = x.shape
    parts = []
    for i in range(0, N, 1024):
        z = x[i:i + 1024].double()
        lse = torch.logsumexp(z, 1)
        logp = z - lse[:, None]
        p = torch.exp(logp)
        h = -torch.where(p > 0, p * logp, torch.zeros_like(p)).sum(1)
        lp = torch.stack([logp[j, t] if t >= 0 else torch.zeros((), dtype=torch.float64, device=DEV)
                          for j, t in enumerate(tok[i:i + 1024])])
        got = [lp, h]
        if s["top"]:
            best, at = torch.sort(z, dim=1, descending=True, stable=True)
            got += [(best[:, :s["top"]] - lse[:, None]), at[:, :s["top"]].to(torch.int32)]
        parts.append(got)
    cols = [torch.cat(c) for c in zip(*parts)]
    out = {"logprob": cols[0], "entropy": cols[1]}
    if s["top"]:
        out |= {"top_logprob": cols[2], "top_token": cols[3]}
    return out


def _w4_exact(s):
    K, N, G = s["K"], s["N"], s["group"]
    kb = -(-K // W4_K)
    q = s["q"].reshape(-1, kb, 64, 4)
    n = torch.arange(N, device=DEV)
    y = torch.zeros((s["x"].shape[0], N), dtype=torch.float64, device=DEV)
    for b in range(kb):
        k = torch.arange(W4_K * b, min(K, W4_K * (b + 1)), device=DEV)
        c, lane_hi, e = (k % W4_K) // 32, k % 32 // 8, k % 8
        word = q[(n // 16)[None, :], b, (16 * lane_hi)[:, None] + (n % 16)[None, :], c[:, None]]
        place = 4 * (e // 2 + 4 * (e % 2))
        val = ((word >> place[:, None].to(torch.int32)) & 15).double() - 8
        y += s["x"][:, k].double() @ (val * s["scales"][k // G][:, n].double())
    return y


def _heads_exact(s):
    r, k, v, S = (s[n].double() for n in ("r", "k", "v", "state"))
    B, T, H, D = r.shape
    g, u = torch.exp(s["decay"].double())[None, :, None, None], s["first"].double()[None, :, None, None]
    n = s["lens"].long() if s["lens"] is not None else torch.full((B,), T, device=DEV)
    y = torch.zeros_like(r)
    for t in range(T):
        live = (t < n)[:, None, None, None]
        kv = k[:, t, :, :, None] * v[:, t, :, None, :]
        o = (r[:, t, :, :, None] * (S + u * kv)).sum(2)
        y[:, t] = torch.where(live[..., 0], o, torch.zeros_like(o))
        S = torch.where(live, g * S + kv, S)
    return {"y": y, "state": S}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "heads" and case["B"] * case["H"] * case["T"] * case["D"] ** 2 > 2e10:
        return None
    return {"scores": _scores_exact, "w4": _w4_exact, "heads": _heads_exact}[case["kind"]](s)
