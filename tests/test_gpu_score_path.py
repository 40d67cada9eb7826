"""The scoring path on the model (cpp_path.score_packed_batched, the engine's
score_tokens_batched and estimate, the command line), and the new operators run
together as one block of a model with heads on 4-bit weights."""
import json

import numpy as np
import pytest
import torch

from krunch_amd import cli, cpp_path, krunch_ac_hip as ops, synthetic
from krunch_amd.inference import HEADER_SIZE, InferenceEngine, coder_bits

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(scope="module")
def small():
    w = synthetic.make_weights(n_layer=2, C=256, F=512, V=1003, seed=3)
    yield InferenceEngine().load(w)
    cpp_path.release_weights(w)


def streams(lens, V, seed):
    rng = np.random.default_rng(seed)
    return [rng.integers(0, V, n).astype(np.int32) for n in lens]


def test_scores_are_those_of_the_packed_logits(small):
    """In head blocks of any size, and over two calls that carry the state."""
    W = small.weights
    B, T, V = 3, 50, 1003
    g = torch.Generator().manual_seed(1)
    ids = torch.randint(0, V, (B, T), generator=g)
    tgt = torch.randint(0, V, (B, T), generator=g)
    tgt[1, 40:] = -1
    st = cpp_path.fresh_state_batched(W, B)
    logits = cpp_path.forward_packed_batched(W, ids, st)
    ref = ops.token_scores(logits, tgt.reshape(-1).to(torch.int32).to(DEV), 4)
    for rows in (8192, 64, 7):
        st = cpp_path.fresh_state_batched(W, B)
        parts = [cpp_path.score_packed_batched(W, ids[:, a:b], tgt[:, a:b], st, 4, rows)
                 for a, b in ((0, 31), (31, 50))]
        got = [torch.cat(c, 1) for c in zip(*parts)]
        for a, b in zip(ref, got):
            assert torch.equal(a.reshape(b.shape), b)
    assert (got[0][1, 40:] == 0).all()
    empty = cpp_path.score_packed_batched(W, ids[:, :0], tgt[:, :0], st, 2)
    assert [tuple(c.shape) for c in empty] == [(B, 0), (B, 0), (B, 0, 2), (B, 0, 2)]
    before = st.buf.clone()
    for bad in ((ids, tgt[:, 1:]), (ids + V, tgt), (ids, tgt - 2)):
        with pytest.raises(ValueError):
            cpp_path.score_packed_batched(W, *bad, st)
    for n in (-1, 33):
        with pytest.raises(ValueError):
            cpp_path.score_packed_batched(W, ids, tgt, st, n)
    assert torch.equal(st.buf, before)


def test_ragged_streams_over_windows(small):
    small.window = 64
    try:
        toks = streams([1, 200, 64, 65, 130, 7], 1003, 2)
        got = small.score_tokens_batched(toks, 3)
        for t, s in zip(toks, got):
            one = small.score_tokens_batched([t], 3)[0]
            assert s.logprob.shape == (len(t),) and s.top_token.shape == (len(t), 3)
            for a, b in zip(s, one):
                assert np.array_equal(a, b)
    finally:
        small.window = 1024
    assert small.score_tokens_batched([]) == []
    for bad in ([np.zeros(0, np.int32)], [np.array([1003])], [np.array([-1])]):
        with pytest.raises(ValueError):
            small.score_tokens_batched(bad)


@pytest.mark.parametrize("w8a8", [False, True])
def test_scores_are_the_coder_s_cost(w8a8):
    """Payload bits against the tokens' counts: the coder's interval of count c out
    of 2^24 is floored at both ends of a range of at least 2^30, so off by at most
    one part in 64 c; a row's most likely token has up to V counts more than
    coder_bits gives it; the end of a stream takes up to 16 bits."""
    w = synthetic.make_weights(n_layer=2, C=256, F=512, V=1003, seed=3)
    eng = InferenceEngine().load(w, w8a8=w8a8)
    toks = synthetic.zipf_tokens(5, 300, seed_base=7, repeat_rate=0.05)
    toks = [np.minimum(t, 1002)[:n] for t, n in zip(toks, (300, 1, 77, 250, 300))]
    for t, s, payload in zip(toks, eng.score_tokens_batched(toks, 1), eng.compress_tokens_batched(toks)):
        V, bits = 1003, coder_bits(s.logprob, 1003)
        counts = np.floor(np.exp(s.logprob.astype(np.float64)) * (2 ** 24 - V)) + 1
        # the scores' own errors (2^-16 of a count's logarithm), the floor's side and the coder
        slack = (1.4427 * 1.05 * (1 / (64 * counts) + 1 / counts) + 2.0 ** -15).sum() + 16
        extra = (np.log2(1 + V / counts) * (s.top_token[:, 0] == t)).sum()
        assert bits - slack - extra <= 8 * (len(payload) - 8) <= bits + slack
    cpp_path.release_weights(w)


def test_estimate_and_the_command_line(tmp_path, monkeypatch):
    monkeypatch.delenv("KRUNCH_WEIGHTS", raising=False)
    monkeypatch.delenv("KRUNCH_TOKENIZER", raising=False)
    eng = InferenceEngine().load(synthetic.make_weights())
    raw = ("scored on MI355X, ünïcödé " * 60).encode()
    for size in (None, 300):
        blob = eng.compress(raw, chunk_size=size)
        est = eng.estimate(raw, chunk_size=size)
        assert est > HEADER_SIZE and abs(est - len(blob)) <= 0.01 * len(blob) + 4 * 8
    src, out = tmp_path / "in", tmp_path / "out"
    src.write_bytes(raw)
    assert cli.main(["estimate", "--in", str(src), "--out", str(out)]) == 0
    line = json.loads(out.read_text())
    assert line["bytes"] == len(raw) and line["estimate"] == eng.estimate(raw)


# ---------------------------------------------------------------- together

C, H, D, V = 256, 4, 64, 777


def block_weights(seed):
    g = torch.Generator().manual_seed(seed)
    make = lambda k, n: ops.quantize_w4((torch.randn(k, n, generator=g) * k ** -0.5).half().to(DEV), 64)
    w = {n: make(C, C) for n in "rkvo"}
    w["fk"], w["fv"], w["head"] = make(C, 4 * C), make(4 * C, C), make(C, V)
    w["decay"] = -torch.exp(torch.linspace(-5.0, 0.5, H)).to(DEV)
    w["first"] = torch.full((H,), 0.4, device=DEV)
    return w


def block(w, x, state, targets, chunked):
    """x fp16 [B, T, C] through one block on 4-bit weights and the head, scored."""
    B, T, _ = x.shape
    rows = x.reshape(B * T, C)
    r, k, v = (ops.det_matmul_w4(rows, w[n]).view(B, T, H, D) for n in "rkv")
    y = ops.wkv_heads(r, k, v, w["decay"], w["first"], state, chunked=chunked)
    rows = ops.det_matmul_w4(y.view(B * T, C), w["o"], epilogue="residual", res=rows)
    key = ops.det_matmul_w4(rows, w["fk"], epilogue="relu2")
    rows = ops.det_matmul_w4(key, w["fv"], epilogue="residual", res=rows)
    logits = ops.det_matmul_w4(rows, w["head"], torch.float32)
    return (r, k, v, y, logits), ops.token_scores(logits, targets.reshape(-1), 5)


def test_block_token_by_token_equals_the_prompt():
    """The recurrent form end to end: every operator's rows are the same bits alone
    and in a batch, so 20 streams x 30 tokens at once equal the tokens one by one,
    here from one captured graph."""
    w = block_weights(1)
    B, T = 20, 30
    g = torch.Generator().manual_seed(2)
    x = (0.5 * torch.randn(B, T, C, generator=g)).half().to(DEV)
    tgt = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32).to(DEV)
    state = torch.zeros(B, H, D, D, device=DEV)
    _, whole = block(w, x, state, tgt, chunked=False)
    step_x, step_t = x[:, :1].contiguous(), tgt[:, :1].contiguous()
    step_state = torch.zeros_like(state)
    block(w, step_x, step_state, step_t, chunked=False)      # before the capture
    step_state.zero_()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, out = block(w, step_x, step_state, step_t, chunked=False)
    for t in range(T):
        step_x.copy_(x[:, t:t + 1])
        step_t.copy_(tgt[:, t:t + 1])
        graph.replay()
        for a, b in zip(whole, out):
            assert torch.equal(a.view(B, T, *a.shape[1:])[:, t], b), t
    assert torch.equal(step_state, state)


def test_block_of_a_prompt_against_its_formulas():
    """The chunked form: each stage in float64 from the values it was given."""
    w = block_weights(3)
    B, T = 2, 200
    g = torch.Generator().manual_seed(4)
    x = (0.5 * torch.randn(B, T, C, generator=g)).half().to(DEV)
    tgt = torch.randint(0, V, (B, T), generator=g, dtype=torch.int32).to(DEV)
    state = torch.zeros(B, H, D, D, device=DEV)
    (r, k, v, y, logits), (lp, h, tl, tt) = block(w, x, state, tgt, chunked=True)
    rd, kd, vd = (t.double().cpu() for t in (r, k, v))
    S, u = torch.zeros(B, H, D, D, dtype=torch.float64), 0.4
    A = S.clone()
    decay = torch.exp(w["decay"].double().cpu())[None, :, None, None]
    for t in range(T):
        kv = kd[:, t, :, :, None] * vd[:, t, :, None, :]
        a = rd[:, t, :, :, None]
        ref, size = (a * (S + u * kv)).sum(2), (a.abs() * (A + u * kv.abs())).sum(2)
        # fp16's half step, and the parts' and sums' 2^-18 of the absolute sum
        assert ((y[:, t].double().cpu() - ref).abs() <= 2.0 ** -11 * ref.abs() + 2.0 ** -18 * size + 2.0 ** -25).all()
        S, A = decay * S + kv, decay * A + kv.abs()
    z = logits.double().cpu()
    ref = torch.log_softmax(z, 1)
    want = ref.gather(1, tgt.reshape(-1, 1).long().cpu())[:, 0]
    assert ((lp.double().cpu() - want).abs() <= 2.0 ** -16).all()
    assert ((h.double().cpu() + (ref.exp() * ref).sum(1)).abs() <= 2.0 ** -15).all()
    best = torch.sort(z, dim=1, descending=True, stable=True)
    assert torch.equal(tt.cpu().long(), best.indices[:, :5])
