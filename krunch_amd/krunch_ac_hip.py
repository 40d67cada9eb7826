"""Drop-in for the reference's `krunch_ac_cuda` extension ops, on the HIP library.

Same op names, argument order and in-place semantics as the pybind module
(`krunch_ac/cuda/main.cpp:114-303,354-466`, `layer_cpp.cpp:824-1052`): the
range-coder ops, det_softmax_cdf, det_matmul, rwkv4_layer_step_cpp,
rwkv4_layer_step_cpp_t1, rwkv4_layer_step_cpp_graphed,
clear_layer_graph_cache, read_phase_times and reset_phase_times;
the caller owns coder state and buffers (mutated in place, launches are
asynchronous on the current stream); ops that produce tensors allocate them.
Argument errors raise RuntimeError, as TORCH_CHECK does. Differences: every
call is bounds-checked against the buffers it is given; the CDF precision is
taken from the CDF itself (cdf[:, -1] = 2^precision) or passed explicitly;
the graphed layer op advances the state once per call (the reference's first
call advances it three times); the phase profiler reports this build's seven
kernel phases rather than the reference's eleven.
"""
from __future__ import annotations

import weakref
from dataclasses import dataclass

import torch

from krunch_amd import _lib

CDF_PRECISION = 24


def _check(cond, msg):
    if not cond:
        raise RuntimeError(msg)


def _cuda(t, dtype, name):
    _check(t.is_cuda, f"{name} must be a device tensor")
    _check(t.dtype == dtype, f"{name} must be {dtype}, got {t.dtype}")
    _check(t.is_contiguous(), f"{name} must be contiguous")


def _nbytes(t):
    return t.numel() * t.element_size()


def _cap(buf):
    """A coder buffer's byte length as the uint32 the C ABI takes (raises
    rather than truncating past 2^32 - 1)."""
    return _lib.u32(_nbytes(buf), "coder buffer bytes")


# ---------------------------------------------------------------------------
# range coder (encode_kernel.cu / decode_kernel.cu ops)
# ---------------------------------------------------------------------------

def encode_step(cdf, symbols, output_buf, state, precision: int = CDF_PRECISION):
    """Encode N rows of one stream: cdf int32 [N, V+1], symbols int32 [N]."""
    _cuda(cdf, torch.int32, "cdf"); _cuda(symbols, torch.int32, "symbols")
    _cuda(output_buf, torch.uint8, "output_buf"); _cuda(state, torch.uint32, "state")
    _check(cdf.dim() == 2 and symbols.numel() == cdf.shape[0], "cdf/symbols shape mismatch")
    _check(state.numel() >= 4, "state must hold 4 uint32")
    _lib.call("kr_encode_step", cdf.data_ptr(), cdf.shape[1], symbols.data_ptr(), cdf.shape[0],
              output_buf.data_ptr(), _cap(output_buf), state.data_ptr(), precision, None,
              _lib.stream_ptr())


def encode_finalize(output_buf, state):
    _cuda(output_buf, torch.uint8, "output_buf"); _cuda(state, torch.uint32, "state")
    _lib.call("kr_encode_finalize", output_buf.data_ptr(), _cap(output_buf), state.data_ptr(),
              None, _lib.stream_ptr())


def decode_init(input_buf, state):
    _cuda(input_buf, torch.uint8, "input_buf"); _cuda(state, torch.uint32, "state")
    _lib.call("kr_decode_init_batched", input_buf.data_ptr(), _cap(input_buf), None, None,
              state.data_ptr(), 1, _lib.stream_ptr())


def decode_step(cdf, input_buf, state, out_sym, precision: int = CDF_PRECISION):
    """Decode one symbol: cdf int32 [V+1]; out_sym int32 [1]."""
    _cuda(cdf, torch.int32, "cdf"); _cuda(input_buf, torch.uint8, "input_buf")
    _cuda(state, torch.uint32, "state"); _cuda(out_sym, torch.int32, "out_sym")
    V = cdf.numel() - 1
    _lib.call("kr_decode_step_batched", cdf.data_ptr(), V, input_buf.data_ptr(),
              _cap(input_buf), None, None, state.data_ptr(), out_sym.data_ptr(), 1, precision,
              _lib.stream_ptr())


def encode_step_batched(cdfs, symbols, output_buf, base_byte_offsets, states,
                        precision: int = CDF_PRECISION):
    _cuda(cdfs, torch.int32, "cdfs"); _cuda(symbols, torch.int32, "symbols")
    _cuda(output_buf, torch.uint8, "output_buf"); _cuda(base_byte_offsets, torch.int32, "offsets")
    _cuda(states, torch.uint32, "states")
    B = symbols.numel()
    _check(cdfs.dim() == 2 and cdfs.shape[0] == B and base_byte_offsets.numel() == B
           and states.numel() == 4 * B, "batched shapes mismatch")
    _lib.call("kr_encode_step_batched", cdfs.data_ptr(), cdfs.shape[1] - 1, symbols.data_ptr(),
              output_buf.data_ptr(), _cap(output_buf), base_byte_offsets.data_ptr(),
              states.data_ptr(), B, precision, None, _lib.stream_ptr())


def encode_finalize_batched(output_buf, base_byte_offsets, states):
    _cuda(output_buf, torch.uint8, "output_buf"); _cuda(base_byte_offsets, torch.int32, "offsets")
    _cuda(states, torch.uint32, "states")
    B = base_byte_offsets.numel()
    _check(states.numel() == 4 * B, "states must be [4*B]")
    _lib.call("kr_encode_finalize_batched", output_buf.data_ptr(), _cap(output_buf),
              base_byte_offsets.data_ptr(), states.data_ptr(), B, None, _lib.stream_ptr())


def decode_init_batched(input_buf, base_byte_offsets, states, byte_limits=None):
    _cuda(input_buf, torch.uint8, "input_buf"); _cuda(base_byte_offsets, torch.int32, "offsets")
    _cuda(states, torch.uint32, "states")
    B = base_byte_offsets.numel()
    _check(states.numel() == 4 * B, "states must be [4*B]")
    _lib.call("kr_decode_init_batched", input_buf.data_ptr(), _cap(input_buf),
              base_byte_offsets.data_ptr(), _lib.ptr(byte_limits), states.data_ptr(), B,
              _lib.stream_ptr())


def decode_step_batched(cdfs, input_buf, base_byte_offsets, states, out_syms, byte_limits=None,
                        precision: int = CDF_PRECISION):
    _cuda(cdfs, torch.int32, "cdfs"); _cuda(input_buf, torch.uint8, "input_buf")
    _cuda(base_byte_offsets, torch.int32, "offsets"); _cuda(states, torch.uint32, "states")
    _cuda(out_syms, torch.int32, "out_syms")
    B = out_syms.numel()
    _check(cdfs.dim() == 2 and cdfs.shape[0] == B and states.numel() == 4 * B,
           "batched shapes mismatch")
    _lib.call("kr_decode_step_batched", cdfs.data_ptr(), cdfs.shape[1] - 1, input_buf.data_ptr(),
              _cap(input_buf), base_byte_offsets.data_ptr(), _lib.ptr(byte_limits),
              states.data_ptr(), out_syms.data_ptr(), B, precision, _lib.stream_ptr())


# ---------------------------------------------------------------------------
# softmax -> CDF (det_softmax_cdf.cu op)
# ---------------------------------------------------------------------------

def _precision_of(cdf_T_value: int) -> int:
    p = int(cdf_T_value).bit_length() - 1
    _check(p >= 1 and (1 << p) == int(cdf_T_value), "cdf_T_value must be a power of two")
    return p


def det_softmax_cdf(logits, cdf_T_value: int):
    """fp16 logits [T, V] -> int32 [T, V+1]: column 0 = 0, columns 1..V the
    per-symbol counts (deficit applied); the caller scans (cpp_path.py:490-501)."""
    _cuda(logits, torch.float16, "logits")
    _check(logits.dim() == 2, "logits must be [T, V]")
    T, V = logits.shape
    out = torch.empty((T, V + 1), dtype=torch.int32, device=logits.device)
    _lib.call("kr_softmax_cdf", logits.data_ptr(), T, V, V, out.data_ptr(), 0,
              _precision_of(cdf_T_value), _lib.stream_ptr())
    return out


def softmax_cdf(logits, cdf_T_value: int = 1 << CDF_PRECISION):
    """fp16 logits [T, V] -> cumulative int32 CDF [T, V+1] in one kernel."""
    _cuda(logits, torch.float16, "logits")
    T, V = logits.shape
    out = torch.empty((T, V + 1), dtype=torch.int32, device=logits.device)
    _lib.call("kr_softmax_cdf", logits.data_ptr(), T, V, V, out.data_ptr(), 1,
              _precision_of(cdf_T_value), _lib.stream_ptr())
    return out


def softmax_probs(logits):
    """fp16 logits [T, V] -> float32 softmax probabilities (the CDF's input)."""
    _cuda(logits, torch.float16, "logits")
    T, V = logits.shape
    out = torch.empty((T, V), dtype=torch.float32, device=logits.device)
    _lib.call("kr_softmax_probs", logits.data_ptr(), T, V, V, out.data_ptr(), _lib.stream_ptr())
    return out


# The operators below launch on the current stream of their tensors' device, and
# check with "condition or _refuse(message)": a message is only made for a call
# that is refused (a small call's time is the host's). Their outputs carry no
# gradient, whatever their inputs require.

def _refuse(msg):
    raise RuntimeError(msg)


def _on_device_of(t, op, *args):
    """op(*args) with t's device current."""
    with torch.cuda.device(t.device):
        return op(*args)


def _elsewhere(t):
    return not _lib.is_current(t.get_device())


TOP_TOKENS_MAX = 32


def token_scores(logits, tokens, n_top: int = 0):
    """Log probabilities of given tokens, entropies and the most likely tokens
    of rows of logits, in nats: logits [N, V] fp16 or fp32 (rows may be strided),
    tokens int32 [N] -> (logprob [N], entropy [N], top_logprob [N, n_top],
    top_token int32 [N, n_top]). A token of -1 is none (logprob 0); other ids
    outside 0..V-1 give NaN. Logits of -inf are masked tokens: never among the
    top ones, whose missing places hold -1 and -inf. A row of only masked tokens
    has logprob -inf and entropy 0, one with a NaN or +inf is NaN. Equal logits
    are ranked by lower id. n_top <= 32. No gradient."""
    logits.is_cuda or _refuse("logits must be a device tensor")
    f32 = logits.dtype is torch.float32
    f32 or logits.dtype is torch.float16 or _refuse(
        f"logits must be float16 or float32, got {logits.dtype}")
    logits.dim() == 2 or _refuse("logits must be [N, V]")
    N, V = logits.shape
    ld, step = logits.stride()
    if N <= 1:
        ld = V
    (V >= 1 and (step == 1 or V == 1) and ld >= V) or _refuse(
        "logits rows must be contiguous and not overlap")
    (tokens.is_cuda and tokens.dtype is torch.int32 and tokens.is_contiguous()) or _refuse(
        "tokens must be a contiguous int32 device tensor")
    tokens.get_device() == logits.get_device() or _refuse("tokens and logits must be on one device")
    tokens.shape == (N,) or _refuse(f"tokens must be [N] = [{N}]")
    0 <= n_top <= min(TOP_TOKENS_MAX, V) or _refuse(
        f"n_top must be in 0..{min(TOP_TOKENS_MAX, V)}, got {n_top}")
    if _elsewhere(logits):
        return _on_device_of(logits, token_scores, logits, tokens, n_top)
    logprob = torch.empty_like(tokens, dtype=torch.float32)
    entropy = torch.empty_like(logprob)
    top_logprob = logprob.new_empty((N, n_top))
    top_token = tokens.new_empty((N, n_top))
    _lib.call("kr_token_scores", logits.data_ptr(), f32, N, V, ld, tokens.data_ptr(),
              logprob.data_ptr(), entropy.data_ptr(), n_top, top_logprob.data_ptr(),
              top_token.data_ptr(), _lib.stream_ptr())
    return logprob, entropy, top_logprob, top_token


def _head_rows(t, name, C):
    """Row stride of a [rows, C] fp16 operand of a head."""
    (t.is_cuda and t.dtype is torch.float16 and t.dim() == 2) or _refuse(
        f"{name} must be a 2-dimensional float16 device tensor")
    t.shape[1] == C or _refuse(f"{name} has {t.shape[1]} columns, the head {C}")
    ld, step = t.stride()
    if t.shape[0] <= 1:
        ld = C
    (step == 1 and C <= ld < 1 << 21 and ld % 8 == 0 and t.data_ptr() % 16 == 0) or _refuse(
        f"{name} rows must be contiguous, 16-byte aligned and not overlap, their stride below 2^21")
    return ld


def _head_vector(t, dtype, name, N, dev):
    (t.is_cuda and t.dtype is dtype and t.is_contiguous() and t.shape == (N,) and t.get_device() == dev) or _refuse(
        f"{name} must be a contiguous {dtype} device tensor [N] = [{N}] on x's device")


def _head_shapes(x, W, targets):
    W.dim() == 2 or _refuse("W must be [V, C]")
    V, C = W.shape
    (V >= 1 and 64 <= C <= 16384 and C % 64 == 0) or _refuse(
        f"W must be [V, C] with C a multiple of 64 up to 16384, got {tuple(W.shape)}")
    ldx, ldw = _head_rows(x, "x", C), _head_rows(W, "W", C)
    N = x.shape[0]
    (max(N, V) <= 1 << 24 and N * V <= 1 << 44) or _refuse("N and V must be at most 2^24, N * V at most 2^44")
    dev = x.get_device()
    W.get_device() == dev or _refuse("x and W must be on one device")
    _head_vector(targets, torch.int32, "targets", N, dev)
    return N, C, V, ldx, ldw


def head_loss(x, W, targets):
    """Cross entropy in nats of the next tokens under a head, without its logits:
    x fp16 [N, C] (what the head reads, normalised), W fp16 [V, C] (as a prepared
    model keeps its head; rows of both may be strided), targets int32 [N] -> (loss
    [N], lse [N]) fp32 with z = x @ W.T, lse = logsumexp(z), loss = lse -
    z[target]. A target of -1 is none (loss 0); other ids outside 0..V-1 give NaN.
    C must be a multiple of 64. z stays in fp32, so a loss differs from
    token_scores' of fp16 logits by their rounding. No autograd:
    head_loss_backward takes lse and gives the gradients."""
    N, C, V, ldx, ldw = _head_shapes(x, W, targets)
    if _elsewhere(x):
        return _on_device_of(x, head_loss, x, W, targets)
    loss = torch.empty_like(targets, dtype=torch.float32)
    lse = torch.empty_like(loss)
    nbytes = _lib.lib().kr_head_loss_workspace_bytes(N, C, V)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.call("kr_head_loss", x.data_ptr(), ldx, N, C, W.data_ptr(), ldw, V, targets.data_ptr(),
              loss.data_ptr(), lse.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_ptr())
    return loss, lse


def head_loss_backward(x, W, targets, lse, dloss, out_dtype=None, dx: bool = True, dW: bool = True):
    """Gradients of head_loss: x, W, targets as there, its lse, and dloss fp32 [N]
    (the gradient of each loss) -> (dx [N, C], dW [V, C]), fp16 or fp32 by
    out_dtype, None for one that is not wanted. Rows with target -1 or dloss 0 have
    no gradient. For fp16 outputs the gradient of the logits is rounded to fp16 relative
    to the largest |dloss|, but for the target's, and dloss may carry a loss scale; for
    fp32 outputs it keeps 22 bits (the products take twice as long). Sums are fp32."""
    N, C, V, ldx, ldw = _head_shapes(x, W, targets)
    dev = x.get_device()
    _head_vector(lse, torch.float32, "lse", N, dev)
    _head_vector(dloss, torch.float32, "dloss", N, dev)
    f32 = out_dtype is torch.float32
    f32 or out_dtype in (None, torch.float16) or _refuse(f"out_dtype must be float16 or float32, got {out_dtype}")
    if _elsewhere(x):
        return _on_device_of(x, head_loss_backward, x, W, targets, lse, dloss, out_dtype, dx, dW)
    dtype = torch.float32 if f32 else torch.float16
    gx = x.new_empty((N, C), dtype=dtype) if dx else None
    gw = x.new_empty((V, C), dtype=dtype) if dW else None
    if N == 0:
        return gx, None if gw is None else gw.zero_()
    if not (dx or dW):
        return None, None
    nbytes = _lib.lib().kr_head_loss_backward_workspace_bytes(N, C, V, 1 if dx else 0, 1 if dW else 0)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
    _lib.call("kr_head_loss_backward", x.data_ptr(), ldx, N, C, W.data_ptr(), ldw, V, targets.data_ptr(),
              lse.data_ptr(), dloss.data_ptr(), f32, _lib.ptr(gx), _lib.ptr(gw), ws.data_ptr(), nbytes,
              _lib.stream_ptr())
    return gx, gw


# ---------------------------------------------------------------------------
# matmul / layer ops (layer_cpp.cpp)
# ---------------------------------------------------------------------------

_WT_CACHE: dict = {}


def _copies(W, frag):
    """Device copies of a [K, N] weight, kept per live tensor object and
    version: pointers to the transposed one and, on request, to the
    fragment-packed one that the layer's products read (frag needs
    K % 32 == 0), and the tensors that hold them. Copies made while the stream
    is capturing are written when the graph runs, not now, so they serve that
    call only."""
    key = id(W)
    hit = known = _WT_CACHE.get(key)
    if hit is None or hit[0]() is not W or hit[1] != W._version:
        K, N = W.shape
        rows = (N + 15) // 16 * 16 if frag else 0
        buf = torch.empty((N + rows) * K, dtype=torch.float16, device=W.device)
        wt = buf.data_ptr()
        wf = wt + 2 * N * K if frag else None
        if frag:
            _lib.call("kr_transpose_pack_f16", W.data_ptr(), N, K, N, wt, K, wf, _lib.stream_ptr())
        else:
            _lib.call("kr_transpose_f16", W.data_ptr(), N, K, N, wt, K, _lib.stream_ptr())
        hit = (weakref.ref(W, lambda _r, k=key: _WT_CACHE.pop(k, None)), W._version, wt, wf, (buf,))
    elif frag and hit[3] is None:
        K, N = W.shape
        buf = torch.empty((N + 15) // 16 * 16 * K, dtype=torch.float16, device=W.device)
        _lib.call("kr_pack_fragments", hit[2], K, N, K, buf.data_ptr(), _lib.stream_ptr())
        hit = (*hit[:3], buf.data_ptr(), (*hit[4], buf))
    if hit is not known and not torch.cuda.is_current_stream_capturing():
        _WT_CACHE[key] = hit
    return hit[2:]


def det_matmul(x, W, out_dtype=None):
    """y = x @ W, x fp16 [M, K], W fp16 [K, N]; fp32 accumulation in a fixed
    K order, so each row's result does not depend on M."""
    _cuda(x, torch.float16, "x"); _cuda(W, torch.float16, "W")
    M, K = x.shape
    _check(W.shape[0] == K, "inner dimensions differ")
    N = W.shape[1]
    dtype = out_dtype or torch.float16
    out = torch.empty((M, N), dtype=dtype, device=x.device)
    ep = 0 if dtype == torch.float32 else 1
    wt, _, _keep = _copies(W, False)
    _lib.call("kr_det_matmul", x.data_ptr(), M, K, wt, K, N, out.data_ptr(), N,
              ep, None, None, _lib.stream_ptr())
    return out


@dataclass
class W4:
    """A [K, N] weight in 4 bits (kr_quantize_w4): q int32 [kr_w4_bytes / 4] in
    blocks of 16 outputs x 128 inputs, scales fp16 [ceil(K / group), N rounded up
    to 16], one per output and group of 32, 64 or 128 inputs."""
    q: torch.Tensor
    scales: torch.Tensor
    K: int
    N: int
    group: int = 64


def quantize_w4(W, group: int = 64) -> W4:
    """W fp16 [K, N] (y = x @ W; a transposed view will do) -> W4: weight q * s
    with s = fp16(max |w| / 7) over a group, q = w / s to the nearest integer in
    -7..7. K must be a multiple of 32. 4 bits a weight and 16 / group for its scale. No
    gradient."""
    (W.is_cuda and W.dtype is torch.float16) or _refuse("W must be a float16 device tensor")
    W.dim() == 2 or _refuse("W must be [K, N]")
    K, N = W.shape
    ldk, ldn = W.stride()
    (K >= 32 and K % 32 == 0) or _refuse(f"K = {K} must be a multiple of 32")
    (N >= 1 and ldk >= 1 and ldn >= 1) or _refuse("W must not be empty or broadcast")
    group in (32, 64, 128) or _refuse(f"group must be 32, 64 or 128, got {group}")
    if _elsewhere(W):
        return _on_device_of(W, quantize_w4, W, group)
    q = torch.empty(_lib.lib().kr_w4_bytes(N, K) // 4, dtype=torch.int32, device=W.device)
    scales = W.new_empty(((K + group - 1) // group, (N + 15) // 16 * 16))
    _lib.call("kr_quantize_w4", W.data_ptr(), ldk, ldn, N, K, group, q.data_ptr(),
              scales.data_ptr(), _lib.stream_ptr())
    return W4(q, scales, K, N, group)


EPILOGUES_W4 = {"none": 1, "sigmoid": 2, "relu2": 3, "residual": 4, "gated": 5}


def det_matmul_w4(x, W: W4, out_dtype=None, epilogue: str = "none", res=None, gate=None):
    """y = x @ W, x fp16 [M, K] (rows may be strided), W in 4 bits; exact products,
    fp32 sums and scales in a fixed order, so each row's result does not depend on
    M. fp16 out, or fp32 with epilogue "none". Epilogues on h = fp16(acc): "sigmoid"
    (h), "relu2" max(h, 0)^2, "residual" res + h, "gated" res + fp16(gate * h), with
    res and gate fp16 [M, N]. No gradient. For few rows: 768 x 50277 is faster in
    fp16 from about 100 rows on at groups of 32, 190 at 64, 260 at 128."""
    (x.is_cuda and x.dtype is torch.float16) or _refuse("x must be a float16 device tensor")
    x.dim() == 2 or _refuse("x must be [M, K]")
    M, K = x.shape
    q, scales, N, group = W.q, W.scales, W.N, W.group
    K == W.K or _refuse(f"inner dimensions differ: x has {K}, W {W.K}")
    ldx, step = x.stride()
    if M <= 1:
        ldx = K
    xp = x.data_ptr()
    (step == 1 and ldx >= K and ldx % 8 == 0 and xp % 16 == 0) or _refuse(
        "x rows must be contiguous, 16-byte aligned and not overlap")
    group in (32, 64, 128) or _refuse(f"group must be 32, 64 or 128, got {group}")
    (K >= 32 and K % 32 == 0 and N >= 1) or _refuse(f"bad W4 shape [{K}, {N}]")
    N16 = (N + 15) // 16 * 16
    (q.dtype is torch.int32 and q.is_contiguous() and q.numel() == N16 * ((K + 127) // 128) * 16
     and q.data_ptr() % 16 == 0) or _refuse("W.q does not hold a [K, N] weight")
    (scales.dtype is torch.float16 and scales.is_contiguous() and scales.data_ptr() % 8 == 0
     and scales.shape == ((K + group - 1) // group, N16)) or _refuse("W.scales must be [groups, N16]")
    dev = x.get_device()
    q.get_device() == scales.get_device() == dev or _refuse("x and W must be on one device")
    f32 = out_dtype is torch.float32
    f32 or out_dtype in (None, torch.float16) or _refuse(
        f"out_dtype must be float16 or float32, got {out_dtype}")
    epilogue in EPILOGUES_W4 or _refuse(f"epilogue must be one of {sorted(EPILOGUES_W4)}")
    f32 and epilogue != "none" and _refuse("an epilogue's output is float16")
    code = 0 if f32 else EPILOGUES_W4[epilogue]
    if code >= 4 or res is not None or gate is not None:
        for t, name, need in ((res, "res", code >= 4), (gate, "gate", code == 5)):
            (t is not None) == need or _refuse(f"epilogue {epilogue} takes {'a' if need else 'no'} {name}")
            if need:
                _cuda(t, torch.float16, name)
                (t.shape == (M, N) and t.get_device() == dev) or _refuse(f"{name} must be [{M}, {N}]")
    if _elsewhere(x):
        return _on_device_of(x, det_matmul_w4, x, W, out_dtype, epilogue, res, gate)
    out = x.new_empty((M, N), dtype=torch.float32) if f32 else x.new_empty((M, N))
    _lib.call("kr_det_matmul_w4", xp, ldx, M, K, q.data_ptr(), scales.data_ptr(), group, N,
              out.data_ptr(), N, code, _lib.ptr(res), _lib.ptr(gate), _lib.stream_ptr())
    return out


def wkv_heads(r, k, v, decay, first, state, lens=None, chunked: bool = True):
    """WKV with a matrix state per head: y_t = r_t (S + u k_t' v_t), then S <- e^w S
    + k_t' v_t. r, k, v fp16 [B, T, H, D], D 64 or 128 (heads contiguous; token
    strides free, so slices of one projection will do), decay (w <= 0) and first
    (u) fp32 [H], state fp32 [B, H, D, D] updated in place; returns y fp16
    [B, T, H, D]. lens int32 [B]: each stream's tokens (its state stops there, later
    rows of y are 0). chunked=True (prompts, scoring) takes 64 tokens at a time on
    the matrix units: equal up to rounding for finite inputs (a NaN or infinity of a
    token also reaches y of up to 63 tokens before it); chunked=False, and calls of
    at most 8 tokens, go token by token, and T tokens then have the bits of T calls,
    as a codec's two directions need. No gradient."""
    r.dim() == 4 or _refuse("r must be [B, T, H, D]")
    shape = r.shape
    B, T, H, D = shape
    (D in (64, 128) and H >= 1) or _refuse(f"r must have heads of 64 or 128 channels, got {tuple(shape)}")
    dev = r.get_device()
    C = H * D
    ld = []
    for t, name in ((r, "r"), (k, "k"), (v, "v")):
        (t.is_cuda and t.dtype is torch.float16) or _refuse(f"{name} must be a float16 device tensor")
        (t.shape == shape and t.get_device() == dev) or _refuse(
            f"{name} must be {tuple(shape)} on r's device")
        if B * T == 0:
            ld.append(C)
            continue
        sb, st, sh, sd = t.stride()
        if T == 1:
            st = sb if B > 1 else C
        (sd == 1 and (sh == D or H == 1) and st >= C and (sb == T * st or B == 1) and st % 8 == 0
         and t.data_ptr() % 16 == 0) or _refuse(
            f"{name}: heads must be contiguous, tokens evenly spaced and 16-byte aligned")
        ld.append(st)
    for t, name in ((decay, "decay"), (first, "first")):
        (t.is_cuda and t.dtype is torch.float32 and t.is_contiguous() and t.numel() == H
         and t.get_device() == dev) or _refuse(
            f"{name} must be a contiguous float32 device tensor [H] = [{H}] on r's device")
    (state.is_cuda and state.dtype is torch.float32 and state.is_contiguous()
     and state.shape == (B, H, D, D) and state.get_device() == dev
     and state.data_ptr() % 16 == 0) or _refuse(
        f"state must be a contiguous float32 device tensor {(B, H, D, D)} on r's device, 16-byte aligned")
    lens is None or (lens.is_cuda and lens.dtype is torch.int32 and lens.is_contiguous()
                     and lens.numel() == B and lens.get_device() == dev) or _refuse(
        f"lens must be a contiguous int32 device tensor [B] = [{B}] on r's device")
    if _elsewhere(r):
        return _on_device_of(r, wkv_heads, r, k, v, decay, first, state, lens, chunked)
    y = r.new_empty(shape)
    ws, nbytes = None, 0
    if chunked and T > 1:
        nbytes = _lib.lib().kr_wkv_heads_workspace_bytes(B, T, H, D)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=r.device)
    _lib.call("kr_wkv_heads", B, T, H, D, r.data_ptr(), ld[0], k.data_ptr(), ld[1], v.data_ptr(),
              ld[2], decay.data_ptr(), first.data_ptr(), _lib.ptr(lens), state.data_ptr(),
              y.data_ptr(), C, 1 if chunked else 0, _lib.ptr(ws), nbytes, _lib.stream_ptr())
    return y


def _delta_tokens(t, name, shape, dev):
    """Token stride of a [B, T, H, D] fp16 operand."""
    (t.is_cuda and t.dtype is torch.float16) or _refuse(f"{name} must be a float16 device tensor")
    (t.shape == shape and t.get_device() == dev) or _refuse(f"{name} must be {tuple(shape)} on q's device")
    B, T, H, D = shape
    if B * T == 0:
        return H * D
    sb, st, sh, sd = t.stride()
    if T == 1:
        st = sb if B > 1 else H * D
    (sd == 1 and (sh == D or H == 1) and st >= H * D and (sb == T * st or B == 1) and st % 8 == 0
     and t.data_ptr() % 16 == 0) or _refuse(
        f"{name}: heads must be contiguous, tokens evenly spaced and 16-byte aligned")
    return st


def _delta_gates(t, name, shape, dev):
    """Token stride of a [B, T, H] fp32 operand."""
    B, T, H, _ = shape
    (t.is_cuda and t.dtype is torch.float32 and t.shape == (B, T, H) and t.get_device() == dev) or _refuse(
        f"{name} must be a float32 device tensor {(B, T, H)} on q's device")
    if B * T == 0:
        return H
    sb, st, sh = t.stride()
    if T == 1:
        st = sb if B > 1 else H
    ((sh == 1 or H == 1) and st >= H and (sb == T * st or B == 1)) or _refuse(
        f"{name}: heads must be contiguous and tokens evenly spaced")
    return st


def _delta_state(t, name, shape, dev):
    B, _, H, D = shape
    (t.is_cuda and t.dtype is torch.float32 and t.is_contiguous() and t.shape == (B, H, D, D)
     and t.get_device() == dev and t.data_ptr() % 16 == 0) or _refuse(
        f"{name} must be a contiguous float32 device tensor {(B, H, D, D)} on q's device, 16-byte aligned")


def _delta_args(q, k, v, log_decay, beta, state, lens):
    q.dim() == 4 or _refuse("q must be [B, T, H, D]")
    shape = q.shape
    B, T, H, D = shape
    (D in (64, 128) and H >= 1) or _refuse(f"q must have heads of 64 or 128 channels, got {tuple(shape)}")
    dev = q.get_device()
    ld = [_delta_tokens(t, name, shape, dev) for t, name in ((q, "q"), (k, "k"), (v, "v"))]
    ld += [_delta_gates(t, name, shape, dev) for t, name in ((log_decay, "log_decay"), (beta, "beta"))]
    _delta_state(state, "state", shape, dev)
    lens is None or (lens.is_cuda and lens.dtype is torch.int32 and lens.is_contiguous()
                     and lens.numel() == B and lens.get_device() == dev) or _refuse(
        f"lens must be a contiguous int32 device tensor [B] = [{B}] on q's device")
    return shape, ld


def gated_delta(q, k, v, log_decay, beta, state, lens=None, chunked: bool = True):
    """The gated delta rule, a matrix state per head whose keys replace what they had
    stored: S <- e^g S; u = beta (v_t - k_t S); S <- S + k_t' u; y_t = q_t S. q, k, v
    fp16 [B, T, H, D], D 64 or 128, log_decay (g <= 0) and beta fp32 [B, T, H] (heads
    contiguous; token strides free, so slices of one projection will do), state fp32
    [B, H, D, D] updated in place; returns y fp16 [B, T, H, D]. Keys are usually
    normalised by the caller and beta is in 0..1. lens int32 [B]: each stream's tokens (its
    state stops there, later rows of y are 0). chunked=True (prompts, scoring, training)
    takes 64 tokens at a time on the matrix units: equal up to rounding for finite inputs;
    chunked=False, and calls of at most 8 tokens, go token by token, and T tokens then
    have the bits of T calls. No autograd: gated_delta_backward gives the gradients."""
    shape, ld = _delta_args(q, k, v, log_decay, beta, state, lens)
    if _elsewhere(q):
        return _on_device_of(q, gated_delta, q, k, v, log_decay, beta, state, lens, chunked)
    B, T, H, D = shape
    y = q.new_empty(shape)
    ws, nbytes = None, 0
    if chunked and T > 1:
        nbytes = _lib.lib().kr_gated_delta_workspace_bytes(B, T, H, D)
        if nbytes:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _lib.call("kr_gated_delta", B, T, H, D, q.data_ptr(), ld[0], k.data_ptr(), ld[1], v.data_ptr(), ld[2],
              log_decay.data_ptr(), ld[3], beta.data_ptr(), ld[4], _lib.ptr(lens), state.data_ptr(),
              y.data_ptr(), H * D, 1 if chunked else 0, _lib.ptr(ws), nbytes, _lib.stream_ptr())
    return y


def gated_delta_backward(q, k, v, log_decay, beta, state, dy, dstate=None, lens=None):
    """Gradients of gated_delta: its inputs, with state as it was BEFORE the call
    (which updates it in place), dy fp16 [B, T, H, D] and dstate fp32 [B, H, D, D], the
    gradient of the state after the call (None: zeros) -> (dq, dk, dv fp16 [B, T, H, D],
    dlog_decay, dbeta fp32 [B, T, H], dstate fp32 [B, H, D, D] of the state before).
    Tokens past lens have gradient 0, and so has a log_decay above 0 or below -10000.
    Its states are computed again: nothing is kept from the forward call."""
    shape, ld = _delta_args(q, k, v, log_decay, beta, state, lens)
    dev = q.get_device()
    ldy = _delta_tokens(dy, "dy", shape, dev)
    dstate is None or _delta_state(dstate, "dstate", shape, dev)
    if _elsewhere(q):
        return _on_device_of(q, gated_delta_backward, q, k, v, log_decay, beta, state, dy, dstate, lens)
    B, T, H, D = shape
    dq, dk, dv = (q.new_empty(shape) for _ in range(3))
    dg, db = (state.new_empty((B, T, H)) for _ in range(2))
    if B * T == 0:
        return dq, dk, dv, dg, db, torch.zeros_like(state) if dstate is None else dstate.detach().clone()
    d0 = torch.empty_like(state)
    nbytes = _lib.lib().kr_gated_delta_backward_workspace_bytes(B, T, H, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=q.device)
    _lib.call("kr_gated_delta_backward", B, T, H, D, q.data_ptr(), ld[0], k.data_ptr(), ld[1], v.data_ptr(),
              ld[2], log_decay.data_ptr(), ld[3], beta.data_ptr(), ld[4], _lib.ptr(lens), state.data_ptr(),
              dy.data_ptr(), ldy, _lib.ptr(dstate), dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), dg.data_ptr(),
              db.data_ptr(), d0.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_ptr())
    return dq, dk, dv, dg, db, d0


def _layer_struct(x, att_xx, aa, bb, pp, ffn_xx, ln1_w, ln1_b, tm_k, tm_v, tm_r, time_decay,
                  time_first, Kw, Vw, Rw, Ow, ln2_w, ln2_b, ffn_tm_k, ffn_tm_r, ffn_Kw, ffn_Vw,
                  ffn_Rw):
    """Validate one layer call and build its kr_layer_weights; returns the
    struct, (C, F) and the device copies it points at (keep them alive)."""
    _cuda(x, torch.float16, "x")
    _check(x.dim() == 3, "x must be [B, T, C]")
    B, T, C = x.shape
    F = ffn_Kw.shape[1]
    dev = x.device
    keep = []

    def h(t):
        t = t.to(device=dev, dtype=torch.float16).reshape(-1).contiguous()
        _check(t.numel() == C, "layer vectors must hold C values")
        keep.append(t)
        return t.data_ptr()

    def f32(t):
        t = t.to(device=dev, dtype=torch.float32).reshape(-1).contiguous()
        _check(t.numel() == C, "time_decay / time_first must hold C values")
        keep.append(t)
        return t.data_ptr()

    def wt(m, k, n):
        _cuda(m, torch.float16, "weight")
        _check(tuple(m.shape) == (k, n), f"weight must be [{k}, {n}], got {tuple(m.shape)}")
        wt_ptr, wf_ptr, held = _copies(m, True)
        keep.append(held)
        return wt_ptr, wf_ptr

    L = _lib.KrLayerWeights()
    L.ln1_w, L.ln1_b, L.tm_k, L.tm_v, L.tm_r = map(h, (ln1_w, ln1_b, tm_k, tm_v, tm_r))
    L.decay, L.first = f32(time_decay), f32(time_first)
    (L.Kt, L.Kf), (L.Vt, L.Vf), (L.Rt, L.Rf), (L.Ot, L.Of) = (wt(m, C, C) for m in (Kw, Vw, Rw, Ow))
    L.ln2_w, L.ln2_b, L.ftm_k, L.ftm_r = map(h, (ln2_w, ln2_b, ffn_tm_k, ffn_tm_r))
    (L.fKt, L.fKf), (L.fVt, L.fVf), (L.fRt, L.fRf) = (wt(ffn_Kw, C, F), wt(ffn_Vw, F, C),
                                                      wt(ffn_Rw, C, C))
    for t, dt, n in ((att_xx, torch.float16, "att_xx"), (aa, torch.float32, "aa"),
                     (bb, torch.float32, "bb"), (pp, torch.float32, "pp"),
                     (ffn_xx, torch.float16, "ffn_xx")):
        _cuda(t, dt, n)
        _check(t.numel() == B * C, f"{n} must be [B, C] = [{B}, {C}]")
    return L, C, F, keep


def _layer_call(L, C, F, x_inout, att_xx, aa, bb, pp, ffn_xx, ws, ws_bytes):
    B, T, _ = x_inout.shape
    _lib.call("kr_layer_step", L, C, F, x_inout.data_ptr(), B, T, att_xx.data_ptr(),
              aa.data_ptr(), bb.data_ptr(), pp.data_ptr(), ffn_xx.data_ptr(), ws.data_ptr(),
              ws_bytes, _lib.stream_ptr())


def rwkv4_layer_step_cpp(x, att_xx, aa, bb, pp, ffn_xx, ln1_w, ln1_b, tm_k, tm_v, tm_r,
                         time_decay, time_first, Kw, Vw, Rw, Ow, ln2_w, ln2_b, ffn_tm_k,
                         ffn_tm_r, ffn_Kw, ffn_Vw, ffn_Rw):
    """One RWKV-4 layer over x [B, T, C] fp16 (any B, T); state mutated in
    place; returns the new x (layer_cpp.cpp:456-637). `time_decay` is
    w = -exp(raw) as the reference's rwkv loader passes it (wkv_kernel.cu:41-45).
    Matrices are [in, out] (y = x @ W); the first call on a weight makes a
    transposed and a fragment-packed copy of it, which live as long as the
    tensor (4 bytes per parameter) and are remade after an in-place change."""
    args = (x, att_xx, aa, bb, pp, ffn_xx, ln1_w, ln1_b, tm_k, tm_v, tm_r, time_decay,
            time_first, Kw, Vw, Rw, Ow, ln2_w, ln2_b, ffn_tm_k, ffn_tm_r, ffn_Kw, ffn_Vw, ffn_Rw)
    L, C, F, _keep = _layer_struct(*args)
    B, T, _ = x.shape
    out = x.contiguous().clone()
    ws_bytes = _lib.lib().kr_forward_workspace_bytes(B * T, C, F)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x.device)
    _layer_call(L, C, F, out, att_xx, aa, bb, pp, ffn_xx, ws, ws_bytes)
    return out


def rwkv4_layer_step_cpp_t1(x, att_xx, aa, bb, pp, ffn_xx, *weights):
    """The B = 1, T = 1 form of rwkv4_layer_step_cpp (layer_cpp.cpp:294-443):
    x [1, 1, C], state tensors [1, C]. Same kernels and bits as the general
    op at that shape (the decode step's)."""
    _check(x.dim() == 3 and x.shape[0] == 1 and x.shape[1] == 1, "x must be [1, 1, C]")
    return rwkv4_layer_step_cpp(x, att_xx, aa, bb, pp, ffn_xx, *weights)


_LAYER_GRAPHS: dict = {}


def rwkv4_layer_step_cpp_graphed(layer_id, x_buf, x_out_buf, att_xx, aa, bb, pp, ffn_xx,
                                 *weights):
    """Graph-replayed rwkv4_layer_step_cpp (layer_cpp.cpp:654-717):
    x_out_buf = layer(x_buf) with the state mutated in place; returns
    x_out_buf. The first call for a (layer_id, T, buffers) key captures the
    layer step into a HIP graph, later calls replay it, so the buffers must
    stay allocated and keep their addresses (as in the reference). Capturing
    executes nothing here, so every call - the first included - advances the
    state exactly once; the reference's warm-up runs and capture advance it
    three times on the first call (cpp_path.py:369-384 records that as a bug).
    The graph also keys on the buffer addresses and shapes, so new buffers get
    a new graph instead of a stale replay. The graph runs on the weight copies
    (transposed, fragment-packed) made at capture time: after an in-place change of a
    weight tensor (same address), call clear_layer_graph_cache()."""
    _cuda(x_buf, torch.float16, "x_buf")
    _cuda(x_out_buf, torch.float16, "x_out_buf")
    _check(x_buf.shape == x_out_buf.shape, "x_buf and x_out_buf must have the same shape")
    bufs = (x_buf, x_out_buf, att_xx, aa, bb, pp, ffn_xx)
    key = (int(layer_id), tuple((t.data_ptr(), tuple(t.shape)) for t in bufs),
           tuple((w.data_ptr(), tuple(w.shape)) for w in weights))
    hit = _LAYER_GRAPHS.get(key)
    if hit is None:
        L, C, F, keep = _layer_struct(x_buf, att_xx, aa, bb, pp, ffn_xx, *weights)
        B, T, _ = x_buf.shape
        ws_bytes = _lib.lib().kr_forward_workspace_bytes(B * T, C, F)
        ws = torch.empty(ws_bytes, dtype=torch.uint8, device=x_buf.device)
        torch.cuda.synchronize(x_buf.device)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x_out_buf.copy_(x_buf)
            _layer_call(L, C, F, x_out_buf, att_xx, aa, bb, pp, ffn_xx, ws, ws_bytes)
        hit = (graph, L, keep, ws)
        _LAYER_GRAPHS[key] = hit
    hit[0].replay()
    return x_out_buf


def clear_layer_graph_cache():
    """Drop every cached layer graph (layer_cpp.cpp:719-722); call when
    weights change or before freeing the buffers a graph was captured on."""
    _LAYER_GRAPHS.clear()


# ---------------------------------------------------------------------------
# phase profiler (layer_cpp.cpp:111-157, read/reset at :825-836)
# ---------------------------------------------------------------------------

def set_phase_profile(on: bool) -> bool:
    """Turn the per-call layer profiler on or off (KRUNCH_PHASE_PROFILE=1 does
    it at first use); returns the previous setting."""
    return bool(_lib.lib().kr_phase_profile(1 if on else 0))


def read_phase_times() -> dict:
    """Accumulated milliseconds per layer phase over the profiled
    rwkv4_layer_step_cpp calls, plus "call_count". This build's phases:
    ln1_mix, kvr_matmul, wkv, ow_matmul_residual, ln2_mix, ffn_rk_matmul,
    ffn_v_matmul_residual (the reference's eleven, grouped as its fused
    kernels run them; a phase absorbed by a fused launch reads 0)."""
    import ctypes
    L = _lib.lib()
    n = L.kr_phase_count()
    ms = (ctypes.c_double * n)()
    calls = ctypes.c_longlong(0)
    _lib.call("kr_read_phase_times", ms, n, ctypes.byref(calls))
    out = {L.kr_phase_name(i).decode(): float(ms[i]) for i in range(n)}
    out["call_count"] = int(calls.value)
    return out


def reset_phase_times():
    _lib.call("kr_reset_phase_times")
