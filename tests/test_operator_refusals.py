"""What the scores, 4-bit products and WKV-with-heads entry points refuse, without a
device: return codes and messages of the C ABI (no launch is reached), device checks
of the Python operators, and their size queries."""
import ctypes

import pytest
import torch

from krunch_amd import _lib, krunch_ac_hip as ops

L = _lib.lib()
BUF = torch.zeros(1 << 14, dtype=torch.uint8)
PTR = (BUF.data_ptr() + 255) // 256 * 256


def refused(rc, text):
    assert rc < 0
    assert text in L.kr_last_error().decode(), L.kr_last_error()


def scores(logits=PTR, f32=0, N=2, V=10, ld=10, tokens=PTR, lp=PTR, h=PTR, top=0, tl=None, tt=None):
    return L.kr_token_scores(logits, f32, N, V, ld, tokens, lp, h, top, tl, tt, None)


def test_token_scores():
    assert scores(N=0) == 0 and scores(N=0, logits=None) == 0
    refused(scores(N=-1), "N=-1")
    refused(scores(N=(1 << 24) + 1), "N=16777217")
    refused(scores(V=0), "V=0")
    refused(scores(V=(1 << 30) + 1, ld=1 << 31), "V=1073741825")
    refused(scores(ld=9), "ld=9")
    refused(scores(top=-1), "n_top=-1")
    refused(scores(V=100, ld=100, top=33), "n_top=33")
    refused(scores(V=4, top=5), "n_top=5")
    refused(scores(top=2), "null top")
    refused(scores(top=2, tl=PTR), "null top")
    for name in ("logits", "tokens", "lp", "h"):
        refused(scores(**{name: None}), "null")
    refused(scores(logits=PTR + 1), "misaligned")
    refused(scores(logits=PTR + 2, f32=1), "misaligned")


def w4(x=PTR, ldx=64, M=2, K=64, q=PTR, s=PTR, group=64, N=8, out=PTR, ldo=8, ep=1, res=None, gate=None):
    return L.kr_det_matmul_w4(x, ldx, M, K, q, s, group, N, out, ldo, ep, res, gate, None)


def test_products():
    assert w4(M=0) == 0
    for kw, text in (({"K": 48, "ldx": 48}, "K=48"), ({"K": 0}, "K=0"), ({"N": 0}, "N=0"), ({"M": -1}, "M=-1"),
                     ({"K": (1 << 20) + 32, "ldx": 1 << 21}, "K=1048608"),
                     ({"M": 1 << 20}, "M=1048576"), ({"group": 16}, "group=16"), ({"group": 0}, "group=0"),
                     ({"ldx": 56}, "ldx=56"), ({"ldx": 68}, "ldx=68"), ({"ldo": 7}, "ldo=7"), ({"ep": 6}, "epilogue"),
                     ({"ep": -1}, "epilogue"), ({"ep": 4}, "needs res"), ({"ep": 5, "res": PTR}, "needs gate"),
                     ({"x": None}, "null"), ({"q": None}, "null"), ({"s": None}, "null"), ({"out": None}, "null"),
                     ({"x": PTR + 8}, "misaligned"), ({"q": PTR + 4}, "misaligned"), ({"s": PTR + 2}, "misaligned")):
        refused(w4(**kw), text)


def test_quantize_and_its_size():
    def quant(W=PTR, ldk=8, ldn=1, N=8, K=64, group=64, q=PTR, s=PTR):
        return L.kr_quantize_w4(W, ldk, ldn, N, K, group, q, s, None)
    for kw, text in (({"K": 40}, "K=40"), ({"N": 0}, "N=0"), ({"group": 48}, "group=48"), ({"ldk": 0}, "strides"),
                     ({"ldn": 0}, "strides"), ({"W": None}, "null"), ({"q": None}, "null"), ({"s": None}, "null"),
                     ({"q": PTR + 8}, "misaligned"), ({"W": PTR + 1}, "misaligned")):
        refused(quant(**kw), text)
    assert L.kr_w4_bytes(1, 32) == 1024 and L.kr_w4_bytes(17, 129 - 1 + 32) == 2 * 2 * 1024
    assert L.kr_w4_bytes(50277, 768) == 3143 * 6 * 1024
    assert L.kr_w4_bytes(0, 32) == 0 and L.kr_w4_bytes(8, 33) == 0


def heads(B=1, T=2, H=2, D=64, r=PTR, ldr=128, k=PTR, ldk=128, v=PTR, ldv=128, w=PTR, u=PTR, lens=None, S=PTR,
          y=PTR, ldy=128, chunked=1, ws=None, nbytes=0):
    return L.kr_wkv_heads(B, T, H, D, r, ldr, k, ldk, v, ldv, w, u, lens, S, y, ldy, chunked, ws, nbytes, None)


def test_wkv_heads():
    assert heads(B=0) == 0 and heads(T=0) == 0
    for kw, text in (({"D": 32}, "D=32"), ({"D": 96}, "D=96"), ({"H": 0}, "H=0"), ({"B": -1}, "B=-1"),
                     ({"T": -1}, "T=-1"), ({"ldr": 120}, "strides"), ({"ldk": 132}, "strides"),
                     ({"ldv": 0}, "strides"), ({"ldy": 127}, "strides"), ({"r": None}, "null"), ({"k": None}, "null"),
                     ({"v": None}, "null"), ({"w": None}, "null"), ({"u": None}, "null"), ({"S": None}, "null"),
                     ({"y": None}, "null"), ({"r": PTR + 8}, "aligned"), ({"S": PTR + 8}, "aligned"),
                     ({"y": PTR + 2}, "aligned")):
        refused(heads(**kw), text)
    need = L.kr_wkv_heads_workspace_bytes(1, 1000, 2, 64)
    assert need % (2 * 64 * 64 * 4) == 0 and need > 0
    refused(heads(T=1000), "workspace")
    refused(heads(T=1000, ws=PTR, nbytes=need - 1), "workspace")
    refused(heads(T=1000, ws=PTR + 8, nbytes=need), "workspace")
    # single tokens and calls that fill the GPU need none
    for shape in ((1, 1, 12, 64), (512, 1, 12, 64), (1, 8, 12, 64), (100, 1000, 12, 64), (0, 9, 1, 64)):
        assert L.kr_wkv_heads_workspace_bytes(*shape) == 0
    assert L.kr_wkv_heads_workspace_bytes(1, 1000, 2, 65) == 0


def test_python_operators_take_device_tensors_only():
    h = torch.zeros(4, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="device"):
        ops.token_scores(h, torch.zeros(4, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="device"):
        ops.quantize_w4(h)
    with pytest.raises(RuntimeError, match="device"):
        ops.det_matmul_w4(h, ops.W4(torch.zeros(1), torch.zeros(1), 64, 8))
    x = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="device"):
        ops.wkv_heads(x, x, x, torch.zeros(1), torch.zeros(1), torch.zeros(1, 1, 64, 64))


def test_the_launch_goes_to_the_tensors_device(monkeypatch):
    """With another device current, the operators run with the tensors' one current."""
    seen = []

    class _Device:
        def __init__(self, d):
            seen.append(d)

        def __enter__(self):
            seen.append("in")

        def __exit__(self, *a):
            seen.append("out")

    monkeypatch.setattr(torch.cuda, "device", _Device)
    t = torch.zeros(3)
    assert ops._on_device_of(t, lambda a, b: seen.append("run") or a + b, 1, 2) == 3
    assert seen == [t.device, "in", "run", "out"]
    monkeypatch.setattr(_lib, "_get_device", lambda: 1)
    assert ops._elsewhere(t)             # a host tensor's index is -1
    monkeypatch.setattr(_lib, "_get_device", lambda: -1)
    assert not ops._elsewhere(t)
