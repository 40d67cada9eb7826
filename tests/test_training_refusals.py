"""What the head's loss, the gated delta rule and their gradients refuse, without a device:
return codes and messages of the C ABI (no launch is reached), device checks of the
Python operators, and the size queries."""
import ctypes

import pytest
import torch

from krunch_amd import _lib, krunch_ac_hip as ops

L = _lib.lib()
BUF = torch.zeros(1 << 14, dtype=torch.uint8)
PTR = (BUF.data_ptr() + 255) // 256 * 256
MORE = 1 << 50


def refused(rc, text):
    assert rc < 0
    assert text in L.kr_last_error().decode(), L.kr_last_error()


def loss(x=PTR, ldx=128, N=2, C=128, W=PTR, ldw=128, V=10, t=PTR, loss=PTR, lse=PTR, ws=PTR, nbytes=MORE):
    return L.kr_head_loss(x, ldx, N, C, W, ldw, V, t, loss, lse, ws, nbytes, None)


def grads(x=PTR, ldx=128, N=2, C=128, W=PTR, ldw=128, V=10, t=PTR, lse=PTR, g=PTR, f32=0, dx=PTR, dW=PTR, ws=PTR,
          nbytes=MORE):
    return L.kr_head_loss_backward(x, ldx, N, C, W, ldw, V, t, lse, g, f32, dx, dW, ws, nbytes, None)


SHAPES = (({"C": 96}, "C=96"), ({"C": 0}, "C=0"), ({"C": 16448, "ldx": 16448, "ldw": 16448}, "C=16448"),
          ({"V": 0}, "V=0"), ({"N": -1}, "N=-1"), ({"N": (1 << 24) + 1}, "N=16777217"),
          ({"V": (1 << 24) + 1}, "V=16777217"), ({"N": 1 << 23, "V": 1 << 22}, "2^44"), ({"ldx": 120}, "strides"),
          ({"ldw": 132}, "strides"), ({"ldx": 1 << 21}, "strides"), ({"x": None}, "null"), ({"W": None}, "null"),
          ({"t": None}, "null"), ({"lse": None}, "null"), ({"x": PTR + 8}, "aligned"), ({"W": PTR + 2}, "aligned"),
          ({"ws": None}, "workspace"), ({"ws": PTR + 16}, "workspace"), ({"nbytes": 100}, "workspace"))


@pytest.mark.parametrize("call", [loss, grads])
def test_head(call):
    for kw, text in SHAPES:
        refused(call(**kw), text)


def test_head_more():
    assert loss(N=0) == 0 and loss(N=0, x=None, ws=None) == 0
    refused(loss(loss=None), "null")
    refused(grads(N=0), "no rows")
    refused(grads(g=None), "null")
    refused(grads(dx=None, dW=None), "null")
    refused(grads(dx=PTR + 8), "aligned")
    refused(grads(dW=PTR + 4, dx=None), "aligned")
    size = L.kr_head_loss_workspace_bytes
    assert size(0, 128, 10) == 0 and size(5, 96, 10) == 0 and size(5, 128, 0) == 0 and size(1 << 23, 128, 1 << 22) == 0
    assert 0 < size(1, 768, 50277) <= 256 + 8 * 256
    # a call's parts are those of 65536 rows at most
    assert size(1 << 20, 768, 50277) == size(1 << 16, 768, 50277) <= (1 << 18) + 8 * (1 << 16) * 786
    for n in ((1 << 16) + 1, (1 << 16) + 100, (1 << 16) + 3000):      # ends with few rows have more parts a row
        assert size(n, 768, 50277) >= size(1 << 16, 768, 50277)
    refused(loss(N=300, V=1000, nbytes=size(300, 128, 1000) - 1), "workspace")
    back = L.kr_head_loss_backward_workspace_bytes
    assert back(0, 128, 10, 1, 1) == 0 and back(5, 96, 10, 1, 1) == 0
    refused(grads(N=300, V=1000, nbytes=back(300, 128, 1000, 1, 1) - 1), "workspace")
    # dz of a piece, x and partial sums, not [N, V]
    assert back(65536, 768, 50277, 1, 1) < (176 << 20) + 65536 * 768 * (2 + 4 * 64) + (1 << 20)
    assert back(8192, 768, 50277, 0, 1) < 200 << 20


def delta(B=1, T=2, H=2, D=64, q=PTR, ldq=128, k=PTR, ldk=128, v=PTR, ldv=128, a=PTR, ldg=2, b=PTR, ldb=2, lens=None,
          S=PTR, y=PTR, ldy=128, chunked=1, ws=None, nbytes=0):
    return L.kr_gated_delta(B, T, H, D, q, ldq, k, ldk, v, ldv, a, ldg, b, ldb, lens, S, y, ldy, chunked, ws, nbytes,
                            None)


def delta_grads(B=1, T=2, H=2, D=64, q=PTR, ldq=128, k=PTR, ldk=128, v=PTR, ldv=128, a=PTR, ldg=2, b=PTR, ldb=2,
                lens=None, S=PTR, y=PTR, ldy=128, dS=None, dq=PTR, dk=PTR, dv=PTR, da=PTR, db=PTR, d0=PTR, ws=PTR,
                nbytes=MORE):
    return L.kr_gated_delta_backward(B, T, H, D, q, ldq, k, ldk, v, ldv, a, ldg, b, ldb, lens, S, y, ldy, dS, dq, dk,
                                     dv, da, db, d0, ws, nbytes, None)


@pytest.mark.parametrize("call", [delta, delta_grads])
def test_gated_delta(call):
    for kw, text in (({"D": 32}, "D=32"), ({"D": 96}, "D=96"), ({"H": 0}, "H=0"), ({"B": -1}, "B=-1"),
                     ({"T": -1}, "T=-1"), ({"B": 1 << 13, "H": 1 << 12, "ldq": 1 << 18}, "B=8192"),
                     ({"ldq": 120}, "strides"), ({"ldk": 132}, "strides"), ({"ldv": 0}, "strides"),
                     ({"ldy": 127}, "strides"), ({"ldg": 1}, "log_decay"), ({"ldb": 0}, "beta"), ({"q": None}, "null"),
                     ({"k": None}, "null"), ({"v": None}, "null"), ({"a": None}, "null"), ({"b": None}, "null"),
                     ({"S": None}, "null"), ({"y": None}, "null"), ({"q": PTR + 8}, "aligned"),
                     ({"S": PTR + 8}, "aligned"), ({"y": PTR + 2}, "aligned")):
        refused(call(**kw), text)


def test_gated_delta_workspaces():
    assert delta(B=0) == 0 and delta(T=0) == 0
    size = L.kr_gated_delta_workspace_bytes
    need = size(1, 1000, 2, 64)
    assert need > 0 and need % (3 * 2 * 64 * 64 * 4) == 0
    refused(delta(T=1000), "workspace")
    refused(delta(T=1000, ws=PTR, nbytes=need - 1), "workspace")
    refused(delta(T=1000, ws=PTR + 8, nbytes=need), "workspace")
    # single tokens, one chunk and calls that fill the GPU need none
    for shape in ((1, 1, 12, 64), (512, 1, 12, 64), (1, 8, 12, 64), (1, 64, 12, 64), (128, 1024, 12, 64), (0, 9, 1, 64)):
        assert size(*shape) == 0
    assert size(1, 1000, 2, 65) == 0
    back = L.kr_gated_delta_backward_workspace_bytes
    assert back(1, 1000, 2, 65) == 0 and back(0, 5, 2, 64) == 0 and back(2, 0, 2, 64) == 0
    # states and rows of every chunk
    assert back(128, 1024, 12, 64) == 128 * 12 * 4 * 64 * (17 * 64 + 16 * 64 + 2 * 16 * 64)
    for kw, text in (({"B": 0}, "B=0"), ({"T": 0}, "T=0"), ({"T": 4194241, "B": 1}, "T=4194241"), ({"dq": None}, "null"),
                     ({"dk": None}, "null"), ({"dv": None}, "null"), ({"da": None}, "null"), ({"db": None}, "null"),
                     ({"d0": None}, "null"), ({"dS": PTR + 4}, "aligned"), ({"dq": PTR + 8}, "aligned"),
                     ({"dk": PTR + 8}, "aligned"), ({"dv": PTR + 8}, "aligned"), ({"d0": PTR + 8}, "aligned"),
                     ({"ws": None}, "workspace"), ({"ws": PTR + 16}, "workspace"), ({"nbytes": 1000}, "workspace")):
        refused(delta_grads(**kw), text)


def test_python_operators_take_device_tensors_only():
    x, W = torch.zeros(4, 64, dtype=torch.float16), torch.zeros(9, 64, dtype=torch.float16)
    t, f = torch.zeros(4, dtype=torch.int32), torch.zeros(4)
    with pytest.raises(RuntimeError, match="device"):
        ops.head_loss(x, W, t)
    with pytest.raises(RuntimeError, match="device"):
        ops.head_loss_backward(x, W, t, f, f)
    for bad in (torch.zeros(9, 60, dtype=torch.float16), torch.zeros(64, dtype=torch.float16), W[:0]):
        with pytest.raises(RuntimeError, match="W must be"):
            ops.head_loss(x, bad, t)
    q = torch.zeros(1, 2, 1, 64, dtype=torch.float16)
    g, S = torch.zeros(1, 2, 1), torch.zeros(1, 1, 64, 64)
    with pytest.raises(RuntimeError, match="device"):
        ops.gated_delta(q, q, q, g, g, S)
    with pytest.raises(RuntimeError, match="device"):
        ops.gated_delta_backward(q, q, q, g, g, S, q)
    for bad, text in ((q[0], "B, T, H, D"), (torch.zeros(1, 2, 1, 96, dtype=torch.float16), "64 or 128")):
        with pytest.raises(RuntimeError, match=text):
            ops.gated_delta(bad, bad, bad, g, g, S)


class _Meta(torch.Tensor):
    """A host tensor that says it is on the device: the checks behind that one."""
    @property
    def is_cuda(self):
        return True


def _on(t):
    return t.as_subclass(_Meta)


def test_python_checks_of_shapes_types_and_strides():
    x, W = (_on(torch.zeros(n, 128, dtype=torch.float16)) for n in (4, 9))
    t, f = _on(torch.zeros(4, dtype=torch.int32)), _on(torch.zeros(4))
    for args, text in (((x.float(), W, t), "float16"), ((x[:, ::2], W, t), "columns"), ((x, W, t.long()), "int32"),
                       ((x, W, t[:3]), r"\[N\]"), ((x.t(), W, t), "columns"),
                       ((_on(torch.zeros(128, 4, dtype=torch.float16)).t(), W, t), "contiguous"),
                       ((_on(torch.zeros(4, 132, dtype=torch.float16))[:, :128], W, t), "contiguous"),
                       ((x[:1].expand(4, 128), W, t), "contiguous")):
        with pytest.raises(RuntimeError, match=text):
            ops.head_loss(*args)
    for args, text in (((x, W, t, f.double(), f), "lse"), ((x, W, t, f, f[:2]), "dloss"),
                       ((x, W, t, f, f, torch.float64), "out_dtype")):
        with pytest.raises(RuntimeError, match=text):
            ops.head_loss_backward(*args)
    q = _on(torch.zeros(2, 3, 2, 64, dtype=torch.float16))
    g, S = _on(torch.zeros(2, 3, 2)), _on(torch.zeros(2, 2, 64, 64))
    ok = [q, q, q, g, g, S]
    for at, bad, text in ((1, q[:1], "k must be"), (2, q.float(), "v must be a float16"), (0, q.transpose(1, 2).contiguous().transpose(1, 2), "q: heads"),
                          (3, g.half(), "log_decay"), (4, g[:, :2], "beta"), (3, g.transpose(1, 2).contiguous().transpose(1, 2), "log_decay: heads"),
                          (5, S[:1], "state"), (5, S.double(), "state"), (5, S.transpose(2, 3), "state")):
        args = list(ok)
        args[at] = bad
        with pytest.raises(RuntimeError, match=text):
            ops.gated_delta(*args)
    for lens in (_on(torch.zeros(3, dtype=torch.int32)), _on(torch.zeros(2, dtype=torch.int64))):
        with pytest.raises(RuntimeError, match="lens"):
            ops.gated_delta(*ok, lens)
    with pytest.raises(RuntimeError, match="dy"):
        ops.gated_delta_backward(*ok, q[:1])
    with pytest.raises(RuntimeError, match="dstate"):
        ops.gated_delta_backward(*ok, q, S[:, :1])


def test_the_bindings_take_what_the_header_declares():
    """Argument counts of the new entry points, as the header has them."""
    import os
    import re
    text = open(os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "krunch_hip.h")).read()
    for name in ("kr_head_loss", "kr_head_loss_workspace_bytes", "kr_head_loss_backward",
                 "kr_head_loss_backward_workspace_bytes", "kr_gated_delta", "kr_gated_delta_workspace_bytes",
                 "kr_gated_delta_backward", "kr_gated_delta_backward_workspace_bytes"):
        decl = re.search(r"^(int|size_t) %s\(([^;]*)\);" % name, text, re.M | re.S)
        params = [p.strip() for p in decl.group(2).split(",")]
        types = [ctypes.c_void_p if "*" in p else ctypes.c_longlong if "long long" in p else
                 ctypes.c_size_t if "size_t" in p else ctypes.c_int for p in params]
        assert _lib._SIGS[name][0] == types, name
