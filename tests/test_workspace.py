"""The layer kernels' scratch is each call's own (the same on the GPU, with two
streams and two threads: test_gpu_score_streams.py)."""
from types import SimpleNamespace

import torch

from krunch_amd import cpp_path


def test_two_calls_share_no_scratch():
    W = {"prepared": SimpleNamespace(C=256, F=512, device=torch.device("cpu"))}
    held = [cpp_path.workspace(W, M) for M in (16, 16, 500, 64)]
    spans = sorted((ws.data_ptr(), ws.data_ptr() + n) for ws, n in held)
    assert all(ws.numel() >= n > 0 for ws, n in held)
    assert all(a[1] <= b[0] for a, b in zip(spans, spans[1:]))
