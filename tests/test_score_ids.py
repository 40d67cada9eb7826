"""Token ids that the scoring calls refuse, without a device (nothing is launched)."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

from krunch_amd import cpp_path
from krunch_amd.inference import InferenceEngine

V = 100
W = {"prepared": SimpleNamespace(V=V, C=256, F=512, n_layer=1, device=torch.device("cpu"))}


# below and above the range, and ids whose low 32 bits are in it
@pytest.mark.parametrize("bad", [-1, V, 2 ** 32 + 5, -2 ** 32, 2 ** 40])
def test_streams(bad):
    eng = InferenceEngine()
    eng._weights, eng._ready = W, True
    for streams in ([np.array([3, bad])], [np.array([1, 2, 3]), np.array([bad])], [[4, bad, 5]]):
        with pytest.raises(ValueError, match="token id out of range"):
            eng.score_tokens_batched(streams)


@pytest.mark.parametrize("bad", [-2, V, 2 ** 32 + 5, 2 ** 32 - 1, -2 ** 32])
def test_packed(bad):
    st = SimpleNamespace(B=1)
    good = torch.tensor([[1, 2]])
    for t in (torch.tensor([[3, bad]]), [[3, bad]]):
        with pytest.raises(ValueError, match="token id out of range"):
            cpp_path.score_packed_batched(W, t, good, st)
        with pytest.raises(ValueError, match="target id out of range"):
            cpp_path.score_packed_batched(W, good, t, st)


@pytest.mark.parametrize("dtype", [np.uint8, np.uint16, np.uint32, np.int16, np.int64])
def test_types(dtype):
    eng = InferenceEngine()
    eng._weights, eng._ready = W, True
    bad, good = np.array([[1, V]], dtype=dtype), np.array([[1, V - 1]], dtype=dtype)
    with pytest.raises(ValueError, match="token id out of range"):
        eng.score_tokens_batched([bad[0]])
    with pytest.raises(ValueError, match="token id out of range"):
        cpp_path.score_packed_batched(W, bad, good, SimpleNamespace(B=1))
    with pytest.raises(ValueError, match="target id out of range"):
        cpp_path.score_packed_batched(W, good, bad, SimpleNamespace(B=1))
