"""Scores of texts beside other calls of the model: on two streams, from two
threads, and beside compress, each with the bits of the call by itself."""
import threading

import pytest
import torch

from krunch_amd import cpp_path, synthetic
from krunch_amd.inference import InferenceEngine

pytestmark = pytest.mark.gpu
V = 1003


@pytest.fixture(scope="module")
def engine():
    w = synthetic.make_weights(n_layer=4, C=256, F=512, V=V, seed=3)
    yield InferenceEngine().load(w)
    cpp_path.release_weights(w)


def text(B, T, seed):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randint(0, V, (B, T), generator=g, dtype=torch.int32).cuda() for _ in range(2))


def score(W, ids, tgt):
    st = cpp_path.fresh_state_batched(W, ids.shape[0])
    out = cpp_path.score_packed_batched(W, ids, tgt, st, 3)
    return [*out, st.buf]


# sizes either way round, so that a later call needs the larger scratch
SIZES = [((20, 100), (3, 40)), ((2, 30), (30, 90))]


@pytest.mark.parametrize("sizes", SIZES)
def test_two_streams(engine, sizes):
    W = engine.weights
    texts = [text(*s, seed=i) for i, s in enumerate(sizes)]
    alone = [score(W, *t) for t in texts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sizes]
    got = [[], []]
    for _ in range(6):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(score(W, *texts[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, alone[i]))


@pytest.mark.parametrize("own_stream", [False, True])
def test_two_threads(engine, own_stream):
    """On one stream (each thread's default one) and on a stream each."""
    W = engine.weights
    texts = [text(*s, seed=i + 5) for i, s in enumerate(SIZES[0])]
    alone = [score(W, *t) for t in texts]
    torch.cuda.synchronize()
    got, failed = [[], []], []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream() if own_stream else torch.cuda.default_stream()):
                for _ in range(6):
                    got[i].append(score(W, *texts[i]))
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            failed.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
    for i in range(2):
        for one in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(one, alone[i]))


def test_beside_compress(engine):
    toks = [t.clip(max=V - 1)[:n] for t, n in zip(synthetic.zipf_tokens(4, 300, seed_base=2), (300, 200, 9, 120))]
    ref = engine.compress_tokens_batched(toks)
    ids, tgt = text(8, 120, 9)
    alone = score(engine.weights, ids, tgt)
    torch.cuda.synchronize()
    side, got = torch.cuda.Stream(), []
    for _ in range(3):
        with torch.cuda.stream(side):
            got += [score(engine.weights, ids, tgt) for _ in range(3)]
        assert engine.compress_tokens_batched(toks) == ref
    torch.cuda.synchronize()
    for one in got:
        assert all(torch.equal(a, b) for a, b in zip(one, alone))
