"""`estimate` on the command line, with a stand-in engine, and the coder's cost of
a probability (the real engine runs in test_gpu_score_path.py)."""
import json

import numpy as np

from krunch_amd import cli
from krunch_amd.inference import coder_bits
from oracle import cdf as ocdf


class _Fake:
    def estimate(self, raw):
        return 37 + len(raw) // 4


def test_estimate_writes_one_json_line(tmp_path, capsysbinary):
    src, out = tmp_path / "a", tmp_path / "o"
    src.write_bytes(b"x" * 100)
    calls = []
    load = lambda *a: calls.append(a) or _Fake()
    assert cli.main(["estimate", "--in", str(src), "--out", str(out), "--w8a8", "--weights", "/w"], load) == 0
    assert json.loads(out.read_text()) == {"bytes": 100, "estimate": 62, "ratio": 0.62}
    assert calls[0][0] == "/w" and calls[0][2] is True
    src.write_bytes(b"")
    assert cli.main(["estimate", "--in", str(src)], load) == 0
    assert json.loads(capsysbinary.readouterr().out) == {"bytes": 0, "estimate": 37, "ratio": 0.0}


def test_coder_bits_are_the_counts_of_the_cdf():
    """Against the CDF's own counts: equal up to the counts' float32 rounding
    (one count), for every token but the row's most likely, which has the rest."""
    rng = np.random.default_rng(5)
    V = 50277
    x = rng.normal(size=(4, V)) * 4
    p = np.exp(x) / np.exp(x).sum(1, keepdims=True)
    counts = np.diff(ocdf.probs_to_cdf(p.astype(np.float32)).astype(np.int64), axis=1)
    for row, c in zip(p, counts):
        for t in [*rng.integers(0, V, 200), int(row.argmin())]:
            if t == row.argmax():
                continue
            want = 24 - np.log2(c[t])
            got = coder_bits(np.log(row[t:t + 1]), V)
            # p is rounded to float32 and its row sum again: 2^-22 of the count, and
            # the floor may then fall on the other side: one count
            tol = (1 + 2.0 ** -22 * c[t]) / c[t] * 1.4427 * 1.05 + 1e-9 if c[t] > 1 else 1.0
            assert abs(got - want) <= tol
    assert coder_bits(np.array([-np.inf, 0.0]), 256) == 24.0 + (24 - np.log2((1 << 24) - 256 + 1))
