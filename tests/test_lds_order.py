"""Orders of LDS accesses that a run seldom shows to be wrong, from the sources (CPU only)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "krunch_amd", "csrc")


def test_a_join_step_that_ends_early_leaves_lds_alone():
    """A step of delta_join_kernel that returns before its barrier, as one without tokens
    does, has not written the column's buffer, which a slower wave may still read from the
    step two before."""
    text = open(os.path.join(CSRC, "kr_delta.hip")).read()
    step = text[text.index("auto take = [&]"):]
    step = step[:step.index("\n    };")]
    early, barrier = step.index("if (!tokens) return;"), step.index("__syncthreads()")
    writes = [x.strip() for x in step[:barrier].split("\n") if re.search(r"\(col \+|S\[i & 1\]\s*\[", x)]
    assert early < barrier and writes
    assert all(x.startswith("if (tokens) ") for x in writes)


def test_a_split_without_steps_copies_nothing():
    """The loop over a split's steps is what waits for its copies: the first one is issued
    only where a step follows, or a workgroup ends with copies to its LDS on the way."""
    text = open(os.path.join(CSRC, "kr_headloss.hip")).read()
    body = text[text.index("void product_tile("):text.index("grad_products_kernel(")]
    first = [x.strip() for x in body.split("\n") if "issue(n_first, ks0, 0)" in x]
    assert first == ["if (ks0 < ks1) issue(n_first, ks0, 0);"]
