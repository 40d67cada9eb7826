"""Orders of LDS accesses that a run seldom shows to be wrong, from the sources (CPU only)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "krunch_amd", "csrc")


def test_a_join_step_that_ends_early_leaves_lds_alone():
    """A step of delta_join_kernel that returns before its barrier has not written the
    column's buffer, which a slower wave may still read from the step two before."""
    text = open(os.path.join(CSRC, "kr_delta.hip")).read()
    step = text[text.index("auto take = [&]"):]
    step = step[:step.index("\n    };")]
    early, barrier = step.index("return;"), step.index("__syncthreads()")
    writes = [m.start() for m in re.finditer(r"\(col \+|S\[i & 1\]\s*\[", step)]
    assert writes and early < barrier
    assert all(w > early for w in writes)
