"""The asynchronous copies to LDS in assembly: what the compiler would pad between
instructions, it does not pad inside an asm block (CPU only, from the sources)."""
import os
import re

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "krunch_amd", "csrc")


def test_m0_is_written_a_wait_state_before_a_copy_takes_it():
    blocks = []
    for name in sorted(os.listdir(CSRC)):
        text = open(os.path.join(CSRC, name)).read()
        blocks += [(name, b) for b in re.findall(r'"([^"\n]*global_load_lds[^"\n]*)"', text)]
    assert blocks
    for name, block in blocks:
        lines = [x.strip() for x in block.split("\\n\\t")]
        write = next(i for i, x in enumerate(lines) if x.startswith("s_mov_b32 m0"))
        copy = next(i for i, x in enumerate(lines) if x.startswith("global_load_lds"))
        assert any(x.startswith("s_nop") for x in lines[write + 1:copy]), (name, block)
