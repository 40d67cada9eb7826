"""The asynchronous copies to LDS in assembly: what the compiler would pad between
instructions, it does not pad inside an asm block (CPU only, from the sources)."""
import os
import re
import subprocess

from krunch_amd import build

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


def test_a_base_from_a_lane_waits_before_a_copy_reads_it(tmp_path):
    """An address that v_readfirstlane puts into scalar registers is read by a copy
    five wait states later."""
    src = tmp_path / "copy.hip"
    src.write_text("""
#include "kr_copy.h"
__global__ void copy(const char* const* bases, unsigned off, unsigned lds, int* out) {
    __shared__ int to[1024];
    out[0] = (int)(uintptr_t)(__attribute__((address_space(3))) int*)to;
    const uint64_t v = (uint64_t)bases[threadIdx.x];
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32));
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
    kr_copy16(reinterpret_cast<const char*>((uint64_t)hi << 32 | lo), off, lds);
}
""")
    out = tmp_path / "copy.s"
    subprocess.run([build.HIPCC, *build.FLAGS, "-w", "-S", "--offload-device-only", str(src), "-o", str(out)], check=True)
    lines = [x.split(";")[0].strip() for x in open(out)]
    lines = [x for x in lines if x and x[0] not in ".#" and not x.endswith(":")]
    at = next(i for i, x in enumerate(lines) if x.startswith("global_load_lds"))
    lo, hi = (int(x) for x in re.search(r"s\[(\d+):(\d+)\]", lines[at]).groups())
    waited = 0
    for x in reversed(lines[:at]):
        if re.match(r"v_readfirstlane_b32 s(%d|%d)," % (lo, hi), x):
            break
        nop = re.match(r"s_nop (\d+)", x)
        waited += 1 + int(nop.group(1)) if nop else 1
    else:
        raise AssertionError("no address from a lane in\n" + "\n".join(lines))
    assert waited >= 5, lines[:at + 1]
