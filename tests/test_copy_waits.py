"""A register that a lane read wrote needs five wait states before a memory instruction takes its address from it; the compiler
inserts them where it sees the instruction, not inside the copies of stage.h, which therefore bring their own."""
import os
import re
import subprocess

import pytest

from gvirt_amd.build import FLAGS

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
PROGRAM = r"""
#include "stage.h"
using namespace xlite;
template <bool ONCE>
__device__ void copy(const uint32_t *where, uint32_t lds)
{
    // a base straight out of lane reads
    const uint32_t lo = __builtin_amdgcn_readfirstlane(where[threadIdx.x]), hi = __builtin_amdgcn_readfirstlane(where[threadIdx.x + 64]);
    const void *base = reinterpret_cast<const void *>(static_cast<uint64_t>(hi) << 32 | lo);
    if (ONCE) {
        stage::copy_1k_once(lds, threadIdx.x * 16, base);
    } else {
        stage::copy_1k(lds, threadIdx.x * 16, base);
    }
}
__global__ void kernel(const uint32_t *where)
{
    extern __shared__ unsigned char smem[];
    copy<false>(where, stage::lds_address(smem));
    copy<true>(where + 128, stage::lds_address(smem) + 1024);
    stage::wait<0>();
}
"""


@pytest.mark.skipif(not os.path.exists(HIPCC), reason="no hipcc")
def test_copies_wait_for_their_base(tmp_path):
    source = tmp_path / "copies.hip"
    source.write_text(PROGRAM)
    text = subprocess.run([HIPCC] + FLAGS + ["--offload-device-only", "-S", "-I",
                           os.path.join(ROOT, "gvirt_amd", "csrc"), str(source), "-o", "-"], capture_output=True, text=True, check=True).stdout
    waited, since, copies = {}, 0, 0
    for line in text.splitlines():
        m = re.match(r"\s+([a-z]\w+)\s*(.*?)(?:\s*;.*)?$", line)
        if not m or line.lstrip().startswith("."):
            continue
        op, args = m.groups()
        if op.startswith("global_load_lds"):
            first, last = (int(x) for x in re.search(r"s\[(\d+):(\d+)\]", args).groups())
            copies += 1
            for r in range(first, last + 1):
                assert since - waited.get(r, -9) >= 5, line
        since += int(args) + 1 if op == "s_nop" else 1
        if op.startswith(("v_readfirstlane", "v_readlane")):
            waited[int(re.match(r"s(\d+)", args).group(1))] = since
        elif op.startswith("s_") and re.match(r"s(\[\d+:)?(\d+)", args):
            a, b = re.match(r"s\[?(\d+)(?::(\d+))?", args).groups()
            for r in range(int(a), int(b or a) + 1):
                waited.pop(r, None)
    assert copies == 2
