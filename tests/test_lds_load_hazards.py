"""Guards on the loads straight into LDS in the built device code (CPU only).

A buffer load into LDS takes its place in LDS from M0 and its buffer from four scalar
registers.  On gfx950 software has to leave wait states before it: one after a scalar write of
M0, five after a vector instruction's write (v_readlane, v_readfirstlane) of the buffer's
registers.  The compiler leaves them between its own instructions and not inside inline
assembly, where the experts' products have these loads; with a state missing a load may take
the old value, and 16 bytes land in another load's place.
"""

import os
import re
import subprocess

import pytest

from purin_amd import build as B
from tests.test_build_guards import LLVM, _code_objects, _disassemble, _need_tools

LOAD = re.compile(r"^buffer_load_\S+\s+(.*)\blds$")


def _scalars(operand):
    m = re.fullmatch(r"s\[(\d+):(\d+)\]", operand)
    if m:
        return set(range(int(m.group(1)), int(m.group(2)) + 1))
    m = re.fullmatch(r"s(\d+)", operand)
    return {int(m.group(1))} if m else set()


def _before(code, i):
    """(instruction, wait states between it and instruction i), nearest first."""
    states = 0
    for text in reversed(code[:i]):
        yield text, states
        m = re.match(r"s_nop (\d+)", text)
        states += int(m.group(1)) + 1 if m else 1
        if states > 5:
            return


def hazards(listing):
    """(loads into LDS, those with a wait state missing before them) of a disassembly."""
    code = [line.split("//")[0].strip() for line in listing.splitlines() if line[:1].isspace()]
    code = [c for c in code if c]
    loads, bad = 0, []
    for i, text in enumerate(code):
        m = LOAD.match(text)
        if not m:
            continue
        loads += 1
        buffer = set().union(*(_scalars(o.split()[0]) for o in m.group(1).split(",") if o.strip()))
        for earlier, states in _before(code, i):
            to = earlier.split(None, 1)[1].split(",")[0].strip() if " " in earlier else ""
            if to == "m0" and states < 1:
                bad.append((earlier, text))
            if earlier.startswith(("v_readlane", "v_readfirstlane")) and states < 5 \
                    and _scalars(to) & buffer:
                bad.append((earlier, text))
    return loads, bad


def test_loads_into_lds_leave_their_wait_states(tmp_path):
    _need_tools()
    if not os.path.exists(B.LIB):
        pytest.skip("libpurin_cp.so is not built")
    loads = 0
    for k, obj in enumerate(_code_objects(B.LIB)):
        if b"k_product16" not in obj:
            continue
        n, bad = hazards(_disassemble(obj, tmp_path, f"l{k}"))
        loads += n
        assert not bad, f"{len(bad)} of {n} loads, the first: {bad[0]}"
    assert loads > 0, "no load into LDS found"


SOURCE = """
#include <hip/hip_runtime.h>
typedef unsigned U4 __attribute__((ext_vector_type(4)));
extern "C" __global__ void k(U4 r, unsigned at, unsigned to, float* out) {
  extern __shared__ float lds[];
  asm volatile("s_mov_b32 m0, %0\\n\\tWAITbuffer_load_dwordx4 %1, %2, 0 offen lds"
               : : "s"(to), "v"(at), "s"(r) : "memory", "m0");
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  out[threadIdx.x] = lds[threadIdx.x];
}
"""


@pytest.mark.parametrize("wait,found", [("", 1), ("s_nop 0\\n\\t", 0)])
def test_the_guard_sees_a_missing_wait_state(tmp_path, wait, found):
    """Control: the same load with and without the state, compiled and never run."""
    _need_tools()
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    if not os.path.exists(hipcc):
        pytest.skip("hipcc not available")
    src, obj = tmp_path / "k.hip", tmp_path / "k.co"
    src.write_text(SOURCE.replace("WAIT", wait))
    subprocess.run([hipcc, "-O3", f"--offload-arch={B.ARCH}", "--offload-device-only",
                    "--no-gpu-bundle-output", str(src), "-o", str(obj)], check=True,
                   capture_output=True)
    text = subprocess.run([f"{LLVM}/llvm-objdump", "-d", "--mcpu=gfx950", str(obj)], check=True,
                          capture_output=True, text=True).stdout
    loads, bad = hazards(text)
    assert loads == 1 and len(bad) == found


def test_the_guard_sees_a_vector_write_of_the_buffer():
    listing = """
\tv_readfirstlane_b32 s9, v3                                 // 000000001900: 7E120503
\ts_mov_b32 m0, s4                                           // 000000001904: BEFC0004
\ts_nop 0                                                    // 000000001908: BF800000
\tbuffer_load_dwordx4 v1, s[8:11], 0 offen lds               // 00000000190C: E05D1000
"""
    assert len(hazards(listing)[1]) == 1
    assert len(hazards(listing.replace("s_nop 0 ", "s_nop 3 "))[1]) == 0
    assert len(hazards(listing.replace("s9,", "s7,"))[1]) == 0
