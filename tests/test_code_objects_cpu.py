"""The gfx950 code of the built library, disassembled: rules of the instruction set that the compiler keeps
by itself but does not see inside inline assembly."""
import os
import re
import shutil
import subprocess

import pytest

import cllm_inference_amd as C

OBJDUMP = shutil.which("llvm-objdump", path="/opt/rocm/llvm/bin:/opt/rocm/bin:" + os.environ.get("PATH", ""))
WRITES_M0 = re.compile(r"s_\w+ m0,")
LOADS_TO_LDS = re.compile(r"(global|scratch|buffer)_load_\w*lds|buffer_load_.* lds\b")


def m0_hazards(lines):
    """(kernel, instruction) of every direct-to-LDS load right behind a scalar write of M0."""
    found, kernel, wrote = [], "", False
    for line in lines:
        if line.endswith(">:"):
            kernel, wrote = line.split("<")[1][:-2], False
            continue
        text = line.split("//")[0].strip()
        if not text:
            continue
        if wrote and LOADS_TO_LDS.match(text):
            found.append((kernel, text))
        wrote = WRITES_M0.match(text) is not None
    return found


def test_the_check_itself():
    mov, load = "\ts_mov_b32 m0, s46   // 00: BEFC002E", "\tglobal_load_lds_dwordx4 v[18:19], off nt  // 04: DDF6"
    assert m0_hazards(["0000 <k>:", mov, load]) == [("k", "global_load_lds_dwordx4 v[18:19], off nt")]
    assert m0_hazards(["0000 <k>:", "\ts_add_i32 m0, s1, s2", "\tbuffer_load_dword v1, s[0:3], 0 offen lds"])
    assert not m0_hazards(["0000 <k>:", mov, "\ts_nop 0", load])
    assert not m0_hazards(["0000 <k>:", mov, "\tbuffer_load_dword v1, v2, s[0:3], 0 offen"])


@pytest.mark.skipif(OBJDUMP is None, reason="no llvm-objdump")
def test_loads_to_lds_wait_for_m0(tmp_path):
    """gfx9: a scalar write of M0 needs one wait state before a direct-to-LDS load reads it (without, the
    load may take the old M0 and write to another place in LDS)."""
    C.load_library()
    so = os.path.join(os.path.dirname(C.__file__), "libcllm_hip.so")
    copy = shutil.copy(so, tmp_path)
    subprocess.run([OBJDUMP, "--offloading", copy], cwd=tmp_path, check=True, capture_output=True)
    objects = [f for f in sorted(os.listdir(tmp_path)) if "gfx950" in f]
    assert len(objects) >= 10
    loads, found = 0, []
    for name in objects:
        out = subprocess.run([OBJDUMP, "-d", "--no-show-raw-insn", str(tmp_path / name)], check=True,
                             capture_output=True, text=True).stdout.splitlines()
        loads += sum("lds_dword" in line for line in out)
        found += m0_hazards(out)
    assert loads > 100
    assert not found, (len(found), sorted({k for k, _ in found})[:5], found[0])
