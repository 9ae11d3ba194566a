"""The device code of the built library, read back: registers saved or loaded while their lanes are off.

hipcc 7.2 has put the saving of registers into accumulation registers, and could put the loading back of some, at
the start of the block that a lane-switching branch jumps to, before the instruction that switches the lanes on again.
Where the branch is taken no lane is on, so nothing is saved, and what is loaded back later is garbage: addresses
among it.  No source line is wrong then, and a test of results finds it only by running it; the code shows it."""
import glob
import os
import re
import shutil
import subprocess

import pytest

from polar_pack_amd import _native as nat
from polar_pack_amd.build import hipcc

OBJDUMP = os.path.join(os.path.dirname(os.path.realpath(hipcc())), "..", "lib", "llvm", "bin", "llvm-objdump")
TARGET = re.compile(r"// ([0-9A-F]+):.*<.*\+0x([0-9a-f]+)>")
FINE = ("v_readlane", "v_writelane", "v_readfirstlane", "v_cmp", "v_nop")     # whatever lanes are on


def objdump():
    for p in (OBJDUMP, "/opt/rocm/llvm/bin/llvm-objdump", shutil.which("llvm-objdump")):
        if p and os.path.exists(p):
            return p
    pytest.skip("no llvm-objdump")


def joins(code):
    """Vector instructions between where a branch with all its lanes off lands and where they are switched on:
    [(address, instructions)] of one function's ``code``, a list of (address, text, line)."""
    at = {a: i for i, (a, _, _) in enumerate(code)}
    first, bad = code[0][0], []
    for i, (_, text, line) in enumerate(code):
        if not text.startswith("s_cbranch_execz"):
            continue
        before = [t for _, t, _ in code[max(i - 4, 0):i]]
        if not any("saveexec" in t or t.startswith("s_xor_b64") and ", exec, " in t or t.startswith("s_andn2_b64 exec")
                   for t in before):
            continue                                     # a uniform branch of the compiler's
        m = TARGET.search(line)
        k, seen = at.get(first + int(m[2], 16) if m else None), []
        while k is not None and k < len(code):
            t = code[k][1]
            if re.match(r"s_(or|mov)_b64 exec,|s_\w+_saveexec_b64", t):
                if seen:
                    bad.append((hex(code[k][0]), seen))
                break
            if t.startswith(("s_cbranch", "s_branch", "s_endpgm", "s_setpc")):
                break
            if re.match(r"v_|ds_|global_|scratch_|buffer_|flat_", t) and not t.startswith(FINE):
                seen.append(t)
            k += 1
    return bad


def functions(text):
    """(name, code) of a disassembly, its lines read one after another."""
    name, code = None, []
    for line in text:
        if line.startswith("\t"):
            body, _, rest = line.partition("//")
            if not rest:
                continue
            code.append((int(rest.split(":")[0], 16), " ".join(body.split()), line))
        elif line.endswith(">:\n"):
            if code:
                yield name, code
            name, code = line.split("<")[1][:-3], []
    if code:
        yield name, code


def test_what_is_looked_for():
    def code(*texts):
        return [(4 * i, t, f"\t{t} // {4 * i:012X}: 00000000 " + (f"<f+0x{4 * to:x}>" if to else ""))
                for i, (t, to) in enumerate(x if isinstance(x, tuple) else (x, 0) for x in texts)]
    start = ["s_and_saveexec_b64 s[0:1], vcc", ("s_cbranch_execz 1", 3), "global_load_dword v1, v[2:3], off"]
    assert not joins(code(*start, "s_or_b64 exec, exec, s[0:1]", "v_accvgpr_write_b32 a0, v0"))
    found = joins(code(*start, "v_accvgpr_write_b32 a0, v0", "s_nop 0", "s_or_b64 exec, exec, s[0:1]"))
    assert found == [("0x14", ["v_accvgpr_write_b32 a0, v0"])]
    assert not joins(code(*start, "v_writelane_b32 v9, s3, 1", "s_or_b64 exec, exec, s[0:1]"))


def test_no_register_is_saved_with_its_lanes_off(tmp_path):
    lib, tool = nat.lib_path(), objdump()
    assert os.path.exists(lib), "build the library first"
    copy = shutil.copy(lib, tmp_path / "lib.so")
    subprocess.run([tool, "--offloading", str(copy)], cwd=tmp_path, check=True, capture_output=True, timeout=120)
    objects = glob.glob(str(tmp_path / "*gfx950*"))
    assert objects
    kernels, bad = 0, []
    for path in objects:
        p = subprocess.Popen([tool, "-d", path], stdout=subprocess.PIPE, text=True)
        for name, code in functions(p.stdout):
            kernels += 1
            bad += [(name, *b) for b in joins(code)]
        assert p.wait() == 0
    assert kernels > 100
    assert not bad, "\n".join(f"{n} at {a}: {len(t)} such as {t[0]}" for n, a, t in bad)
