"""What the compiler made of the kernels, read from the library that was built here.

Behind an `if` that only some lanes take, the lanes are brought back by one instruction, s_or_b64 exec, exec, <what the if had saved>, at
the place where both ways meet.  Whatever stands between that place and that instruction runs without the lanes that skipped the `if`.
The compiler's register allocator has put copies there when it moved values that live across the `if` to other registers: an
earlier form of the fp32 wide convolution with statistics (two sets of fragments next to the sums) moved its running sums so, and
every lane whose row lay past the tensor lost them.  No kernel may have such a place."""
import os
import re
import shutil
import subprocess

import pytest

from vision_amd import _lib

LLVM = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin")
VECTOR = re.compile(r"(v_(?!readlane|readfirstlane|writelane|cmp|nop)|scratch_|ds_|global_|flat_|buffer_)")


def narrowed(lines):
    """[(function, instructions)] of the places where lanes meet again behind vector instructions; `lines` as llvm-objdump prints them."""
    found, name, body = [], None, []

    def look():
        targets, saved = {}, None                            # where an `if` that no lane takes jumps to -> registers it saved the lanes in
        for at, text in body:
            m = re.match(r"s_(?:and|or|andn2)_saveexec_b64 (\S+),", text) or re.match(r"s_xor_b64 (\S+), exec,", text)
            if m:
                saved = m.group(1)
            m = re.match(r"s_cbranch_execz (\d+)", text)
            if m and saved:
                words = int(m.group(1))
                targets.setdefault(at + 4 + 4 * (words - 65536 if words >= 32768 else words), set()).add(saved)
        for i, (at, _) in enumerate(body):
            if at not in targets:
                continue
            seen = []
            for _, text in body[i:]:
                m = re.match(r"s_or_b64 exec, exec, (\S+)", text) or re.match(r"s_(?:andn2|or)_saveexec_b64 (\S+),", text)
                if m:
                    if m.group(1) in targets[at] and any(VECTOR.match(s) for s in seen):
                        found.append((name, seen))
                    break
                if text.startswith(("s_cbranch", "s_branch", "s_endpgm")):
                    break
                seen.append(text)

    for line in lines:
        m = re.match(r"[0-9a-f]+ <(\w+)>:", line)
        if m:
            look()
            name, body = m.group(1), []
        elif "//" in line:
            text, _, rest = line.partition("//")
            body.append((int(rest.split(":")[0], 16), text.strip()))
    look()
    return found


# 0x100 if (lanes of vcc) { 0x108 v5 += 1 }, and at 0x10c, where both ways meet, a copy of v7 in place of the lanes' return
PLANTED = """0000000000000100 <kernel>:
\ts_and_saveexec_b64 s[0:1], vcc    // 000000000100: BE8020EA
\ts_cbranch_execz 1                 // 000000000104: BF880001 <kernel+0xc>
\tv_add_u32_e32 v5, 1, v5           // 000000000108: 680A0A81
{first}
{second}
\ts_endpgm                          // 000000000114: BF810000
"""
COPY, BACK = ("\tv_mov_b32_e32 v6, v7    // %012x: 7E0C0307", "\ts_or_b64 exec, exec, s[0:1]     // %012x: 87FE007E")


def test_the_scan_sees_a_copy_before_the_lanes_are_back():
    bad = PLANTED.format(first=COPY % 0x10c, second=BACK % 0x110)
    assert narrowed(bad.splitlines()) == [("kernel", ["v_mov_b32_e32 v6, v7"])]
    assert not narrowed(PLANTED.format(first=BACK % 0x10c, second=COPY % 0x110).splitlines())


@pytest.mark.skipif(not os.path.exists(os.path.join(LLVM, "llvm-objdump")), reason="no llvm-objdump")
def test_no_kernel_moves_values_before_the_lanes_are_back(tmp_path):
    lib = str(tmp_path / "lib.so")
    shutil.copy(_lib.LIB_PATH, lib)
    objdump = os.path.join(LLVM, "llvm-objdump")
    subprocess.run([objdump, "--offloading", lib], check=True, capture_output=True)
    objects = sorted(str(p) for p in tmp_path.iterdir() if p.name.endswith("gfx950"))
    assert objects
    kernels, found = 0, []
    for path in objects:
        with subprocess.Popen([objdump, "-d", path], stdout=subprocess.PIPE, text=True) as p:
            lines = p.stdout.read().splitlines()
        assert p.returncode == 0
        kernels += sum(bool(re.match(r"[0-9a-f]+ <\w+>:", x)) for x in lines)
        found += narrowed(lines)
    assert kernels > 100 and not found, found[:5]
