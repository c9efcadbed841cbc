"""
Wait states that the hardware does not keep by itself, in the machine code of the library as it is built. The compiler puts them in for its own
instructions and does not look into inline assembly. Of the manually inserted wait states that the CDNA 3 and 4 instruction set manuals list:

* a vector instruction writes a scalar register, a vector memory instruction reads it: 5 in between;
* a scalar instruction writes M0, a memory instruction that loads into LDS reads it: 1 in between.

`s_nop n` counts n + 1, any other instruction 1.
"""

import collections
import pathlib
import re
import shutil
import subprocess

import pytest

SCALAR_TO_MEMORY, M0_TO_LDS = 5, 1
# Vector instructions whose second operand is a scalar result too.
TWO_RESULTS = re.compile(r"v_(add|sub|subrev|addc|subb|subbrev)_co|v_(addc|subb|subbrev)_|v_mad_[iu]64|v_div_scale")
MEMORY = re.compile(r"(buffer|global|scratch|flat)_")
BRANCH = re.compile(r"s_(c?branch\S*)\s+(\S+)")


def _scalars(operand: str) -> tuple:
    if match := re.fullmatch(r"s\[(\d+):(\d+)\]", operand):
        return tuple(range(int(match[1]), int(match[2]) + 1))
    if match := re.fullmatch(r"s(\d+)", operand):
        return (int(match[1]),)
    return {"vcc": ("vcc_lo", "vcc_hi"), "vcc_lo": ("vcc_lo",), "vcc_hi": ("vcc_hi",), "m0": ("m0",)}.get(operand, ())


def violations(lines: list[str]) -> list[str]:
    """Of a disassembly, one instruction or `<label>:` a line. Ages are counted along the text and along every branch."""
    at_label: dict[str, dict] = collections.defaultdict(dict)  # smallest ages that branches bring
    found: list[str] = []
    for last_pass in (False, False, True):  # forward and backward branches, then a branch to a branch
        ages: dict = {}  # written scalar register -> wait states since then
        for line in lines:
            if label := re.search(r"<(\S+)>:$", line):
                for register, age in at_label[label[1]].items():
                    ages[register] = min(age, ages.get(register, age))
                continue
            line = line.split("//")[0].strip()
            if not line:
                continue
            name, *rest = line.split(None, 1)
            operands = [o.split()[0] for o in rest[0].split(",") if o.strip()] if rest else []
            if last_pass and MEMORY.match(name):
                for register in {r for o in operands for r in _scalars(o)}:
                    if register != "m0" and ages.get(register, SCALAR_TO_MEMORY) < SCALAR_TO_MEMORY:
                        found.append(f"{line}: {register} written {ages[register]} wait states before")
                if line.endswith(" lds") and ages.get("m0", M0_TO_LDS) < M0_TO_LDS:
                    found.append(f"{line}: M0 written {ages['m0']} wait states before")
            if branch := BRANCH.match(line):
                for register, age in ages.items():
                    known = at_label[branch[2]]
                    known[register] = min(age + 1, known.get(register, age + 1))
            states = int(operands[0], 0) + 1 if name == "s_nop" else 1
            ages = {register: age + states for register, age in ages.items() if age + states < SCALAR_TO_MEMORY}
            if name.startswith("v_"):
                results = operands[: 2 if TWO_RESULTS.match(name) else 1]
                ages.update((r, 0) for o in results for r in _scalars(o))
            elif name.startswith("s_") and operands and operands[0] == "m0":
                ages["m0"] = 0
    return found


def test_what_counts():
    scalar = "v_readlane_b32 s15, v215, 0"
    assert violations([scalar, "s_add_i32 m0, s8, 0x1800", "buffer_load_dwordx4 v31, s[12:15], s92 offen lds"]) == [
        "buffer_load_dwordx4 v31, s[12:15], s92 offen lds: 15 written 1 wait states before",
        "buffer_load_dwordx4 v31, s[12:15], s92 offen lds: M0 written 0 wait states before",
    ]
    assert not violations([scalar, "s_add_i32 m0, s8, 0x1800", "s_nop 3", "buffer_load_dwordx4 v31, s[12:15], s92 offen lds"])
    assert len(violations([scalar, "s_nop 3 // 0000: BF80", "global_load_dword v0, v1, s[14:15]"])) == 1
    assert not violations([scalar, "s_nop 4", "global_load_dword v0, v1, s[14:15]"])
    assert len(violations(["0000 <L0>:", "buffer_load_dword v0, v1, s[0:3], 0 offen", "v_cmp_eq_u32_e64 s[2:3], v0, v1", "s_cbranch_scc1 L0"])) == 2
    assert len(violations([scalar, "s_branch L1", "s_nop 7", "0000 <L1>:", "buffer_load_dword v0, v1, s[12:15], 0 offen"])) == 1
    assert not violations(["s_mov_b32 s15, 0", "buffer_load_dword v0, v1, s[12:15], 0 offen", "s_mov_b32 m0, s1", "ds_read_b32 v0, v1"])


def test_library_keeps_its_wait_states(library, tmp_path):
    from fast_llm_amd import _lib
    from fast_llm_amd.build import _hipcc

    objdump = pathlib.Path(_hipcc()).resolve().parent.parent / "lib" / "llvm" / "bin" / "llvm-objdump"
    objdump = objdump if objdump.exists() else shutil.which("llvm-objdump") or pytest.skip("no disassembler")
    copy = shutil.copy(_lib.LIBRARY_PATH, tmp_path)
    subprocess.run([str(objdump), "--offloading", copy], check=True, capture_output=True)
    images = sorted(tmp_path.glob("*gfx950"))
    assert images
    loads_into_lds, found = 0, []
    for image in images:
        command = [str(objdump), "-d", "--no-show-raw-insn", "--symbolize-operands", str(image)]
        lines = subprocess.run(command, check=True, capture_output=True, text=True).stdout.splitlines()
        function: list[str] = []
        for line in [*lines, "0 <_Z>:"]:  # a function at a time: its labels are its own
            if re.search(r"<_Z\S*>:$", line):
                found += violations(function)
                function = []
            elif line.startswith("\t") or line.endswith(">:"):
                function.append(line)
                loads_into_lds += line.split("//")[0].rstrip().endswith(" lds")
    assert loads_into_lds > 1000  # the disassembly is that of the library's products
    assert not found, f"{len(found)}, among them {sorted(set(found))[:8]}"
