"""The built code object's kernels as instructions, for tests that follow what the compiler made of the source."""
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HSACO = os.path.join(ROOT, "helix_amd", "csrc", "_build", "helix_kernels.hsaco")
OBJDUMP = "/opt/rocm/llvm/bin/llvm-objdump"


def kernels(pattern):
    """{name: its instructions} of the kernels whose names match. An instruction is (mnemonic, operands, target), target
    the place in the list that a branch goes to, else None."""
    if not (os.path.exists(HSACO) and os.path.exists(OBJDUMP)):
        pytest.skip("needs the built code object and llvm-objdump")
    out = subprocess.run([OBJDUMP, "-d", HSACO], check=True, capture_output=True, text=True).stdout
    found = {}
    for block in re.split(r"\n(?=[0-9a-f]+ <)", out):
        name = re.match(r"[0-9a-f]+ <(\w+)>", block)
        if name and re.fullmatch(pattern, name.group(1)):
            found[name.group(1)] = instructions(block)
    return found


def instructions(text):
    lines = []
    for line in text.splitlines():
        m = re.match(r"\s+(\S+)\s*(.*?)\s*//\s*([0-9A-Fa-f]+):", line)
        if m:
            target = re.search(r"<\w+\+0x([0-9a-f]+)>", line) if m.group(1).startswith(("s_branch", "s_cbranch")) else None
            lines.append((m.group(1), m.group(2), int(m.group(3), 16), int(target.group(1), 16) if target else None))
    place = {address - lines[0][2]: i for i, (_, _, address, _) in enumerate(lines)}
    return [(name, rest, None if target is None else place[target]) for name, rest, _, target in lines]
