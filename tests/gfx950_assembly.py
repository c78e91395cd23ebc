"""The assembly that the compiler writes of this repository's kernels, and which instructions may follow which how
closely. The compiler keeps the distances that the ISA asks of software, but neither inside inline assembly nor beside
it, whose instructions it does not know."""
from __future__ import annotations

import re
import subprocess
from collections import deque

from conftest import dpa_mod

_REG = re.compile(r"\b([vas])(?:(\d+)\b|\[(\d+):(\d+)\])")


def assembly_of(source: str, folder) -> str:
    build = dpa_mod("build")
    out = folder / f"{source}.s"
    subprocess.run([build.hipcc(), *build.HIPCC_FLAGS, "--offload-device-only", "-S", str(build.CSRC_DIR / f"{source}.hip"),
                    "-o", str(out)], check=True, stdout=subprocess.PIPE, stderr=subprocess.STDOUT)
    return out.read_text()


def _registers(text: str) -> set[str]:
    return {f"{m[1]}{i}" for m in _REG.finditer(text)
            for i in (range(int(m[2]), int(m[2]) + 1) if m[2] else range(int(m[3]), int(m[4]) + 1))}


class Instruction:
    def __init__(self, line: str):
        self.text = line
        self.op, _, rest = line.partition(" ")
        operands = re.split(r",\s*(?![^\[]*\])", rest.strip())
        self.matrix = self.op.startswith("v_mfma")
        self.vector = self.op.startswith("v_") and not self.matrix
        swap = self.op.startswith(("v_swap", "v_permlane16_swap", "v_permlane32_swap"))
        self.writes = _registers(" ".join(operands[:2 if swap else 1])) if self.op.startswith("v_") else set()
        self.touches = _registers(rest)
        self.writes_m0 = operands[0] == "m0"
        self.to_lds = "load" in self.op and "_lds_" in self.op
        self.states = int(operands[0]) + 1 if self.op == "s_nop" else 1
        self.target = operands[0] if self.op.startswith(("s_branch", "s_cbranch")) else None
        self.ends = self.op in ("s_branch", "s_endpgm", "s_setpc_b64")


class Kernel:
    def __init__(self, code: list[Instruction], labels: dict[str, int]):
        self.code = code
        self.next = [([] if c.ends else [i + 1]) + ([labels[c.target]] if c.target else []) for i, c in enumerate(code)]

    def behind(self, start: int, states: int) -> dict[int, int]:
        """The instructions that may come less than `states` wait states behind `start`, and after how many."""
        best: dict[int, int] = {}
        queue = deque((j, 0) for j in self.next[start])
        while queue:
            i, passed = queue.popleft()
            if i >= len(self.code) or passed >= states or best.get(i, states) <= passed:
                continue
            best[i] = passed
            queue.extend((j, passed + self.code[i].states) for j in self.next[i])
        return best

    def closer(self, states: int, first, second) -> list[str]:
        """Pairs less than `states` wait states apart: first(instruction), second(it, the one behind)"""
        return [f"{c.text} | {passed} states | {self.code[j].text}" for i, c in enumerate(self.code) if first(c)
                for j, passed in self.behind(i, states).items() if second(c, self.code[j])]


def kernels_of(assembly: str) -> dict[str, Kernel]:
    found: dict[str, Kernel] = {}
    name, code, labels = None, [], {}
    for line in assembly.splitlines():
        line = line.split(";")[0].strip()
        if m := re.match(r"(_Z\w+):", line):
            name, code, labels = m[1], [], {}
        elif m := re.match(r"(\.LBB\w+):", line):
            labels[m[1]] = len(code)
        elif line.startswith(".Lfunc_end"):
            if name and code:
                found[name] = Kernel(code, labels)
            name = None
        elif name and re.match(r"[a-z]\w+(\s|$)", line):
            code.append(Instruction(line.replace("\t", " ")))
    return found


def m0_too_close(kernel: Kernel) -> list[str]:
    """One state from a scalar write of m0 to a load to LDS, which reads it."""
    return kernel.closer(1, lambda c: c.writes_m0, lambda c, d: d.to_lds)


def products_too_close(kernel: Kernel) -> list[str]:
    """Two states from a vector instruction's result to a matrix instruction that reads it, twelve from a matrix instruction
    of eight passes to any other that touches its result."""
    return (kernel.closer(2, lambda c: c.vector and c.writes, lambda c, d: d.matrix and c.writes & d.touches)
            + kernel.closer(12, lambda c: c.matrix, lambda c, d: not d.matrix and c.writes & d.touches))
