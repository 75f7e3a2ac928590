"""Wait states in the built gfx950 code objects of libt5hip.so (no GPU needed).

A vector-memory instruction that reads a scalar register needs five wait states after the vector unit
has written it (v_readfirstlane, v_readlane, compares).  The compiler puts them in for its own
instructions, but does not look inside inline asm, where the kernels' global -> LDS copies stand: a copy
that read its descriptor too early would read a stale one, and could fetch from anywhere.
"""
import re
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
SO = ROOT / "witchcraft_amd" / "libt5hip.so"
OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
NEEDED = 5

LINE = re.compile(r"^\t(\S+)\s*(.*?)\s*// ([0-9A-F]{12}): .*?(?:<(\S+?)(?:\+0x([0-9a-f]+))?>)?$")
VMEM = ("buffer_", "global_", "flat_", "scratch_")


class Instruction:
    def __init__(self, name, operands, kernel):
        self.name, self.operands, self.kernel, self.before = name, operands, kernel, []

    def states(self):
        return int(self.operands, 0) + 1 if self.name == "s_nop" else 1


def _scalars(text):
    out = set()
    for lo, hi, one, vcc in re.findall(r"\bs\[(\d+):(\d+)\]|\bs(\d+)\b|\b(vcc)\b", text):
        out.update((106, 107) if vcc else [int(one)] if one else range(int(lo), int(hi) + 1))
    return out


def _written(i):
    """Scalar registers that a vector instruction writes."""
    if not i.name.startswith("v_"):
        return set()
    ops = i.operands.split(",")
    return _scalars(ops[0]) | (_scalars(ops[1]) if len(ops) > 1 and ("_co_" in i.name or "div_scale" in i.name) else set())


def _code(asm):
    """Instructions of a disassembly, each with those that may run right before it."""
    code, place, symbols, jumps, kernel = [], {}, {}, [], None
    for line in asm.splitlines():
        m = re.match(r"^([0-9a-f]+) <(\S+)>:", line)
        if m:
            kernel = m.group(2)
            symbols[kernel] = int(m.group(1), 16)
            continue
        m = LINE.match(line)
        if not m:
            continue
        i = Instruction(m.group(1), m.group(2), kernel)
        if code and code[-1].kernel == kernel and code[-1].name not in ("s_branch", "s_endpgm", "s_setpc_b64"):
            i.before.append(code[-1])
        if i.name.startswith(("s_cbranch", "s_branch")) and m.group(4):
            jumps.append((i, m.group(4), int(m.group(5) or "0", 16)))
        place[int(m.group(3), 16)] = i
        code.append(i)
    for i, symbol, offset in jumps:
        place[symbols[symbol] + offset].before.append(i)
    return code


@pytest.fixture(scope="module")
def objects(tmp_path_factory):
    if not SO.exists():
        pytest.skip("libt5hip.so is not built")
    if not OBJDUMP.exists():
        pytest.skip("ROCm LLVM tools are not installed")
    tmp = tmp_path_factory.mktemp("code")
    lib = tmp / SO.name
    shutil.copy(SO, lib)
    subprocess.run([str(OBJDUMP), "--offloading", str(lib)], cwd=tmp, check=True, stdout=subprocess.DEVNULL,
                   stderr=subprocess.DEVNULL)
    return [_code(subprocess.run([str(OBJDUMP), "-d", str(co)], check=True, capture_output=True, text=True).stdout)
            for co in sorted(tmp.glob(SO.name + ".*gfx950"))]


def _nearest_write(i, limit):
    """Fewest wait states between a vector write of a scalar register that i reads and i; limit if more."""
    reads, found = _scalars(i.operands), limit
    todo, seen = [(j, 0) for j in i.before], {}
    while todo and reads:
        j, states = todo.pop()
        if states >= found or seen.get(id(j), limit) <= states:
            continue
        seen[id(j)] = states
        if _written(j) & reads:
            found = states
        todo += [(k, states + j.states()) for k in j.before]
    return found


def test_vector_memory_waits_for_its_scalars(objects):
    seen = 0
    for code in objects:
        for i in code:
            if i.name.startswith(VMEM) and _scalars(i.operands):
                seen += 1
                assert _nearest_write(i, NEEDED) >= NEEDED, (i.kernel, i.name, i.operands)
    assert seen > 1000


def test_buffer_copies_bring_their_own_wait_states(objects):
    """Whatever stands in front of a copy, or of a run of them, its own instructions before the load are enough."""
    copies = [i for code in objects for i in code if i.name.startswith("buffer_load") and i.operands.endswith("lds")]
    assert len(copies) > 500
    for i in copies:
        states, j = 0, i
        while states < NEEDED:
            (j,) = j.before
            own = j.name == "s_nop" or j.operands.startswith("m0,") or (j.name.startswith("buffer_load") and j.operands.endswith("lds"))
            assert own, (i.kernel, j.name, j.operands, states)
            states += j.states()
