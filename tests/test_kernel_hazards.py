"""Wait states that gfx950 leaves to software, in the built kernels' own machine code.

The compiler adds them to the code that it makes and does not look into inline assembly. Each test walks back from every
memory instruction over all ways that lead to it, an instruction a wait state, s_nop n n + 1. Runs on the CPU; skipped when the
kernels are not built.
"""
import re
import subprocess
from functools import lru_cache
from pathlib import Path

import pytest
from test_kernel_resources import _gfx_elf, _objects

OBJDUMP = Path("/opt/rocm/llvm/bin/llvm-objdump")
LINE = re.compile(r"\s+(\S+)\s*(.*?)\s*// ([0-9A-F]+): ")
TARGET = re.compile(r"<\S+?\+0x([0-9a-f]+)>\s*$")
MEMORY = ("global_", "buffer_", "flat_", "scratch_")


class Code:
    """Instructions as (name, operands), and the numbers of those that may come right before each."""

    def __init__(self, text):
        self.ops, at, jumps = [], {}, []
        for line in text.splitlines():
            m = LINE.match(line)
            if not m:
                continue
            name, operands, address = m[1], m[2], int(m[3], 16)
            to = TARGET.search(line)
            if to and name.startswith(("s_branch", "s_cbranch")):
                jumps.append((len(self.ops), int(to[1], 16)))
                operands = ""
            at[address] = len(self.ops)
            self.ops.append((name, operands))
        assert self.ops
        self.before = [[] for _ in self.ops]
        for i, (name, _) in enumerate(self.ops[:-1]):
            if name not in ("s_branch", "s_endpgm", "s_setpc_b64"):
                self.before[i + 1].append(i)
        for i, to in jumps:
            self.before[at[min(at) + to]].append(i)

    def too_close(self, i, states, writes):
        """The number of an instruction that `writes` fewer than `states` wait states before i, or None."""
        ways, seen = [(i, 0)], {}
        while ways:
            j, waited = ways.pop()
            for k in self.before[j]:
                name, operands = self.ops[k]
                if writes(name, operands):
                    return k
                upto = waited + (int(operands, 0) + 1 if name == "s_nop" else 1)
                if upto < states and seen.get(k, states) > upto:
                    seen[k] = upto
                    ways.append((k, upto))
        return None


@lru_cache(maxsize=None)
def code(co, folder):
    elf = folder / (co.stem + ".elf")
    elf.write_bytes(_gfx_elf(co.read_bytes()))
    return Code(subprocess.run([OBJDUMP, "-d", str(elf)], capture_output=True, text=True, check=True).stdout)


@pytest.fixture(scope="module")
def folder(tmp_path_factory):
    return tmp_path_factory.mktemp("code")


needs_kernels = pytest.mark.skipif(not _objects() or not OBJDUMP.exists(), reason="kernels not built, or nothing to read them with")


def scalars(operands):
    """Scalar registers that an instruction's operands name."""
    found = {int(n) for n in re.findall(r"\bs(\d+)\b", operands)}
    for first, last in re.findall(r"\bs\[(\d+):(\d+)\]", operands):
        found |= set(range(int(first), int(last) + 1))
    return found | set(re.findall(r"\bvcc\b", operands))


def to_lds(name, operands):
    return name.startswith(MEMORY) and ("_lds_" in name or re.search(r"\blds\b", operands))


def test_walk():
    """Ways back over branches and past waits."""
    text = """
\ts_mov_b32 m0, s1 // 000000001000: 00
\ts_cbranch_scc0 2 // 000000001004: 00 <k+0xc>
\ts_nop 0 // 000000001008: 00
\tglobal_load_lds_dwordx4 v1, s[2:3] // 00000000100C: 00
\ts_mov_b32 m0, s2 // 000000001010: 00
\tglobal_load_lds_dwordx4 v1, s[2:3] // 000000001014: 00
\ts_endpgm // 000000001018: 00
"""
    c = Code(text)
    assert c.before[3] == [2, 1]
    m0 = lambda name, operands: operands.startswith("m0")  # noqa: E731
    assert c.too_close(3, 1, m0) is None and c.too_close(3, 2, m0) == 0 and c.too_close(5, 1, m0) == 4


@needs_kernels
@pytest.mark.parametrize("co", _objects(), ids=lambda p: p.stem)
def test_m0_before_loads_to_lds(co, folder):
    """A scalar write of M0 is one wait state or more before a load to LDS, which reads it."""
    c = code(co, folder)
    for i, (name, operands) in enumerate(c.ops):
        if to_lds(name, operands):
            at = c.too_close(i, 1, lambda n, o: n.startswith("s_") and re.match(r"m0\b", o))
            assert at is None, f"{co.stem}: {c.ops[at]} then {c.ops[i]}"


@needs_kernels
@pytest.mark.parametrize("co", _objects(), ids=lambda p: p.stem)
def test_scalars_before_memory(co, folder):
    """A vector instruction's write of a scalar register is five wait states or more before a memory instruction that reads it."""
    c = code(co, folder)
    for i, (name, operands) in enumerate(c.ops):
        read = scalars(operands) if name.startswith(MEMORY) else set()
        if not read:
            continue

        def writes(n, o):
            results = 2 if "_co_" in n or n.startswith(("v_div_scale", "v_mad_u64", "v_mad_i64")) else 1
            return n.startswith("v_") and scalars(",".join(o.split(",")[:results])) & read

        at = c.too_close(i, 5, writes)
        assert at is None, f"{co.stem}: {c.ops[at]} then {c.ops[i]}"
