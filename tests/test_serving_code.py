"""Host-only checks of the built serving kernels' own gfx950 code: what a documented rule says about memory that no
output shows."""
import re
import subprocess

import pytest

from tests.conftest import load_package
from tests.test_lds_dma_drain import OBJDUMP, _code_object

pytestmark = pytest.mark.skipif(not OBJDUMP.exists(), reason="needs llvm-objdump")


@pytest.fixture(scope="module")
def kernels(tmp_path_factory):
    """{mangled name: [(address, instruction, branch target or None)]}"""
    pkg = load_package()
    if not pkg.SERVING_LIB_PATH.exists():
        pkg.build_library()
    elf = tmp_path_factory.mktemp("co") / "gfx950.elf"
    elf.write_bytes(_code_object(pkg.SERVING_LIB_PATH))
    text = subprocess.run([str(OBJDUMP), "-d", str(elf)], capture_output=True, text=True, check=True).stdout
    table, code, base = {}, None, 0
    for line in text.splitlines():
        if (m := re.match(r"([0-9a-f]{16}) <(\S+)>:", line)):
            base, code = int(m[1], 16), table.setdefault(m[2], [])
        elif code is not None and (m := re.match(r"\t(.*?)\s*// ([0-9A-F]+):(.*)", line)):
            target = re.search(r"\+0x([0-9a-f]+)>", m[3]) if "branch" in m[1] else None
            start = base if "branch" in m[1] and target is None else None       # a branch to the first instruction
            code.append((int(m[2], 16), m[1], base + int(target[1], 16) if target else start))
    return table


def _wide_loads_before_a_decision(code):
    """Addresses of the 16-byte loads that some path from the entry reaches before it has read a 4-byte value from
    memory (kernel arguments aside, which lie at s[0:1]) and branched after that."""
    index = {addr: i for i, (addr, _, _) in enumerate(code)}
    seen, bad, todo = set(), set(), [(0, 0)]                # state: 1 a value read, 2 a branch behind it
    while todo:
        i, state = todo.pop()
        while i < len(code) and (i, state) not in seen:
            seen.add((i, state))
            addr, ins, target = code[i]
            if ins.startswith("global_load_dwordx4") and state < 2:
                bad.add(addr)
            elif state == 0 and (ins.startswith("global_load_dword ") or
                                 ins.startswith("s_load_dword") and "s[0:1]" not in ins):
                state = 1
            elif state == 1 and ins.startswith("s_cbranch"):
                state = 2
            elif ins.startswith("s_endpgm"):
                break
            if target is not None:
                todo.append((index[target], state))
                if ins.startswith("s_branch"):
                    break
            i += 1
    return bad


def test_append_reads_rows_of_sequences_alone(kernels):
    """Rows of tokens in no sequence are not read (their buffers may end before them): every load of a row comes
    behind a branch on the offsets."""
    appends = {n: c for n, c in kernels.items() if re.search(r"append_kernelI", n) and not n.endswith(".kd")}
    assert len(appends) == 2
    for name, code in appends.items():
        assert sum(ins.startswith("global_load_dwordx4") for _, ins, _ in code) >= 2, name
        assert not _wide_loads_before_a_decision(code), name
