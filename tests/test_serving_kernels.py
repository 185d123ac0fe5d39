"""Host-only checks of the built serving kernels: registers from the compiler's remarks, and that no wave of the
attention ends with a copy into LDS in flight (it clamps the prefetches past its last tile instead of leaving them
out)."""
import re
import subprocess

import pytest

from tests.conftest import load_package
from tests.test_lds_dma_drain import OBJDUMP, _code_object, _ends_with_copy_in_flight


@pytest.fixture(scope="module")
def pkg():
    p = load_package()
    if not p.SERVING_LIB_PATH.exists() or not p.fav4_bshd.RESOURCE_LOG.exists():
        p.build_library()
    return p


def _resources(pkg, pattern):
    table = pkg.fav4_bshd.parse_resource_usage(pkg.fav4_bshd.RESOURCE_LOG.read_text())
    return {n: r for n, r in table.items() if re.search(pattern, n)}


@pytest.mark.parametrize("pattern,count,waves", [(r"\d+prefix_kernelI", 12, 2), (r"prefix_merge_kernelI", 3, 4),
                                                 (r"append_kernelI", 2, 7)])
def test_kernels_keep_their_waves(pkg, pattern, count, waves):
    """The attention has 256 registers a wave; the merge and the append are bound by latency, so by their waves."""
    kernels = _resources(pkg, pattern)
    assert len(kernels) == count, sorted(kernels)
    for name, r in kernels.items():
        assert r["Occupancy [waves/SIMD]"] >= waves, (name, r)
        assert r["ScratchSize [bytes/lane]"] == 0 and r["VGPRs Spill"] == 0, (name, r)


def test_a_workgroup_of_eight_waves_fits_a_cu(pkg):
    """LDS: 160 KiB a CU."""
    for name, r in _resources(pkg, r"\d+prefix_kernelI").items():
        assert r["LDS Size [bytes/block]"] <= 160 << 10, (name, r)


@pytest.mark.skipif(not OBJDUMP.exists(), reason="needs llvm-objdump")
def test_no_wave_ends_with_a_copy_in_flight(pkg, tmp_path):
    elf = tmp_path / "gfx950.elf"
    elf.write_bytes(_code_object(pkg.SERVING_LIB_PATH))
    text = subprocess.run([str(OBJDUMP), "-d", str(elf)], capture_output=True, text=True, check=True).stdout
    table, code, base = {}, None, 0
    for line in text.splitlines():
        if (m := re.match(r"([0-9a-f]{16}) <(\S+)>:", line)):
            base, code = int(m[1], 16), table.setdefault(m[2], [])
        elif code is not None and (m := re.match(r"\t(.*?)\s*// ([0-9A-F]+):(.*)", line)):
            target = re.search(r"\+0x([0-9a-f]+)>", m[3]) if "branch" in m[1] else None
            start = base if "branch" in m[1] and target is None else None
            code.append((int(m[2], 16), m[1], base + int(target[1], 16) if target else start))
    kernels = {n: c for n, c in table.items() if re.search(r"\d+prefix_kernelI", n) and not n.endswith(".kd")}
    assert len(kernels) == 12
    for name, code in kernels.items():
        assert any(ins.startswith("buffer_load") and ins.endswith(" lds") for _, ins, _ in code), name
        assert not _ends_with_copy_in_flight(code), name
