"""Host-only checks of the 4-bit caches' built kernels: registers and LDS from the compiler's remarks."""
import re

import pytest

from tests.conftest import load_package


@pytest.fixture(scope="module")
def table():
    pkg = load_package()
    if not pkg.MX4_LIB_PATH.exists() or not pkg.fav4_bshd.RESOURCE_LOG.exists():
        pkg.build_library()
    return pkg.fav4_bshd.parse_resource_usage(pkg.fav4_bshd.RESOURCE_LOG.read_text())


# Least waves a SIMD: the workgroups that the launches count on being resident at once.
@pytest.mark.parametrize("pattern,count,waves", [(r"mx4_decode_kernelILi1ELi4E", 4, 3), (r"mx4_decode_kernelILi1ELi8E", 4, 2),
                                                 (r"mx4_decode_kernelILi1ELi12E", 4, 3),
                                                 (r"mx4_decode_kernelILi2E", 8, 2), (r"mx4_prefill_kernelI", 4, 2),
                                                 (r"mx4_prefill_line_kernelI", 4, 2), (r"mx4_merge_kernelI", 3, 7),
                                                 (r"mx4_store_kernelI", 2, 7), (r"mx4_read_kernel", 1, 8)])
def test_kernels_keep_their_waves(table, pattern, count, waves):
    kernels = {n: r for n, r in table.items() if re.search(pattern, n)}
    assert len(kernels) == count, sorted(kernels)
    for name, r in kernels.items():
        assert r["Occupancy [waves/SIMD]"] >= waves, (name, r)
        assert r["ScratchSize [bytes/lane]"] == 0 and r["VGPRs Spill"] == 0, (name, r)


def test_workgroups_fit_a_cu(table):
    """LDS: 160 KiB a CU, for three workgroups of a decode line, two of a prefill one."""
    for pattern, each in ((r"mx4_decode_kernelILi1ELi4E", 3), (r"mx4_decode_kernelILi2ELi4E", 2),
                          (r"mx4_decode_kernelILi\dELi(8|12)E", 1), (r"mx4_prefill_(line_)?kernelILi4E", 2),
                          (r"mx4_prefill_(line_)?kernelILi8E", 1)):
        kernels = {n: r for n, r in table.items() if re.search(pattern, n)}
        assert kernels
        for name, r in kernels.items():
            assert each * r["LDS Size [bytes/block]"] <= 160 << 10, (name, r)
