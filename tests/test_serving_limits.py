"""Host-only checks of the serving operators' limits: the largest sizes that are taken, and the ones behind them."""
import ctypes as C

import pytest

from tests.test_serving_abi import INVALID, append_args, lib, pkg, prefix_args  # noqa: F401

TOP = (1 << 31) - 1


# A page of 2^20 keys that a table holds 2^11 times is within the caches' limits.
@pytest.mark.parametrize("page", [32, 64, 96, 1024, 1 << 20])
def test_prefix_refuses_key_counts_near_2_31(pkg, lib, page):
    """Positions are ints, and the kernels add a tile's width to them."""
    def args(keys):
        return prefix_args(pkg, batch=1, total_q=1, max_seqlen_k=keys, page_size=page, num_pages=1,
                           max_pages_per_seq=-(-keys // page), max_pages_per_prefix=-(-keys // page))
    most = (TOP - 255) // page * page
    for keys, ok in ((TOP, False), (TOP - 62, False), (most + 1, False), (most, True), (most - page + 1, True)):
        a = args(keys)
        assert (lib.fav4_bshd_prefix_paged_workspace_size(C.byref(a), 0) > 0) == ok, keys
        if not ok:
            assert lib.fav4_bshd_forward_prefix_paged(C.byref(a), 0, 0x1000000, 1 << 40, None) == INVALID


@pytest.mark.parametrize("batch", [TOP, TOP - 62])
def test_append_refuses_batches_near_2_31(pkg, lib, batch):
    """A wave's search for a token's sequence takes 64 equal steps through the offsets, which are ints."""
    assert lib.fav4_bshd_append_paged(C.byref(append_args(pkg, batch=batch)), None) == INVALID
