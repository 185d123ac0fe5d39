"""Attention over 4-bit paged caches (fav4_bshd_forward_paged_mx4) against 64-bit references."""
import numpy as np
import pytest
import torch

from tests.mx4 import Cache4, assert_guard_rows_untouched

pytestmark = pytest.mark.gpu

RAGGED = [0, 1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 500, 1000]


def run(runner, batch, causal, lse=True, **more):
    o, l = batch.outputs(lse)
    batch.attend(runner, o, l, causal, **more)
    torch.cuda.synchronize()
    batch.check(o, l, causal)
    assert_guard_rows_untouched(batch)
    return o, l


@pytest.mark.parametrize("heads,kv_heads", [(8, 8), (32, 8), (8, 1), (15, 3), (40, 2)])
@pytest.mark.parametrize("page", [16, 48, 64])
def test_decode(gpu_runner, heads, kv_heads, page):
    run(gpu_runner, Cache4(heads, kv_heads, page, [(1, k) for k in RAGGED]), 0)


@pytest.mark.parametrize("lens", [[(1, 1)], [(1, 0)], [(1, 16)], [(1, 64)], [(1, 777)], [(0, 50), (1, 3), (0, 0)]], ids=str)
@pytest.mark.parametrize("lse", [False, True])
def test_few_sequences(gpu_runner, lens, lse):
    for causal in (0, 2):
        run(gpu_runner, Cache4(8, 2, 32, lens), causal, lse)


# Rows a sequence: 2 to 64 (few), past that many; sequences with fewer keys than queries have rows that see none.
@pytest.mark.parametrize("sq", [2, 4, 5, 8, 13, 16, 17, 40, 64, 65, 129])
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (6, 2), (4, 4)])
def test_bottom_right(gpu_runner, sq, heads, kv_heads):
    lens = [(sq, k) for k in (0, 1, sq - 1, sq, sq + 1, 63, 64, 65, 200, 700)] + [(1, 33), (0, 5), (sq // 2, 300)]
    run(gpu_runner, Cache4(heads, kv_heads, 16, lens), 2)


@pytest.mark.parametrize("sq", [3, 30, 100])
def test_dense_with_several_queries(gpu_runner, sq):
    run(gpu_runner, Cache4(8, 2, 32, [(sq, k) for k in (0, 1, 31, 64, 257, 900)]), 0)


@pytest.mark.parametrize("heads,kv_heads,sq", [(32, 8, 1), (8, 1, 1), (8, 2, 4), (16, 2, 8), (4, 4, 1)])
@pytest.mark.parametrize("causal", [0, 2])
def test_long_keys_are_split(gpu_runner, heads, kv_heads, sq, causal):
    """More keys than one workgroup takes: parts and their merge, beside short, empty and query-less sequences."""
    lens = [(sq, 5000), (sq, 1), (sq, 0), (0, 100), (sq, 2049), (sq, 300), (sq, 4096), (1, 3000)]
    run(gpu_runner, Cache4(heads, kv_heads, 64, lens), causal)


@pytest.mark.parametrize("lens", [[(1, 20000)], [(4, 9000)], [(1, 2500)] * 3], ids=str)
def test_one_long_sequence(gpu_runner, lens):
    run(gpu_runner, Cache4(8, 1, 64, lens), 2)


@pytest.mark.parametrize("lens", [[(300, 300)], [(100, 2000), (257, 3000), (1, 700), (64, 64)], [(1000, 1000), (513, 600)],
                                  [(200, 5000)]], ids=str)
@pytest.mark.parametrize("heads,kv_heads", [(8, 2), (4, 1), (3, 3)])
@pytest.mark.parametrize("causal", [0, 2])
def test_prefill(gpu_runner, lens, heads, kv_heads, causal):
    run(gpu_runner, Cache4(heads, kv_heads, 64, lens), causal)


def test_many_sequences(gpu_runner):
    """More sequences than a wave has lanes, in both kinds of call."""
    rng = np.random.default_rng(5)
    lens = [(1, int(k)) for k in rng.integers(0, 300, 150)]
    run(gpu_runner, Cache4(4, 2, 16, lens), 0)
    run(gpu_runner, Cache4(4, 2, 16, lens[:140] + [(1, 2500)]), 0)
    run(gpu_runner, Cache4(4, 2, 16, [(int(q), int(k)) for q, k in zip(rng.integers(0, 60, 100), rng.integers(0, 300, 100))]), 2)


@pytest.mark.parametrize("lse", [False, True])
def test_a_row_tile_for_every_cu(gpu_runner, lse):
    """256 row tiles of 256 rows."""
    run(gpu_runner, Cache4(32, 8, 64, [(512, 2000)] * 4), 0, lse)


@pytest.mark.parametrize("count", [40, 64, 65])
@pytest.mark.parametrize("causal", [0, 2])
def test_row_tiles_of_many_lengths(gpu_runner, count, causal):
    """Row tiles of many rows in the order of their key tiles, among them idle sequences, equal ones, ones without keys and
    ones with fewer keys than queries."""
    rng = np.random.default_rng(count)
    sq = rng.choice([0, 1, 33, 64, 65, 130, 257, 300], count)
    sk = np.where(rng.random(count) < 0.5, sq, rng.integers(0, 700, count))
    batch = Cache4(8, 4, 16, [(int(q), int(k)) for q, k in zip(sq, sk)])
    run(gpu_runner, batch, causal)
    run(gpu_runner, batch, causal, total_k=1)
    run(gpu_runner, batch, causal, total_k=int(sk.sum()))


def test_results_are_the_same_from_call_to_call(gpu_runner):
    for lens, causal in (([(1, 5000), (1, 77)] * 4, 0), ([(150, 1500)] * 2, 2)):
        batch = Cache4(8, 2, 64, lens)
        first = [x.clone() for x in run(gpu_runner, batch, causal)]
        again = run(gpu_runner, batch, causal)
        assert all(torch.equal(x.view(torch.int8), y.view(torch.int8)) for x, y in zip(first, again))
