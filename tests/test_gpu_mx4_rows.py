"""Storing in 4-bit caches and reading back: many sequences, streams, and more rows than one pass of the grids."""
import numpy as np
import pytest
import torch

from tests.mx4 import quantise, values
from tests.serving import D
from tests.test_gpu_mx4_append import Tokens

pytestmark = pytest.mark.gpu


def check_gather(runner, t, **more):
    """Every sequence's new rows, read back."""
    k, v = (torch.full_like(x, 3.0, memory_format=torch.contiguous_format) for x in (t.k, t.v))
    starts = torch.tensor([b - a for a, b in t.lens], dtype=torch.int32, device=t.dev)
    torch.cuda.synchronize()
    runner.call_gather_paged_mx4(*t.caches, k, v, t.cu, t.table_d, starts=starts, **more)
    torch.cuda.synchronize()
    at = np.where(t.at >= 0, t.at, 0)
    for j, x in ((0, k), (2, v)):
        ref = values(t.caches[j], t.caches[j + 1])[at, :, t.place]
        ref[torch.from_numpy(t.at < 0)] = 0
        got = x[:t.n].double()
        assert ((got == ref) | (got.isnan() & ref.isnan())).all()
        assert (x[t.n:] == 3).all()


@pytest.mark.parametrize("count", [65, 300, 5000])
@pytest.mark.parametrize("idle", [0.0, 0.9])
def test_many_sequences(gpu_runner, count, idle):
    """More sequences than a wave has lanes and than it finds in two steps, among them runs of more idle ones than lanes,
    also in front and at the end."""
    rng = np.random.default_rng(count)
    new = np.where(rng.random(count) < idle, 0, rng.integers(0, 4, count))
    for a in (0, count // 2, count - 70):
        if count > 65:
            new[a:a + 70] = 0
    new[count * 2 // 3] = 130                     # rows of one sequence over many waves
    t = Tokens([(int(n), int(n + c)) for n, c in zip(new, rng.integers(0, 40, count))], tail=3)
    want = t.want()
    t.append(gpu_runner)
    torch.cuda.synchronize()
    t.check(want)
    check_gather(gpu_runner, t)


@pytest.mark.parametrize("how", ["handle", "current", "default"])
def test_streams(gpu_runner, how):
    """Calls on a stream of their own, handed over as a raw handle and as torch's current one, and on the default one."""
    t = Tokens([(40, 100), (3, 3), (17, 17)])
    want = t.want()
    stream = torch.cuda.default_stream() if how == "default" else torch.cuda.Stream()
    torch.cuda.synchronize()
    if how == "current":
        with torch.cuda.stream(stream):
            t.append(gpu_runner)
            stream.synchronize()
            t.check(want)
            check_gather(gpu_runner, t)
    else:
        t.append(gpu_runner, stream=stream.cuda_stream)
        stream.synchronize()
        t.check(want)
        check_gather(gpu_runner, t, stream=stream.cuda_stream)


def test_more_rows_than_a_pass_of_the_grids(gpu_runner):
    """2^25 + 1003 rows of one sequence: the append takes 2^24 a pass, the reading 2^25.  Looked at are rows at both ends
    and on both sides of those borders."""
    n, page, dev = (1 << 25) + 1003, 64, "cuda:0"
    gen = torch.Generator(device=dev).manual_seed(6)
    k = torch.randn(n, 1, D, generator=gen, device=dev, dtype=torch.bfloat16)
    pages = -(-n // page)
    table = torch.randperm(pages, generator=gen, device=dev, dtype=torch.int32)[None].contiguous()
    caches = gpu_runner.mx4_caches(pages, 1, page, dev)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32, device=dev)
    gpu_runner.call_append_paged_mx4(None, k, k, None, *caches, i32(0, n), i32(n), table)
    k_rows, v_rows = torch.empty_like(k), torch.empty_like(k)
    gpu_runner.call_gather_paged_mx4(*caches, k_rows, v_rows, i32(0, n), table)
    for border in (0, 1 << 24, 1 << 25, n):
        rows = torch.arange(max(0, border - 500), min(n, border + 500), device=dev)
        codes, scales = quantise(k[rows].float().cpu().numpy())
        at, place = table[0, rows // page].long(), rows % page
        want = torch.from_numpy(values(codes, scales))
        for j, got in ((0, k_rows), (2, v_rows)):
            assert np.array_equal(caches[j][at, :, place].cpu().numpy(), codes)
            assert np.array_equal(caches[j + 1][at, :, place].cpu().numpy(), scales)
            assert torch.equal(got[rows].double().cpu(), want)
    assert torch.equal(k_rows, v_rows)
