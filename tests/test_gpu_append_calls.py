"""GPU checks of appending to paged K/V caches called as a serving engine calls it: padded batches, and the same call
from two streams."""
import numpy as np
import pytest
import torch

from tests.serving import D, assert_rotated
from tests.test_gpu_append import Append

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("in_place", [False, True])
def test_tokens_before_the_first_offset(gpu_runner, in_place):
    """Offsets that start behind 0: those tokens' rows stay as they are, and nothing of theirs is stored."""
    x = Append(8, 2, 16, [(2, 2), (5, 30), (0, 7), (3, 40)], 64, False, False, False, in_place, behind=3)
    x.seqlens[0] = 2
    x.cu_d[0] = 2                                        # the first sequence has no tokens left
    x.call(gpu_runner)
    torch.cuda.synchronize()
    left = x.q_in[:2] if in_place else torch.full_like(x.q_in[:2], float("nan"))
    assert torch.equal(x.q_out[:2].view(torch.int16), left.view(torch.int16))
    page = x.table[0, 0]
    for now, was in ((x.kc, x.before[0]), (x.vc, x.before[1])):
        assert torch.equal(now[page].view(torch.int16), was[page].view(torch.int16))
    # The rest as ever: sequence 0 as one that stores nothing.
    slots, rows = x.where()
    kept = np.arange(2, 10)
    at = torch.from_numpy(slots[kept].astype(np.int64)).to(x.dev)
    assert_rotated(x.q_out[2:10], x.q_in[2:10], x.cos[at], x.sin[at], False, "q")
    flat = torch.from_numpy(rows[kept].astype(np.int64)).to(x.dev)
    assert_rotated(x.kc.view(-1, 2, D)[flat], x.k[2:10], x.cos[at], x.sin[at], False, "k")
    assert torch.equal(x.vc.view(-1, 2, D)[flat].view(torch.int16), x.v[2:10].view(torch.int16))


def test_a_graph_of_a_padded_batch(gpu_runner):
    """Captured for 40 tokens of 6 sequences, replayed with fewer and none, with eager calls between."""
    x = Append(8, 2, 16, [(7, 30), (9, 40), (4, 33), (8, 50), (6, 20), (6, 6)], 128, True, True, False, False)
    graph = torch.cuda.CUDAGraph()
    x.call(gpu_runner)
    torch.cuda.synchronize()
    x.check()
    with torch.cuda.graph(graph):
        x.call(gpu_runner)
    for new in ([1, 1, 1, 1, 1, 1], [0, 9, 0, 8, 0, 0], [0] * 6, [7, 9, 4, 8, 6, 6]):
        x.lens = [(n, sk) for n, (_, sk) in zip(new, x.lens)]
        x.cu = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        x.cu_d.copy_(torch.from_numpy(x.cu))
        for t in (x.q, x.k, x.v):
            t.copy_(torch.randn(t.shape, device=x.dev).to(torch.bfloat16))
        for once in (graph.replay, lambda: x.call(gpu_runner)):
            x.q_in = x.q.clone()
            x.q_out.fill_(float("nan"))
            x.before = x.kc.clone(), x.vc.clone()
            once()
            torch.cuda.synchronize()
            x.check()


def test_two_streams(gpu_runner):
    """Two batches at once, each on a stream of its own."""
    xs = [Append(16, 4, 64, [(300, 700), (1, 65), (200, 200)], 128, i == 1, False, False, False, seed=5 + i) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(5):
        for x, s in zip(xs, streams):
            x.call(gpu_runner, stream=s.cuda_stream)
    torch.cuda.synchronize()
    for x in xs:
        x.check()
