"""Calls of the 4-bit caches' operators that their rules allow, or that they bound: offsets out of order and out of range,
pages that several sequences share, two calls at once, tensors that are part of a graph of gradients."""
import numpy as np
import pytest
import torch

from tests.mx4 import Cache4, assert_guard_rows_untouched, values
from tests.test_gpu_mx4_append import Tokens
from tests.test_gpu_mx4_forms import FORMS, batch_of

pytestmark = pytest.mark.gpu


def guarded(shape, dtype, fill, dev, guard=1 << 16):
    """A tensor in the middle of a buffer, and a check that what lies around it has not changed."""
    size = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
    room = torch.full((guard + size + guard,), 0xa5, dtype=torch.uint8, device=dev)
    inner = room[guard:guard + size].view(dtype).view(shape)
    inner.fill_(fill)
    return inner, lambda: bool((room[:guard] == 0xa5).all()) and bool((room[guard + size:] == 0xa5).all())


def bad_offsets(n, total, seed):
    """Offsets of n sequences in no order, some negative and some past the end."""
    rng = np.random.default_rng(seed)
    out = rng.integers(0, total + 1, n + 1)
    out[rng.random(n + 1) < 0.2] = -5
    out[rng.random(n + 1) < 0.2] = total + 1000
    out[0], out[-1] = [(0, total), (-7, total + 9), (total, 0)][seed % 3]
    return torch.tensor(out, dtype=torch.int32)


@pytest.mark.parametrize("seed", range(3))
@pytest.mark.parametrize("form", FORMS)
def test_attention_with_bad_offsets(gpu_runner, form, seed):
    """Undefined results, and no byte written around O, the LSE and the workspace."""
    batch = batch_of(form, 64)
    n, pages = len(batch.lens), batch.table.shape[1]
    o, o_ok = guarded(tuple(batch.q.shape), torch.bfloat16, 0, batch.dev)
    lse, lse_ok = guarded((batch.heads, batch.total), torch.float32, 0, batch.dev)
    need = gpu_runner.paged_mx4_workspace_size(n, batch.heads, batch.kv_heads, batch.max_q, batch.max_k, batch.total, 64,
                                               pages, batch.caches[0].shape[0], 2)
    ws, ws_ok = guarded((need,), torch.uint8, 0, batch.dev)
    good = batch.cu.clone()
    batch.cu.copy_(bad_offsets(n, batch.total, seed))
    for causal in (0, 2):
        batch.attend(gpu_runner, o, lse, causal, workspace=ws)
        torch.cuda.synchronize()
        assert o_ok() and lse_ok() and ws_ok()
    # The next call in the same buffers is as ever.
    batch.cu.copy_(good)
    batch.attend(gpu_runner, o, lse, 2, workspace=ws)
    batch.check(o, lse, 2)


@pytest.mark.parametrize("seed", range(6))
def test_rows_with_bad_offsets(gpu_runner, seed):
    """Storing and reading back: no byte written around the caches, Q and the rows."""
    t = Tokens([(1 + i % 5, 40 + i) for i in range(100 if seed < 3 else 20)])
    caches = [guarded(tuple(x.shape), torch.uint8, 0, t.dev) for x in t.caches]
    t.caches = [x for x, _ in caches]
    t.q_out, q_ok = guarded(tuple(t.q.shape), torch.bfloat16, 0, t.dev)
    (k, k_ok), (v, v_ok) = (guarded(tuple(t.k.shape), torch.bfloat16, 0, t.dev) for _ in range(2))
    t.cu.copy_(bad_offsets(len(t.lens), t.n, seed))
    t.append(gpu_runner)
    for starts in (None, t.seqlens):
        gpu_runner.call_gather_paged_mx4(*t.caches, k, v, t.cu, t.table_d, starts=starts)
    torch.cuda.synchronize()
    assert q_ok() and k_ok() and v_ok() and all(ok() for _, ok in caches)


@pytest.mark.parametrize("form", FORMS)
def test_shared_pages(gpu_runner, form):
    """Every sequence begins with the first one's pages, and one has a page twice."""
    batch = batch_of(form, 64)
    first = batch.pages[0]
    for b, (_, sk) in enumerate(batch.lens):
        n = min(len(first), sk // 64)             # whole pages of both
        n = min(n, batch.lens[0][1] // 64)
        batch.pages[b] = np.concatenate([first[:n], batch.pages[b][n:]])
    if len(batch.pages[0]) > 2:
        batch.pages[0][1] = batch.pages[0][0]
    for b, pages in enumerate(batch.pages):
        batch.table[b, :len(pages)] = pages
    batch.table_d.copy_(torch.from_numpy(batch.table))
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    batch.check(o, lse, 2)
    rows = sum(sk for _, sk in batch.lens)
    k, v = (torch.empty(rows, batch.kv_heads, 128, dtype=torch.bfloat16, device=batch.dev) for _ in range(2))
    cu = torch.tensor(np.cumsum([0] + [sk for _, sk in batch.lens]), dtype=torch.int32, device=batch.dev)
    gpu_runner.call_gather_paged_mx4(*batch.caches, k, v, cu, batch.table_d)
    want = [torch.cat([batch.keys(b)[j] for b in range(len(batch.lens))]) for j in (0, 1)]
    assert torch.equal(k.double(), want[0]) and torch.equal(v.double(), want[1])


def test_two_calls_at_once(gpu_runner):
    """Eager calls on two streams, each with its own workspace, over the same caches."""
    batches = [batch_of("few_line", 64), batch_of("few_line", 64)]
    batches[1].caches = batches[0].caches
    batches[1].q = batches[0].q.flip(0).contiguous()
    streams = [torch.cuda.Stream() for _ in batches]
    outs, spaces = [b.outputs(True) for b in batches], []
    for batch, out in zip(batches, outs):
        spaces.append(batch.attend(gpu_runner, *out, 2))
    for _ in range(5):
        for o, lse in outs:
            o.fill_(float("nan")), lse.fill_(float("nan"))
        torch.cuda.synchronize()
        for batch, out, stream, ws in zip(batches, outs, streams, spaces):
            with torch.cuda.stream(stream):
                for _ in range(3):
                    batch.attend(gpu_runner, *out, 2, workspace=ws)
        torch.cuda.synchronize()
        for batch, (o, lse) in zip(batches, outs):
            batch.check(o, lse, 2)


def test_tensors_of_a_graph_of_gradients(gpu_runner):
    """The operators have no backward pass; inputs that need gradients are read as they are, and nothing is recorded."""
    t = Tokens([(5, 20), (3, 9)])
    want = t.want()
    t.k, t.v, t.q = (x.detach().requires_grad_() * 1 for x in (t.k, t.v, t.q))
    t.append(gpu_runner)
    torch.cuda.synchronize()
    t.k, t.v, t.q = (x.detach() for x in (t.k, t.v, t.q))
    t.check(want)
    assert not t.q_out.requires_grad
    k, v = torch.empty_like(t.k), torch.empty_like(t.v)
    gpu_runner.call_gather_paged_mx4(*t.caches, k, v, t.cu, t.table_d, starts=t.seqlens - t.cu.diff())
    assert torch.equal(k.double(), values(t.caches[0], t.caches[1])[t.at, :, t.place])
    batch = Cache4(4, 2, 16, [(2, 60)])
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2, q=batch.q.detach().requires_grad_())
    batch.check(o, lse, 2)
    assert_guard_rows_untouched(batch)
