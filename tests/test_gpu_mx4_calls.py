"""Calls of the 4-bit caches' operators as a serving loop makes them: no numbers in keys and queries, padded batches,
workspaces of exactly their size, captured graphs, streams, caches past 4 GiB, and decode steps of all three."""
import numpy as np
import pytest
import torch

from tests.mx4 import Cache4, assert_guard_rows_untouched, quantise, values
from tests.serving import D, SCALE, angles
from tests.test_gpu_mx4_append import Tokens

pytestmark = pytest.mark.gpu

# The kinds of call: whole sequences and lines of few rows, of one row tile and two, row tiles of 128 and of 256 rows,
# whole and on a line.
KINDS = {"whole": [(1, 300), (1, 77), (1, 640)], "line": [(1, 5000), (1, 300), (1, 2100)] * 3,
         "long_whole": [(4, 2100), (3, 1500), (4, 900), (1, 2099)] * 8,
         "drafts": [(5, 400), (5, 90)], "drafts_line": [(5, 6000), (5, 90), (3, 3500)],
         "prompts": [(150, 150), (200, 333)], "chunks": [(100, 4000), (40, 1500), (70, 70)],
         "long_chunks": [(300, 9000), (250, 2000)], "many_prompts": [(150, 150), (200, 333)] * 4,
         "many_chunks": [(100, 4000), (40, 1500), (70, 70)] * 4}


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("which,scale", [(1, 255), (3, 255), (3, 253), (1, 254)])
def test_keys_that_are_no_numbers(gpu_runner, kind, which, scale):
    """Rows that see such a key get NaN, all others what they get without it."""
    batch = Cache4(8, 2, 16, KINDS[kind])
    nan = torch.zeros(batch.total, 8, dtype=torch.bool, device=batch.dev)
    for b, (sq, sk) in enumerate(batch.lens):
        # In one head and one block: a key that only the last queries see, or (every other sequence) an early one.
        key, head = (sk - 1, 1) if b % 2 == 0 else (sk // 3, 0)
        batch.caches[which][batch.table[b, key // 16], head, key % 16, b % 4] = scale
        first = max(0, key - (sk - sq))
        nan[int(batch.offsets[b]) + first:int(batch.offsets[b + 1]), head * 4:head * 4 + 4] = True
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    batch.check(o, lse, 2, nan_rows=nan)


@pytest.mark.parametrize("kind", KINDS)
def test_queries_that_are_no_numbers(gpu_runner, kind):
    batch = Cache4(8, 2, 32, KINDS[kind])
    nan = torch.zeros(batch.total, 8, dtype=torch.bool, device=batch.dev)
    for b in range(len(batch.lens)):
        row, head = int(batch.offsets[b]), (3 * b + 1) % 8
        batch.q[row, head, 5 * b % D] = float("nan")
        nan[row, head] = True
    nan &= torch.tensor([sk > 0 and sk - sq >= 0 for sq, sk in batch.lens for _ in range(sq)], device=batch.dev)[:, None]
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    batch.check(o, lse, 2, nan_rows=nan)


@pytest.mark.parametrize("kind", KINDS)
def test_large_scores(gpu_runner, kind):
    """Scores of some hundreds: one key takes all of a row's weight.  (FP32 scores are off by at most 128 * 2^-24 of the
    products' sum, 16 times that of the tests with queries of 1: 1e-3 of a weight.)"""
    batch = Cache4(8, 2, 16, KINDS[kind])
    batch.q *= 16
    o, _ = batch.outputs(False)
    batch.attend(gpu_runner, o, None, 2)
    batch.check(o, None, 2, weight_err=3.2e-3)


@pytest.mark.parametrize("kind", KINDS)
def test_without_lse(gpu_runner, kind):
    """O does not depend on whether the LSE is asked for."""
    batch = Cache4(8, 2, 64, KINDS[kind])
    with_lse = batch.outputs(True)
    batch.attend(gpu_runner, *with_lse, 2)
    o, _ = batch.outputs(False)
    batch.attend(gpu_runner, o, None, 2)
    batch.check(*with_lse, 2)
    assert torch.equal(o, with_lse[0])


@pytest.mark.parametrize("kind", KINDS)
def test_scale(gpu_runner, kind):
    """A quarter of the scale is a quarter of the queries, bit by bit: powers of two do not change a rounding."""
    batch = Cache4(8, 2, 16, KINDS[kind])
    outs = []
    for scale, q in ((SCALE / 4, batch.q), (None, batch.q / 4)):
        o, lse = batch.outputs(True)
        batch.attend(gpu_runner, o, lse, 2, q=q, scale=scale)
        outs.append((o, lse))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    batch.check(*outs[1], 2, q=batch.q / 4)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("total_k", [None, 1, 1 << 30])
def test_workspaces_and_padded_batches(gpu_runner, kind, total_k):
    """A workspace of exactly its size, in the middle of a guarded one and full of NaN; rows behind the last sequence,
    idle sequences, and sizes larger than the batch needs."""
    batch = Cache4(8, 2, 16, KINDS[kind] + [(0, 0)] * 3, extra_pages=4)
    batch.q = torch.cat([batch.q, torch.full((9, 8, D), float("nan"), dtype=torch.bfloat16, device=batch.dev)])
    o, lse = batch.outputs(True)
    sizes = dict(max_q=batch.max_q + 7, max_k=batch.max_k + 30)
    need = gpu_runner.paged_mx4_workspace_size(len(batch.lens), 8, 2, sizes["max_q"], sizes["max_k"], o.shape[0], 16,
                                               batch.table.shape[1], batch.caches[0].shape[0], 2)
    guard = 4096
    room = torch.full((guard + need + guard,), 0xff, dtype=torch.uint8, device=batch.dev)
    used = batch.attend(gpu_runner, o, lse, 2, workspace=room[guard:guard + need], total_k=total_k, **sizes)
    assert used.data_ptr() == room.data_ptr() + guard
    batch.check(o, lse, 2)
    assert (room[:guard] == 0xff).all() and (room[guard + need:] == 0xff).all()
    assert o[batch.total:].isnan().all() and lse[:, batch.total:].isnan().all()
    assert_guard_rows_untouched(batch)
    with pytest.raises(RuntimeError):
        batch.attend(gpu_runner, o, lse, 2, workspace=room[guard:guard + need - 1], **sizes)
    # What the workspace held does not matter.
    first = o.clone(), lse.clone()
    room[guard:guard + need] = torch.randint(0, 256, (need,), dtype=torch.uint8, device=batch.dev)
    batch.attend(gpu_runner, o, lse, 2, workspace=room[guard:guard + need], total_k=total_k, **sizes)
    assert torch.equal(first[0][:batch.total], o[:batch.total]) and torch.equal(first[1][:, :batch.total], lse[:, :batch.total])


@pytest.mark.parametrize("heads,lens", [(300, [(256, 4000)]), (600, [(130, 1500), (90, 900)]), (800, [(2, 700)])])
def test_more_heads_than_cus(gpu_runner, heads, lens):
    """A range for each K/V head, in a workspace of exactly its size between guards."""
    batch = Cache4(heads, heads, 64, lens)
    o, lse = batch.outputs(True)
    need = gpu_runner.paged_mx4_workspace_size(len(lens), heads, heads, batch.max_q, batch.max_k, o.shape[0], 64,
                                               batch.table.shape[1], batch.caches[0].shape[0], 2)
    guard = 1 << 20
    room = torch.full((guard + need + guard,), 0xff, dtype=torch.uint8, device=batch.dev)
    batch.attend(gpu_runner, o, lse, 2, workspace=room[guard:guard + need])
    batch.check(o, lse, 2)
    assert (room[:guard] == 0xff).all() and (room[guard + need:] == 0xff).all()
    assert_guard_rows_untouched(batch)


def test_one_device(gpu_runner):
    """A host tensor among the GPU's is refused, whichever it is."""
    t = Tokens([(3, 10), (2, 5)])
    blocks, (k, v) = gpu_runner.mx4_blocks, (torch.empty_like(x[:t.n]) for x in (t.k, t.v))
    cos, sin = angles(64, 128, t.dev)
    o, lse = torch.empty_like(t.q), torch.empty(t.q.shape[1], t.q.shape[0], device=t.dev)
    positions = torch.zeros(t.q.shape[0], dtype=torch.int32, device=t.dev)
    for call, args in ((blocks.append, [t.q, t.k, t.v, t.q_out, *t.caches, t.cu, t.seqlens, t.table_d, cos, sin, False, positions]),
                       (blocks.gather, [*t.caches, k, v, t.cu, t.table_d, t.seqlens]),
                       (blocks.paged, [t.q, *t.caches, o, lse, t.cu, t.seqlens, t.table_d, 3, 10, None, None])):
        call(*args)
        for i, x in enumerate(args):
            if isinstance(x, torch.Tensor):
                with pytest.raises(AssertionError, match="one device"):
                    call(*args[:i], x.cpu(), *args[i + 1:])


def test_more_sequences_than_a_line_is_laid_out_for(gpu_runner):
    """600 sequences, some of them of many rows: past what a workgroup keeps in LDS."""
    rng = np.random.default_rng(3)
    lens = [(int(q), int(k)) for q, k in zip(np.where(np.arange(600) % 100 == 7, 70, 1), rng.integers(0, 200, 600))]
    batch = Cache4(4, 4, 16, lens)
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2)
    batch.check(o, lse, 2)


@pytest.mark.parametrize("page", [16, 64])
def test_lengths_and_pages_out_of_range(gpu_runner, page):
    """Key counts past max_seqlen_k are cut to it, negative ones are none; entries behind a sequence's keys are not used,
    whatever they are, also where a tile reaches past them."""
    for kind in ("whole", "line", "drafts", "chunks", "many_prompts", "many_chunks"):
        batch = Cache4(8, 2, page, KINDS[kind] + [(1, 0)])
        most = max(sk for _, sk in batch.lens)
        want, got = batch.outputs(True), None
        batch.attend(gpu_runner, *want, 0)
        want = [x.clone() for x in want]
        longest = [i for i, (_, sk) in enumerate(batch.lens) if sk == most]
        batch.seqlens[longest] = most + 12345
        batch.seqlens[-1] = -7
        got = batch.outputs(True)
        batch.attend(gpu_runner, *got, 0)
        assert all(torch.equal(x, y) for x, y in zip(want, got))


@pytest.mark.parametrize("kind", KINDS)
def test_graph_follows_the_lengths(gpu_runner, kind):
    """A captured call, replayed between eager work: it reads the lengths on the device."""
    batch = Cache4(8, 2, 16, KINDS[kind])
    o, lse = batch.outputs(True)
    ws = batch.attend(gpu_runner, o, lse, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        batch.attend(gpu_runner, o, lse, 2, workspace=ws)
    full = batch.lens
    for step in range(4):
        lens = [(sq, max(sq, sk - 37 * step)) for sq, sk in full]
        batch.lens = lens
        batch.seqlens.copy_(torch.tensor([sk for _, sk in lens], dtype=torch.int32))
        o.fill_(float("nan")), lse.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        batch.check(o, lse, 2)
        eager = torch.full_like(o, float("nan")), torch.full_like(lse, float("nan"))
        batch.attend(gpu_runner, *eager, 2, total_k=None)
        assert torch.equal(o, eager[0]) and torch.equal(lse, eager[1])


def test_two_graphs_with_workspaces_of_their_own(gpu_runner):
    batches = [Cache4(8, 1, 32, [(1, 4000), (1, 900)], seed=s) for s in (1, 2)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in batches], [], []
    workspaces = []                   # both live as long as the graphs: entering a capture gives unused memory back
    for batch, stream in zip(batches, streams):
        out = batch.outputs(True)
        ws = batch.attend(gpu_runner, *out, 0)
        workspaces.append(ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            batch.attend(gpu_runner, *out, 0, workspace=ws)
        graphs.append(graph), outs.append(out)
    for _ in range(5):
        for o, lse in outs:
            o.fill_(float("nan")), lse.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for batch, (o, lse) in zip(batches, outs):
            batch.check(o, lse, 0)


def test_streams(gpu_runner):
    """Calls on a stream of their own, handed over as a raw handle and as torch's current one."""
    batch = Cache4(8, 2, 16, KINDS["line"])
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    for raw in (True, False):
        o, lse = batch.outputs(True)
        stream.wait_stream(torch.cuda.current_stream())
        if raw:
            batch.attend(gpu_runner, o, lse, 2, stream=stream.cuda_stream)
        else:
            with torch.cuda.stream(stream):
                batch.attend(gpu_runner, o, lse, 2)
        stream.synchronize()
        batch.check(o, lse, 2)
    o, lse = batch.outputs(True)
    batch.attend(gpu_runner, o, lse, 2, stream=0)
    torch.cuda.synchronize()
    batch.check(o, lse, 2)


def test_caches_past_4_gib(gpu_runner):
    """Codes of more than 2^32 bytes, the pages in use at both ends."""
    page, kv_heads, heads = 64, 8, 16
    pool = (1 << 32) // (page * kv_heads * 64) + 40
    t = Tokens([(90, 90), (65, 65)], heads, kv_heads, page)
    caches = [torch.zeros((pool, kv_heads, page, w), dtype=torch.uint8, device=t.dev) for w in (64, 4, 64, 4)]
    table = t.table.copy()
    table[t.table >= 0] = pool - 1 - np.arange((t.table >= 0).sum()) * 7
    t.table_d.copy_(torch.from_numpy(table))
    t.caches, t.at = caches, table[np.repeat([0, 1], [90, 65]), t.slot // page].astype(np.int64)
    t.append(gpu_runner)
    for j, x in ((0, t.turned(t.k)), (2, t.v[:t.n].float().cpu().numpy())):
        codes, scales = quantise(x)
        assert (caches[j][t.at, :, t.place].cpu().numpy() == codes).all()
        assert (caches[j + 1][t.at, :, t.place].cpu().numpy() == scales).all()
    k, v = torch.empty_like(t.k), torch.empty_like(t.v)
    gpu_runner.call_gather_paged_mx4(*caches, k, v, t.cu, t.table_d)
    for j, x in ((0, k), (2, v)):
        assert torch.equal(x.double(), values(caches[j], caches[j + 1])[t.at, :, t.place])
    batch = Cache4(heads, kv_heads, page, [(90, 90), (65, 65)])
    batch.caches, batch.pages, batch.table_d, batch.q = caches, [table[b, :2].astype(np.int64) for b in (0, 1)], t.table_d, t.q_out
    for lens, q in (([(90, 90), (65, 65)], t.q_out), ([(1, 90), (1, 65)], t.q_out[:2].contiguous())):
        batch.lens, batch.q, batch.total = lens, q, q.shape[0]
        batch.offsets = np.concatenate([[0], np.cumsum([s for s, _ in lens])]).astype(np.int32)
        batch.cu = torch.from_numpy(batch.offsets).to(t.dev)
        batch.max_q = max(s for s, _ in lens)
        o, lse = batch.outputs(True)
        batch.attend(gpu_runner, o, lse, 2)
        batch.check(o, lse, 2)


def test_decode_steps(gpu_runner):
    """A prefill, then decode steps in one graph: append, attend, and the new rows read back; each step against 64-bit
    attention over what the caches hold, and those against the rows that went in."""
    dev, heads, kv_heads, page, batch = "cuda:0", 8, 2, 16, 3
    gen = torch.Generator().manual_seed(4)
    rand = lambda *s: torch.randn(*s, generator=gen).to(torch.bfloat16).to(dev)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=dev)
    lens, steps = [33, 5, 100], 6
    caches = gpu_runner.mx4_caches(24, kv_heads, page, dev)
    table = torch.randperm(24, generator=gen).to(torch.int32).view(batch, 8).to(dev)
    cos, sin = angles(128, 128, dev)
    state = Cache4.__new__(Cache4)
    state.heads, state.kv_heads, state.page, state.dev, state.caches = heads, kv_heads, page, dev, caches
    state.pages = [table[b].cpu().numpy().astype(np.int64) for b in range(batch)]

    def check(new, q, o, k_rows, v_rows, k, v):
        state.lens = [(n, s) for n, s in zip(new, lens)]
        state.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        state.q = q
        state.check(o, None, 2)
        at = 0
        for b, (n, s) in enumerate(state.lens):
            all_k, all_v = state.keys(b)
            assert torch.equal(k_rows[at:at + n].double(), all_k[s - n:]) and torch.equal(v_rows[at:at + n].double(), all_v[s - n:])
            at += n

    cu, seqlens = i32([0, 33, 38, 138]), i32(lens)
    q, k, v = rand(138, heads, D), rand(138, kv_heads, D), rand(138, kv_heads, D)
    o, q_out, k_rows, v_rows = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    gpu_runner.call_append_paged_mx4(q, k, v, q_out, *caches, cu, seqlens, table, cos=cos, sin=sin)
    gpu_runner.call_paged_mx4(q_out, *caches, o, None, cu, seqlens, table, 100, 128, causal=2)
    gpu_runner.call_gather_paged_mx4(*caches, k_rows, v_rows, cu, table)
    check(lens, q_out, o, k_rows, v_rows, k, v)

    cu, starts = i32([0, 1, 2, 3]), i32([0, 0, 0])
    q, k, v = rand(3, heads, D), rand(3, kv_heads, D), rand(3, kv_heads, D)
    o, q_out, k_rows, v_rows = torch.empty_like(q), torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
    ws = torch.empty(gpu_runner.paged_mx4_workspace_size(batch, heads, kv_heads, 1, 128, 3, page, 8, 24, 2),
                     dtype=torch.uint8, device=dev)

    def step():
        gpu_runner.call_append_paged_mx4(q, k, v, q_out, *caches, cu, seqlens, table, cos=cos, sin=sin)
        gpu_runner.call_paged_mx4(q_out, *caches, o, None, cu, seqlens, table, 1, 128, workspace=ws, causal=2)
        gpu_runner.call_gather_paged_mx4(*caches, k_rows, v_rows, cu, table, starts=starts)

    graph = None
    for i in range(steps):
        lens = [s + 1 for s in lens]
        seqlens.copy_(i32(lens))
        starts.copy_(seqlens - 1)
        for x in (q, k, v):
            x.copy_(rand(*x.shape))
        if graph is None:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                step()
        graph.replay()
        torch.cuda.synchronize()
        check([1, 1, 1], q_out, o, k_rows, v_rows, k, v)
